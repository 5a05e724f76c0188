// CacheAppend: new tokens' keys and values into their pages, as 8-bit codes with one scale for each page and head.
//
//   fresh page:  scale = max|x| / top over its new tokens, code = x / scale to the nearest, ties to even         (top: 127, or e4m3's 448)
//   begun page:  scale' = max(scale, max|x| / top); where that is larger, the codes before are recoded, code' = code * (scale / scale') to the nearest
//
// A page with an infinity or a NaN has no codes: its scale is NaN and stays it, its codes are 0. A workgroup has one head of one page, keys or values: the scale is a
// maximum over all of it. Memory bounds a prompt: rows come in twice, the second time out of the caches, and codes leave in whole dwords. Values lie in a page with
// the tokens of one element side by side, as the products that read them want them, and turn round in LDS.
#include <type_traits>

#include "cache.hiph"
#include "rows.hiph"

namespace mnb {
namespace {

constexpr int kThreads = 256;

// x / scale as a code's byte. The quotient as RowScale has it; e4m3 needs it correctly rounded down to 2^-11, where the remainder is exact for scales of 2^-90 or more.
template <bool E4M3>
struct Coder {
    RowScale s;
    __device__ __forceinline__ explicit Coder(float scale)
    {
        s.scale = scale;
        s.inverse = scale > 0.f ? 1.0f / scale : 0.f;
    }
    __device__ __forceinline__ float quotient(float v) const
    {
        float q = v * s.inverse;
        q = fmaf(fmaf(-q, s.scale, v), s.inverse, q);
        if (s.scale < 8.0779357e-28f) q = v / s.scale;
        return s.scale > 0.f ? fminf(fmaxf(q, -448.f), 448.f) : 0.f;
    }
    __device__ __forceinline__ uint32_t four(float a, float b, float c, float d) const
    {
        if constexpr (E4M3) {
            int w = __builtin_amdgcn_cvt_pk_fp8_f32(quotient(a), quotient(b), 0, false);
            return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(quotient(c), quotient(d), w, true));
        } else {
            return (s.code(a) & 0xff) | (s.code(b) & 0xff) << 8 | (s.code(c) & 0xff) << 16 | static_cast<uint32_t>(s.code(d)) << 24;
        }
    }
};

// Four codes times `ratio` (<= 1), to the nearest; ratio 0 clears them.
template <bool E4M3>
__device__ __forceinline__ uint32_t recoded(uint32_t w, float ratio)
{
    if constexpr (E4M3) {
        const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w), false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w), true);
        const int a = __builtin_amdgcn_cvt_pk_fp8_f32(lo[0] * ratio, lo[1] * ratio, 0, false);
        return ratio > 0.f ? static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(hi[0] * ratio, hi[1] * ratio, a, true)) : 0u;
    } else {
        uint32_t out = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float v = static_cast<float>(static_cast<int8_t>(w >> (8 * i)));
            out |= (static_cast<uint32_t>(static_cast<int>(__builtin_rintf(v * ratio))) & 0xff) << (8 * i);
        }
        return ratio > 0.f ? out : 0u;
    }
}

__device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) { return a > b ? a : b; }

template <typename T, bool BF16, bool E4M3>
__global__ __launch_bounds__(kThreads) void append_kernel(RocmCacheAppendArgs a)
{
    __shared__ uint32_t slots_max[4];
    extern __shared__ uint32_t turned[];                 // values: [head_size][page + 4] bytes
    const RocmCache& c = a.cache;
    const int page = c.page, head = blockIdx.y, d = c.head_size;
    const bool values = blockIdx.z != 0;
    auto pages_of = [&](int b) {
        const Sequence s = sequence_of(c, b, static_cast<int>(a.rows));
        return s.rows ? (s.past % page + s.rows + page - 1) / page : 0;
    };
    int b, k, unused;
    if (!find_piece(c.sequences, blockIdx.x, pages_of, [](int) { return 0; }, &b, &k, &unused)) return;
    const Sequence s = sequence_of(c, b, static_cast<int>(a.rows));
    const int begun = s.past % page;
    const int slot = k == 0 ? begun : 0;                 // the page's first new token
    const int passed = k == 0 ? 0 : k * page - begun;    // new tokens in pages before
    const int count = s.rows - passed < page - slot ? s.rows - passed : page - slot;
    const int p = page_of(c, b, s.past / page + k);
    if (p < 0) return;
    const int64_t at = static_cast<int64_t>(p) * c.kv_heads + head;
    uint32_t* const codes = reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(values ? c.v : c.k) + at * page * d);
    float* const scale_at = (values ? c.v_scale : c.k_scale) + at;
    const int64_t step = values ? a.v_step : a.k_step;
    const T* const from = static_cast<const T*>(values ? a.v : a.k) + (s.first + passed) * step + head * d;

    const int pieces = d / 8, tokens = kThreads / pieces;        // pieces of eight elements in a row of the head, rows at once
    const int row0 = threadIdx.x / pieces, piece = threadIdx.x - row0 * pieces;
    uint32_t amax = 0;
    if (row0 < tokens) {
        for (int t = row0; t < count; t += tokens) {
            Eight<T, BF16> x;
            float e[8];
            x.load(from + t * step + piece * 8);
            x.get(e);
#pragma unroll
            for (int i = 0; i < 8; ++i) amax = larger(amax, __float_as_uint(e[i]) & 0x7fffffffu);
        }
    }
    const float old = slot ? *scale_at : 0.f;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    amax = over_workgroup(amax, slots_max, wave, kThreads / 64, larger);
    float scale = amax >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : __uint_as_float(amax) / (E4M3 ? 448.0f : 127.0f);
    const bool none = !(scale == scale) || !(old == old);
    if (none) scale = __uint_as_float(0x7fc00000u);
    else if (old > scale) scale = old;
    if (threadIdx.x == 0) *scale_at = scale;

    if (slot && (none || scale != old)) {
        const float ratio = none || !(scale > 0.f) ? 0.f : old / scale;
        if (!values) {
            const int words = slot * d / 4;
            for (int i = threadIdx.x; i < words; i += kThreads) codes[i] = recoded<E4M3>(codes[i], ratio);
        } else {
            const int words = (slot + 3) / 4, each = page / 4, all = d * words;
            for (int i = threadIdx.x; i < all; i += kThreads) {
                const int row = i / words, j = i - row * words, left = slot - 4 * j;
                const uint32_t w = codes[row * each + j], keep = left >= 4 ? 0u : 0xffffffffu << (8 * left);
                codes[row * each + j] = (recoded<E4M3>(w, ratio) & ~keep) | (w & keep);
            }
        }
    }
    const Coder<E4M3> coder(none ? 0.f : scale);
    if (row0 < tokens) {
        for (int t = row0; t < count; t += tokens) {
            Eight<T, BF16> x;
            float e[8];
            x.load(from + t * step + piece * 8);
            x.get(e);
            const uint32_t lo = coder.four(e[0], e[1], e[2], e[3]), hi = coder.four(e[4], e[5], e[6], e[7]);
            if (!values) {
                uint2* const to = reinterpret_cast<uint2*>(codes + ((slot + t) * d + piece * 8) / 4);
                *to = make_uint2(lo, hi);
            } else {
                uint8_t* const to = reinterpret_cast<uint8_t*>(turned) + slot + t;
#pragma unroll
                for (int i = 0; i < 8; ++i) to[(piece * 8 + i) * (page + 4)] = static_cast<uint8_t>((i < 4 ? lo : hi) >> (8 * (i & 3)));
            }
        }
    }
    if (!values) return;
    // rows of one element: whole dwords of new tokens, and bytes where old ones (or nobody's) are in the same dword
    __syncthreads();
    const int first = slot / 4, words = (slot + count + 3) / 4 - first, each = page / 4, all = d * words;
    for (int i = threadIdx.x; i < all; i += kThreads) {
        const int row = i / words, j = first + (i - row * words);
        const uint32_t w = turned[row * (each + 1) + j];
        if (4 * j >= slot && 4 * j + 4 <= slot + count) {
            codes[row * each + j] = w;
        } else {
            uint8_t* const to = reinterpret_cast<uint8_t*>(codes + row * each + j);
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (4 * j + e >= slot && 4 * j + e < slot + count) to[e] = static_cast<uint8_t>(w >> (8 * e));
        }
    }
}

}  // namespace
}  // namespace mnb

extern "C" int rocm_launch_cache_append(const RocmCacheAppendArgs* args, rocm_stream_t stream)
{
    using namespace mnb;
    const RocmCache& c = args->cache;
    if (args->rows <= 0 || c.sequences <= 0) return 0;
    if (c.page < 16 || c.page > ROCM_CACHE_MAX_PAGE || (c.page & (c.page - 1)) != 0 || c.head_size < 16 || c.head_size > ROCM_CACHE_MAX_HEAD || c.head_size % 16 != 0 || args->rows >= (1 << 30) ||
        c.kv_heads < 1 || c.kv_heads > 65535)
        return static_cast<int>(hipErrorInvalidValue);
    hipStream_t s = static_cast<hipStream_t>(stream);
    // a sequence with n tokens touches at most n / page + 2 pages, and at most n
    const int64_t pages = args->rows < c.sequences ? args->rows : args->rows / c.page + 2 * static_cast<int64_t>(c.sequences);
    const dim3 grid(static_cast<unsigned>(pages < args->rows ? pages : args->rows), static_cast<unsigned>(c.kv_heads), 2);
    const unsigned lds = static_cast<unsigned>(c.head_size * (c.page + 4));
    auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, grid, dim3(kThreads), lds, s, *args);
        return static_cast<int>(hipGetLastError());
    };
    auto typed = [&](auto t, auto bf) {
        using T = decltype(t);
        constexpr bool BF16 = decltype(bf)::value;
        return c.code_dtype == ROCM_DT_E4M3 ? go(append_kernel<T, BF16, true>) : go(append_kernel<T, BF16, false>);
    };
    if (args->dtype == ROCM_DT_F32) return typed(float{}, std::false_type{});
    if (args->dtype == ROCM_DT_BF16) return typed(uint16_t{}, std::true_type{});
    return typed(uint16_t{}, std::false_type{});
}
