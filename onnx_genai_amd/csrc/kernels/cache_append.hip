// CacheAppend: new tokens' keys and values into their pages, as 8-bit codes with one scale for each page and head.
//
//   fresh page:  scale = max|x| / top over its new tokens, code = x / scale to the nearest, ties to even         (top: 127, or e4m3's 448)
//   begun page:  scale' = max(scale, max|x| / top); where that is larger, the codes before are recoded, code' = code * (scale / scale') to the nearest
//
// A page with an infinity or a NaN has no codes: its scale is NaN and stays it, its codes are 0. A workgroup has one head of one page, keys or values: the scale is a
// maximum over all of it, and keeps its rows in registers from the maximum to the codes. Memory bounds a prompt. Values lie in a page with the tokens of one element
// side by side, as the products that read them want them; a thread has four tokens of eight elements, and so whole dwords of either layout.
//
// 8192 tokens of 8 heads of 128, bf16 to e4m3 (50 MB in and out): 11.2 us, 4.5 TB/s (20.5 with the rows read a second time for the codes). One token each of 48 sequences, 4 heads: 4.6 us, a
// launch and three trips to memory one after the other: lengths, table, rows and scale.
#include <type_traits>

#include "cache.hiph"
#include "rows.hiph"

namespace mnb {
namespace {

constexpr int kThreads = 256;

// Scales from which the quotient that RowScale makes, corrected by its remainder, is the correctly rounded one: int8 needs it from 1/4 on (2^-101), e4m3 down to 2^-11 (2^-90).
template <bool E4M3>
constexpr float kLeastExact = E4M3 ? 8.0779357e-28f : 3.9443045e-31f;

// x / scale as codes, to the nearest, ties to even. EXACT: the scale is kLeastExact or more, and a quotient is at most a rounding above the largest code, to which it goes. Else the quotient is a
// division's, or 0 where the scale is not above 0; and a scale of so few of the smallest f32 steps that it is rounded by much gives quotients far above the largest code, which end there.
template <bool E4M3, bool EXACT>
struct Coder {
    float scale, inverse;
    __device__ __forceinline__ explicit Coder(float s) : scale(s), inverse(EXACT ? 1.0f / s : 0.f) {}
    __device__ __forceinline__ float quotient(float v) const
    {
        if constexpr (EXACT) {
            const float q = v * inverse;
            return fmaf(fmaf(-q, scale, v), inverse, q);
        } else {
            constexpr float kTop = E4M3 ? 448.0f : 127.0f;
            return scale > 0.f ? fminf(fmaxf(v / scale, -kTop), kTop) : 0.f;
        }
    }
    __device__ __forceinline__ uint32_t four(float a, float b, float c, float d) const
    {
        if constexpr (E4M3) {
            int w = __builtin_amdgcn_cvt_pk_fp8_f32(quotient(a), quotient(b), 0, false);
            return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(quotient(c), quotient(d), w, true));
        } else {
            // 1.5 * 2^23 + q has the nearest integer in its lowest bits
            auto bits = [&](float v) { return __float_as_uint(as_f32(quotient(v)) + 12582912.0f); };
            const uint32_t lo = __builtin_amdgcn_perm(bits(b), bits(a), 0x0c0c0400u), hi = __builtin_amdgcn_perm(bits(d), bits(c), 0x0c0c0400u);
            return lo | hi << 16;
        }
    }
};

// The larger of the bits of |x| over eight elements and `most`: 16-bit types two at a time, as their bits order as the values do.
template <typename T, bool BF16>
__device__ __forceinline__ void larger_of(const Eight<T, BF16>& x, uint32_t& most)
{
    if constexpr (sizeof(T) == 2) {
        typedef __attribute__((ext_vector_type(2))) unsigned short short2_t;
        const uint32_t d[4] = {x.raw.x, x.raw.y, x.raw.z, x.raw.w};
#pragma unroll
        for (int i = 0; i < 4; ++i)
            most = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(short2_t, most), __builtin_bit_cast(short2_t, d[i] & 0x7fff7fffu)));
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint32_t bits = __float_as_uint(x.raw[i]) & 0x7fffffffu;
            most = bits > most ? bits : most;
        }
    }
}
template <typename T, bool BF16>
__device__ __forceinline__ uint32_t as_f32_bits(uint32_t most)
{
    if constexpr (sizeof(T) == 2) {
        const uint16_t m = static_cast<uint16_t>((most >> 16) > (most & 0xffff) ? most >> 16 : most);
        return BF16 ? static_cast<uint32_t>(m) << 16 : __float_as_uint(f16_bits_to_f32(m));
    } else {
        return most;
    }
}

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

// UNITS: units of four tokens by eight elements that a thread has at most.
template <typename T, bool BF16, bool E4M3, int UNITS>
__global__ __launch_bounds__(kThreads, UNITS == 1 && sizeof(T) == 2 ? 8 : 1) void append_kernel(RocmCacheAppendArgs a)
{
    __shared__ uint32_t slots_max[4];
    const RocmCache& c = a.cache;
    const int page = c.page, head = blockIdx.y, d = c.head_size;
    const bool values = blockIdx.z != 0;
    auto pages_of = [&](int b) {
        const Sequence s = sequence_of(c, b, static_cast<int>(a.rows));
        return s.rows ? (s.past % page + s.rows + page - 1) / page : 0;
    };
    int b, k;
    if (!find_piece(c.sequences, blockIdx.x, pages_of, &b, &k)) return;
    const Sequence s = sequence_of(c, b, static_cast<int>(a.rows));
    const int begun = s.past % page;
    const int slot = k == 0 ? begun : 0;                 // the page's first new token
    const int passed = k == 0 ? 0 : k * page - begun;    // new tokens in pages before
    const int end = slot + (s.rows - passed < page - slot ? s.rows - passed : page - slot);
    const int p = page_of(c, b, s.past / page + k);
    if (p < 0) return;
    const int64_t at = static_cast<int64_t>(p) * c.kv_heads + head;
    uint32_t* const codes = reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(values ? c.v : c.k) + at * page * d);
    float* const scale_at = (values ? c.v_scale : c.k_scale) + at;
    const int64_t step = values ? a.v_step : a.k_step;
    // row of slot 0 (which is in front of the page's first new token, or is it)
    const T* const from = static_cast<const T*>(values ? a.v : a.k) + (s.first + passed - slot) * step + head * d;

    // Unit u: slots 4 quad .. 4 quad + 3, elements 8 piece ... Keys leave as rows of a token, so pieces run first; values as rows of an element, four tokens to a
    // dword, so quads do (four pieces first there too: 64 bytes of a row together).
    const int pieces = d / 8, quad0 = slot / 4, quads = (end + 3) / 4 - quad0, units = pieces * quads;
    auto place = [&](int u, int& quad, int& piece) {
        if (!values) {
            quad = u / pieces;
            piece = u - quad * pieces;
        } else {
            piece = u / quads;
            quad = u - piece * quads;
        }
        quad += quad0;
    };
    const float old = slot ? *scale_at : 0.f;
    Eight<T, BF16> x[UNITS][4];
    uint32_t amax = 0;
#pragma unroll
    for (int j = 0; j < UNITS; ++j) {
        const int u = threadIdx.x + j * kThreads;
        int quad = 0, piece = 0;
        place(u, quad, piece);
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            const int there = 4 * quad + t;
            x[j][t].zero();
            if (u < units && there >= slot && there < end) x[j][t].load(from + there * step + piece * 8);
        }
    }
#pragma unroll
    for (int j = 0; j < UNITS; ++j)
#pragma unroll
        for (int t = 0; t < 4; ++t) larger_of(x[j][t], amax);
    amax = as_f32_bits<T, BF16>(amax);
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
            __syncthreads();                             // (new codes go to bytes of the same dwords)
        }
    }
    auto write = [&](auto exact) {
        const Coder<E4M3, decltype(exact)::value> coder(none ? 0.f : scale);
#pragma unroll
        for (int j = 0; j < UNITS; ++j) {
            const int u = threadIdx.x + j * kThreads;
            if (u >= units) continue;
            int quad, piece;
            place(u, quad, piece);
            uint32_t w[4][2];                                // of token t: eight codes
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                float e[8];
                x[j][t].get(e);
                w[t][0] = coder.four(e[0], e[1], e[2], e[3]);
                w[t][1] = coder.four(e[4], e[5], e[6], e[7]);
            }
            const int begins = slot - 4 * quad > 0 ? slot - 4 * quad : 0, ends = end - 4 * quad < 4 ? end - 4 * quad : 4;          // new tokens of the four
            if (!values) {
                uint32_t* const to = codes + (4 * quad * d + piece * 8) / 4;
                if (ends - begins == 4) {
#pragma unroll
                    for (int t = 0; t < 4; ++t) *reinterpret_cast<uint2*>(to + t * d / 4) = make_uint2(w[t][0], w[t][1]);
                } else {
                    for (int t = begins; t < ends; ++t) {
                        const uint32_t lo = t == 0 ? w[0][0] : t == 1 ? w[1][0] : t == 2 ? w[2][0] : w[3][0], hi = t == 0 ? w[0][1] : t == 1 ? w[1][1] : t == 2 ? w[2][1] : w[3][1];
                        *reinterpret_cast<uint2*>(to + t * d / 4) = make_uint2(lo, hi);
                    }
                }
            } else {
                uint32_t four[8];                            // of element i: the codes of the four tokens
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const uint32_t sel = 0x0c0c0400u + (i & 3) * 0x0101u;
                    four[i] = __builtin_amdgcn_perm(w[1][i >> 2], w[0][i >> 2], sel) | __builtin_amdgcn_perm(w[3][i >> 2], w[2][i >> 2], sel) << 16;
                }
                uint8_t* const to = reinterpret_cast<uint8_t*>(codes) + piece * 8 * page + 4 * quad;
                if (ends - begins == 4) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) *reinterpret_cast<uint32_t*>(to + i * page) = four[i];
                } else {
                    // (the other bytes of the dword are old tokens', or nobody's and to be left alone)
                    for (int t = begins; t < ends; ++t)
#pragma unroll
                        for (int i = 0; i < 8; ++i) to[i * page + t] = static_cast<uint8_t>(four[i] >> (8 * t));
                }
            }
        }
    };
    if (!none && scale >= kLeastExact<E4M3>) write(std::true_type{});
    else write(std::false_type{});
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
    if (pages >= (1 << 24)) return static_cast<int>(hipErrorInvalidValue);          // (a grid has fewer than 2^32 threads a side)
    const dim3 grid(static_cast<unsigned>(pages < args->rows ? pages : args->rows), static_cast<unsigned>(c.kv_heads), 2);
    const int units = c.head_size / 8 * (c.page / 4);          // of a whole page; few new tokens fill the first of a thread's alone
    auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, grid, dim3(kThreads), 0, s, *args);
        return static_cast<int>(hipGetLastError());
    };
    auto typed = [&](auto t, auto bf) {
        using T = decltype(t);
        constexpr bool BF16 = decltype(bf)::value;
        auto coded = [&](auto e4m3) {
            constexpr bool E4M3 = decltype(e4m3)::value;
            if (units <= kThreads) return go(append_kernel<T, BF16, E4M3, 1>);
            if (units <= 2 * kThreads) return go(append_kernel<T, BF16, E4M3, 2>);
            return go(append_kernel<T, BF16, E4M3, 4>);
        };
        return c.code_dtype == ROCM_DT_E4M3 ? coded(std::true_type{}) : coded(std::false_type{});
    };
    if (args->dtype == ROCM_DT_F32) return typed(float{}, std::false_type{});
    if (args->dtype == ROCM_DT_BF16) return typed(uint16_t{}, std::true_type{});
    return typed(uint16_t{}, std::false_type{});
}
