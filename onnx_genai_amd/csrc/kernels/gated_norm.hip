// GatedResidualNorm: the norm behind a block, its gate, the residual stream, and the norm before the next block, in one pass.
//
//   p = post ? unit(block) * post_gamma + post_beta : block
//   z = residual_scale * residual + block_scale * gate * p              -> z, rounded once
//   n = unit(z) * pre_gamma + pre_beta                                  -> n, rounded once, or its 8-bit codes and their scale
//   unit(x) = x / sqrt(mean(x^2) + eps), or (x - mean) / sqrt(var + eps) with `layer`
//
// Memory bounds it: a row is read once into registers, and every statistic, in f32, is taken there (the variance from the differences to the mean, not from
// the difference of two sums). n is made from z as it was before its rounding.
// Measured: 8192 rows of 4096 in bf16 54-56 us (268 MB: 4.9 TB/s, the rate of a copy), one row of 3584 3.6 us, two of them the launch. 333 rows of 2881 in f16 with
// layer norm and gates 6 us: what few rows wait for is their trips to memory one after the other, rows and gate, then, behind the two sums, gamma and beta.
// Codes: scale = max|n| / 127, code = n / scale to the nearest, ties to even.
#include <type_traits>

#include "rows.hiph"

namespace mnb {
namespace {

struct GatedNormParams {
    RocmGatedNormArgs a;
    int vectors;               // pieces of eight elements in a row, the last one perhaps short
    int per_gate;              // rows of a gate
};

__device__ __forceinline__ float add(float a, float b) { return a + b; }
__device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) { return a > b ? a : b; }

// A workgroup has a row; NV: pieces a thread holds. (Four rows of at most 512 elements to a workgroup, a wave each, were level: 32768 rows of 512 23.4 us.)
template <typename T, bool BF16, int NV>
__global__ __launch_bounds__(1024) void gated_norm_kernel(GatedNormParams p)
{
    using V8 = Eight<T, BF16>;
    const RocmGatedNormArgs& a = p.a;
    __shared__ float slots[4][16];
    __shared__ uint32_t slots_max[16];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int waves = blockDim.x >> 6;
    // rows of one gate along x, gates along y: no division for the gate
    const int64_t row = static_cast<int64_t>(blockIdx.y) * p.per_gate + blockIdx.x;
    const int first = threadIdx.x, step = blockDim.x;
    const int h = static_cast<int>(a.hidden);
    const int64_t at = row * h;
    const float inv_h = 1.0f / static_cast<float>(h);
    const T* const residual = static_cast<const T*>(a.residual) + at;
    const T* const block = a.block ? static_cast<const T*>(a.block) + at : nullptr;

    V8 r[NV], y[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int i = first + j * step, left = h - i * 8;
        r[j].zero();
        y[j].zero();
        if (left >= 8) {
            r[j].load(residual + i * 8);
            if (block) y[j].load(block + i * 8);
        } else if (left > 0) {
            r[j].load_first(residual + i * 8, left);
            if (block) y[j].load_first(block + i * 8, left);
        }
    }
    // a weight's eight elements, of the row's type or f32
    auto weight = [&](const void* w, int dtype, int64_t offset, int i, float (&v)[8]) {
        const int left = h - i * 8;
        if (dtype == ROCM_DT_F32) {
            Eight<float, false> e;
            if (left >= 8) e.load(static_cast<const float*>(w) + offset + i * 8);
            else e.load_first(static_cast<const float*>(w) + offset + i * 8, left);
            e.get(v);
        } else {
            V8 e;
            if (left >= 8) e.load(static_cast<const T*>(w) + offset + i * 8);
            else e.load_first(static_cast<const T*>(w) + offset + i * 8, left);
            e.get(v);
        }
    };

    // mean and 1 / sqrt(spread) of x[NV][8]; elements beyond the row are zero and are kept out of the variance
    auto moments = [&](const float (&x)[NV][8], float* slot, float& mean, float& rstd) {
        mean = 0.f;
        if (a.layer) {
            float s = 0.f;
#pragma unroll
            for (int j = 0; j < NV; ++j)
#pragma unroll
                for (int e = 0; e < 8; ++e) s += x[j][e];
            mean = over_workgroup(s, slot, wave, waves, add) * inv_h;
        }
        float s = 0.f;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int left = h - (first + j * step) * 8;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float d = e < left ? x[j][e] - mean : 0.f;
                s = fmaf(d, d, s);
            }
        }
        rstd = 1.0f / sqrtf(over_workgroup(s, slot + 16, wave, waves, add) * inv_h + a.epsilon);
    };

    float z[NV][8];
#pragma unroll
    for (int j = 0; j < NV; ++j) y[j].get(z[j]);
    if (block) {
        float mean = 0.f, rstd = 1.f;
        if (a.post) moments(z, slots[0], mean, rstd);
        const int64_t gate_at = static_cast<int64_t>(blockIdx.y) * h;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int i = first + j * step;
            if (i >= p.vectors) continue;
            float w[8];
            if (a.post) {
#pragma unroll
                for (int e = 0; e < 8; ++e) z[j][e] = (z[j][e] - mean) * rstd;
                if (a.post_gamma) {
                    weight(a.post_gamma, a.post_gamma_dtype, 0, i, w);
#pragma unroll
                    for (int e = 0; e < 8; ++e) z[j][e] *= w[e];
                }
                if (a.post_beta) {
                    weight(a.post_beta, a.post_beta_dtype, 0, i, w);
#pragma unroll
                    for (int e = 0; e < 8; ++e) z[j][e] += w[e];
                }
            }
            if (a.gate) {
                weight(a.gate, a.gate_dtype, gate_at, i, w);
#pragma unroll
                for (int e = 0; e < 8; ++e) z[j][e] *= w[e];
            }
        }
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int i = first + j * step, left = h - i * 8;
        float v[8];
        r[j].get(v);
#pragma unroll
        for (int e = 0; e < 8; ++e) z[j][e] = e < left ? fmaf(a.residual_scale, v[e], a.block_scale * z[j][e]) : 0.f;
        if (a.z && left > 0) {
            V8 o;
            o.set(z[j]);
            T* const to = static_cast<T*>(a.z) + at + i * 8;
            if (left >= 8) o.store(to);
            else o.store_first(to, left);
        }
    }
    if (!a.n) return;

    float mean, rstd;
    moments(z, slots[2], mean, rstd);
    uint32_t amax = 0;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int i = first + j * step, left = h - i * 8;
        if (i >= p.vectors) continue;
        float w[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) z[j][e] = (z[j][e] - mean) * rstd;
        if (a.pre_gamma) {
            weight(a.pre_gamma, a.pre_gamma_dtype, 0, i, w);
#pragma unroll
            for (int e = 0; e < 8; ++e) z[j][e] *= w[e];
        }
        if (a.pre_beta) {
            weight(a.pre_beta, a.pre_beta_dtype, 0, i, w);
#pragma unroll
            for (int e = 0; e < 8; ++e) z[j][e] += w[e];
        }
        if (a.n_scale) {
#pragma unroll
            for (int e = 0; e < 8; ++e) amax = larger(amax, e < left ? __float_as_uint(z[j][e]) & 0x7fffffffu : 0u);
        } else {
            V8 o;
            o.set(z[j]);
            T* const to = static_cast<T*>(a.n) + at + i * 8;
            if (left >= 8) o.store(to);
            else o.store_first(to, left);
        }
    }
    if (!a.n_scale) return;
    const RowScale scale(over_workgroup(amax, slots_max, wave, waves, larger));
    if (first == 0) a.n_scale[row] = scale.scale;
    int8_t* const codes = static_cast<int8_t*>(a.n) + at;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int i = first + j * step, left = h - i * 8;
        if (left <= 0) continue;
        uint32_t d[2] = {0, 0};
#pragma unroll
        for (int e = 0; e < 8; ++e) d[e >> 2] |= static_cast<uint32_t>(scale.code(z[j][e]) & 0xff) << (8 * (e & 3));
        struct __attribute__((packed)) Bytes8 {
            uint32_t x, y;
        };
        if (left >= 8) *reinterpret_cast<Bytes8*>(codes + i * 8) = Bytes8{d[0], d[1]};
        else
            for (int e = 0; e < left; ++e) codes[i * 8 + e] = static_cast<int8_t>(d[e >> 2] >> (8 * (e & 3)));
    }
}

}  // namespace
}  // namespace mnb

extern "C" int rocm_launch_gated_norm(const RocmGatedNormArgs* args, rocm_stream_t stream)
{
    using namespace mnb;
    if (args->rows <= 0 || args->hidden <= 0) return 0;
    if (args->hidden > ROCM_GATED_NORM_MAX_HIDDEN || args->rows > 0x7fffffff) return static_cast<int>(hipErrorInvalidValue);
    hipStream_t s = static_cast<hipStream_t>(stream);
    const int64_t gates = args->gate ? args->rows / args->rows_per_gate : 1, per_gate = args->rows / gates;
    // A grid has 65535 rows and fewer than 2^32 threads: further gates, and further rows of a gate, go in further launches.
    constexpr int64_t kMostGates = 65535, kMostRows = 1 << 21;
    auto go = [&](auto kernel, unsigned threads) {
        const int64_t gates_at_once = per_gate > kMostRows ? 1 : kMostGates, rows_at_once = per_gate > kMostRows ? kMostRows : per_gate;
        for (int64_t g = 0; g < gates; g += gates_at_once)
            for (int64_t r = 0; r < per_gate; r += rows_at_once) {
                const int64_t rows = per_gate - r < rows_at_once ? per_gate - r : rows_at_once, first = g * per_gate + r;
                GatedNormParams part{*args, static_cast<int>((args->hidden + 7) / 8), static_cast<int>(rows)};
                const int64_t item = args->dtype == ROCM_DT_F32 ? 4 : 2, skip = first * args->hidden;
                auto on = [&](auto* x, int64_t bytes) { return x ? reinterpret_cast<decltype(x)>(reinterpret_cast<uintptr_t>(x) + static_cast<uintptr_t>(bytes)) : x; };
                part.a.residual = on(args->residual, skip * item);
                part.a.block = on(args->block, skip * item);
                part.a.z = on(args->z, skip * item);
                part.a.n = on(args->n, skip * (args->n_scale ? 1 : item));
                part.a.n_scale = on(args->n_scale, first * 4);
                part.a.gate = on(args->gate, g * args->hidden * (args->gate_dtype == ROCM_DT_F32 ? 4 : 2));
                const dim3 grid(static_cast<unsigned>(rows), static_cast<unsigned>(gates - g < gates_at_once ? gates - g : gates_at_once));
                hipLaunchKernelGGL(kernel, grid, dim3(threads), 0, s, part);
                const hipError_t e = hipGetLastError();
                if (e != hipSuccess) return static_cast<int>(e);
            }
        return 0;
    };
    const int vectors = static_cast<int>((args->hidden + 7) / 8);
    auto typed = [&](auto t, auto bf) {
        using T = decltype(t);
        constexpr bool BF16 = decltype(bf)::value;
        const unsigned threads = static_cast<unsigned>(vectors + 63) / 64 * 64;
        if (threads <= 1024) return go(gated_norm_kernel<T, BF16, 1>, threads);
        if (threads <= 2048) return go(gated_norm_kernel<T, BF16, 2>, (threads / 2 + 63) / 64 * 64);
        return go(gated_norm_kernel<T, BF16, 4>, 1024);
    };
    if (args->dtype == ROCM_DT_F32) return typed(float{}, std::false_type{});
    if (args->dtype == ROCM_DT_BF16) return typed(uint16_t{}, std::true_type{});
    return typed(uint16_t{}, std::false_type{});
}
