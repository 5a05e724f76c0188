// RotaryEmbedding: pairs (a, b) of a head's elements turned by their row's position,
//   a' = a cos - b sin,  b' = b cos + a sin,  angle of pair i = position * frequency_i,
// pairs (i, i + part / 2), or (2 i, 2 i + 1) with `interleaved`. Elements beyond `part` of a head, and what lies behind the heads, pass through.
//
// Memory bounds it: a row is read once and written once. A workgroup has a row, or some heads of it where there are few rows, so that the angles, taken in 64 bits,
// are computed once for all of its heads: positions reach millions, where a 32-bit product of position and frequency is off by tenths of a radian. The
// angle is kept in turns, of which the whole ones are dropped exactly; what is left, within an eighth of a turn of a quarter, goes through the Taylor series.
//
// 8192 rows of 48 heads of 128 in bf16 (201 MB read and written): 39.6 us, 5.1 TB/s, what a copy takes. One row: 4.5 us, a launch and two trips to memory.
#include <type_traits>

#include "rows.hiph"

namespace mnb {
namespace {

constexpr int kThreads = 256;

// cos and sin of 2 pi t, t any number of turns. Quarters are taken off exactly; the series for |x| <= pi / 4 end where the next term is below 2^-48.
__device__ __forceinline__ void cos_sin_of_turns(double t, double& c, double& s)
{
    const double r = t - __builtin_rint(t);
    const double quarters = __builtin_rint(4.0 * r);
    const double x = 6.283185307179586 * (r - 0.25 * quarters), x2 = x * x;
    double sn = 1.0 / 6227020800.0, cn = -1.0 / 87178291200.0;
    sn = fma(sn, x2, -1.0 / 39916800.0);
    sn = fma(sn, x2, 1.0 / 362880.0);
    sn = fma(sn, x2, -1.0 / 5040.0);
    sn = fma(sn, x2, 1.0 / 120.0);
    sn = fma(sn, x2, -1.0 / 6.0);
    sn = fma(sn * x2, x, x);
    cn = fma(cn, x2, 1.0 / 479001600.0);
    cn = fma(cn, x2, -1.0 / 3628800.0);
    cn = fma(cn, x2, 1.0 / 40320.0);
    cn = fma(cn, x2, -1.0 / 720.0);
    cn = fma(cn, x2, 1.0 / 24.0);
    cn = fma(cn, x2, -0.5);
    cn = fma(cn, x2, 1.0);
    const int q = static_cast<int>(quarters) & 3;
    const double a = (q & 1) ? sn : cn, b = (q & 1) ? cn : sn;
    c = (q == 1 || q == 2) ? -a : a;
    s = (q & 2) ? -b : b;
}

__device__ __forceinline__ int64_t position_of(const RocmRotaryArgs& a, int64_t row, int64_t in_run)
{
    const int64_t i = a.one_position ? 0 : row;
    const int64_t p = a.positions_dtype == ROCM_DT_I64 ? static_cast<const int64_t*>(a.positions)[i] : static_cast<const int32_t*>(a.positions)[i];
    return a.one_position ? p + in_run : p;
}

struct RotaryPlan {
    int64_t first_row;
    int heads_at_once;      // heads a workgroup turns
    int turned;             // pieces of eight elements (of eight pairs, unless interleaved) that turn, in a head
    int passed;             // pieces of a head that pass through; 0 where y is x
    int extra;              // pieces behind the last head that pass through
};

template <typename T, bool BF16, bool INTERLEAVED>
__global__ __launch_bounds__(kThreads) void rotary_kernel(RocmRotaryArgs a, RotaryPlan p)
{
    using V8 = Eight<T, BF16>;
    __shared__ float cosines[ROCM_ROTARY_MAX_PAIRS], sines[ROCM_ROTARY_MAX_PAIRS];
    const int64_t row = p.first_row + blockIdx.x, run = row / a.inner, in_run = row - run * a.inner;
    const int64_t base = run * a.outer_step + in_run * a.row_step;
    const int half = a.part / 2;
    const int64_t position = position_of(a, row, in_run);
    for (int i = threadIdx.x; i < half; i += kThreads) {
        float c, s;
        if (a.cos_cache) {
            // a position without a row in the caches gives NaN
            const bool there = position >= 0 && position < a.cache_rows;
            c = there ? load_as_f32(a.cos_cache, a.cache_dtype, position * half + i) : __uint_as_float(0x7fc00000u);
            s = there ? load_as_f32(a.sin_cache, a.cache_dtype, position * half + i) : __uint_as_float(0x7fc00000u);
        } else {
            double cd, sd;
            cos_sin_of_turns(static_cast<double>(position) * a.turns[i], cd, sd);
            c = static_cast<float>(cd * a.magnitude);
            s = static_cast<float>(sd * a.magnitude);
        }
        cosines[i] = c;
        sines[i] = s;
    }
    __syncthreads();

    const T* const x = static_cast<const T*>(a.x) + base;
    T* const y = static_cast<T*>(a.y) + base;
    auto get = [](float (&e)[8], const T* from, int left) {
        V8 v;
        if (left >= 8) v.load(from);
        else v.load_first(from, left);
        v.get(e);
    };
    auto put = [](const float (&e)[8], T* to, int left) {
        V8 v;
        v.set(e);
        if (left >= 8) v.store(to);
        else v.store_first(to, left);
    };
    const int first_head = blockIdx.y * p.heads_at_once;
    const int heads = a.heads - first_head < p.heads_at_once ? a.heads - first_head : p.heads_at_once;
    const int pieces = p.turned + p.passed, all = heads * pieces;
    for (int u = threadIdx.x; u < all; u += kThreads) {
        const int h = u / pieces, j = u - h * pieces;
        const int64_t head = (first_head + h) * a.head_step;
        if (j >= p.turned) {
            const int at = a.part + (j - p.turned) * 8;
            float e[8];
            get(e, x + head + at, a.head_size - at);
            put(e, y + head + at, a.head_size - at);
        } else if (INTERLEAVED) {
            const int at = j * 8, left = a.part - at;
            float e[8];
            get(e, x + head + at, left);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int pair = at / 2 + i < half ? at / 2 + i : half - 1;
                const float c = cosines[pair], s = sines[pair], first = e[2 * i], second = e[2 * i + 1];
                e[2 * i] = fmaf(first, c, -(second * s));
                e[2 * i + 1] = fmaf(second, c, first * s);
            }
            put(e, y + head + at, left);
        } else {
            const int at = j * 8, left = half - at;
            float e[8], f[8];
            get(e, x + head + at, left);
            get(f, x + head + half + at, left);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int pair = at + i < half ? at + i : half - 1;
                const float c = cosines[pair], s = sines[pair], first = e[i], second = f[i];
                e[i] = fmaf(first, c, -(second * s));
                f[i] = fmaf(second, c, first * s);
            }
            put(e, y + head + at, left);
            put(f, y + head + half + at, left);
        }
    }
    if (blockIdx.y == 0) {
        const int64_t behind = static_cast<int64_t>(a.heads) * a.head_step;
        for (int u = threadIdx.x; u < p.extra; u += kThreads) {
            const int64_t at = static_cast<int64_t>(u) * 8, left = a.extra - at;
            float e[8];
            get(e, x + behind + at, left < 8 ? static_cast<int>(left) : 8);
            put(e, y + behind + at, left < 8 ? static_cast<int>(left) : 8);
        }
    }
}

}  // namespace
}  // namespace mnb

extern "C" int rocm_launch_rotary(const RocmRotaryArgs* args, rocm_stream_t stream)
{
    using namespace mnb;
    if (args->rows <= 0) return 0;
    if (args->heads < 1 || args->part < 2 || args->part % 2 != 0 || args->part > args->head_size || args->part / 2 > ROCM_ROTARY_MAX_PAIRS || args->inner < 1) return static_cast<int>(hipErrorInvalidValue);
    hipStream_t s = static_cast<hipStream_t>(stream);
    RotaryPlan plan{};
    plan.turned = args->interleaved ? (args->part + 7) / 8 : (args->part / 2 + 7) / 8;
    if (args->x != args->y) {
        plan.passed = (args->head_size - args->part + 7) / 8;
        plan.extra = static_cast<int>((args->extra + 7) / 8);
    }
    // A row to a workgroup once there are eight rows for each CU, as many as run on it at once; before that a row's heads are dealt out, and its angles repeated for each part. (777 rows of
    // 64 heads of 80: 8.1 us with three workgroups a row, some of which run in a second round, with one a row 8.7; two were not timed.)
    const int64_t most = 8 * static_cast<int64_t>(rocm_ffi_compute_units());
    int64_t parts = args->rows >= most ? 1 : (most + args->rows - 1) / args->rows;
    if (parts > args->heads) parts = args->heads;
    plan.heads_at_once = static_cast<int>((args->heads + parts - 1) / parts);
    const unsigned groups = static_cast<unsigned>((args->heads + plan.heads_at_once - 1) / plan.heads_at_once);
    auto go = [&](auto kernel) {
        constexpr int64_t kMostRows = 1 << 21;
        for (int64_t r = 0; r < args->rows; r += kMostRows) {
            plan.first_row = r;
            const int64_t rows = args->rows - r < kMostRows ? args->rows - r : kMostRows;
            hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(rows), groups), dim3(kThreads), 0, s, *args, plan);
            const hipError_t e = hipGetLastError();
            if (e != hipSuccess) return static_cast<int>(e);
        }
        return 0;
    };
    auto typed = [&](auto t, auto bf) {
        using T = decltype(t);
        constexpr bool BF16 = decltype(bf)::value;
        return args->interleaved ? go(rotary_kernel<T, BF16, true>) : go(rotary_kernel<T, BF16, false>);
    };
    if (args->dtype == ROCM_DT_F32) return typed(float{}, std::false_type{});
    if (args->dtype == ROCM_DT_BF16) return typed(uint16_t{}, std::true_type{});
    return typed(uint16_t{}, std::false_type{});
}
