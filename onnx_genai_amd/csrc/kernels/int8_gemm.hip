// MatMulInt8: a product in 8-bit integers with one scale per token and one per output channel.
//
//   s_m = max_k |a_mk| / 127,  q_mk = a_mk / s_m to the nearest, ties to even          (quantize_rows_kernel, or the caller's codes)
//   y_mn = (sum_k q_mk b_nk) * s_m * s_n + bias                                         (the sum is an exact int32 for K < 2^17)
//
// Codes lie in rows of kp = K rounded up to 128 bytes, zeros behind K: the products read whole steps of K, and what they read of B behind the end of its row
// (the next row, or nothing) meets a zero.
#include <type_traits>

#include "mfma_common.hiph"
#include "rows.hiph"

namespace mnb {
namespace {

typedef __attribute__((ext_vector_type(4))) int i32x4_t;
typedef __attribute__((ext_vector_type(16))) int i32x16_t;

__device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) { return a > b ? a : b; }

// One workgroup a row: the largest magnitude, then the codes from a second read, which comes from L2. Memory bounds it.
template <typename T, bool BF16>
__global__ __launch_bounds__(256) void quantize_rows_kernel(const T* __restrict__ a, int64_t k, int64_t kp, int8_t* __restrict__ codes, float* __restrict__ scales)
{
    using V8 = Eight<T, BF16>;
    __shared__ uint32_t slots[16];
    const int64_t row = blockIdx.x;
    const T* const x = a + row * k;
    const int vectors = static_cast<int>(kp / 8);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    auto piece = [&](int i, float (&v)[8]) {
        V8 e;
        const int left = static_cast<int>(k) - i * 8;
        if (left >= 8) e.load(x + i * 8);
        else if (left > 0) e.load_first(x + i * 8, left);
        else e.zero();
        e.get(v);
    };
    uint32_t amax = 0;
    for (int i = threadIdx.x; i < vectors; i += 256) {
        float v[8];
        piece(i, v);
#pragma unroll
        for (int e = 0; e < 8; ++e) amax = larger(amax, __float_as_uint(v[e]) & 0x7fffffffu);
    }
    const RowScale scale(over_workgroup(amax, slots, wave, 4, larger));
    if (threadIdx.x == 0) scales[row] = scale.scale;
    for (int i = threadIdx.x; i < vectors; i += 256) {
        float v[8];
        piece(i, v);
        uint32_t d[2] = {0, 0};
#pragma unroll
        for (int e = 0; e < 8; ++e) d[e >> 2] |= static_cast<uint32_t>(scale.code(v[e]) & 0xff) << (8 * (e & 3));
        *reinterpret_cast<uint2*>(codes + row * kp + i * 8) = make_uint2(d[0], d[1]);
    }
}

// Rows of k bytes -> rows of kp bytes, zeros behind.
__global__ __launch_bounds__(256) void pad_codes_kernel(const int8_t* __restrict__ from, int64_t k, int64_t kp, int8_t* __restrict__ to)
{
    const int64_t row = blockIdx.y;
    const int64_t i = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) * 8;
    if (i >= kp) return;
    uint32_t d[2] = {0, 0};
#pragma unroll
    for (int e = 0; e < 8; ++e)
        if (i + e < k) d[e >> 2] |= static_cast<uint32_t>(static_cast<uint8_t>(from[row * k + i + e])) << (8 * (e & 3));
    *reinterpret_cast<uint2*>(to + row * kp + i) = make_uint2(d[0], d[1]);
}

struct Int8Params {
    const int8_t* a;           // [m, lda] codes
    const float* a_scale;
    const int8_t* b;           // [n, ldb]
    const void* b_scale;
    const void* bias;
    void* y;
    int32_t* partial;          // [slices][m][n] sums of a slice of K, or NULL
    int64_t m, n, lda, ldb;
    int steps;                 // of 128 k
    int steps_per_slice;
    int b_scale_dtype, bias_dtype, y_dtype;
};

__device__ __forceinline__ void store_scaled(const Int8Params& p, int64_t row, int64_t col, int32_t sum, float a_scale, float b_scale)
{
    const float v = static_cast<float>(sum) * a_scale * b_scale;
    store_from_f32(p.y, p.y_dtype, row * p.n + col, with_bias(v, p.bias, p.bias_dtype, row, p.n, col, p.y_dtype));
}

// Few rows: a workgroup has 16 columns, its waves split K. v_mfma_i32_16x16x64_i8: lane l holds 16 bytes of k of row (or column) l % 16, k from (l / 16) * 16.
// RT: tiles of 16 rows.
template <int RT>
__global__ __launch_bounds__(512) void int8_rows_kernel(Int8Params p)
{
    __shared__ int32_t sums[8][RT * 4][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const int c = lane & 15, g = lane >> 4;
    const int64_t n0 = static_cast<int64_t>(blockIdx.x) * 16;
    const int64_t cols = p.n - n0 < 16 ? p.n - n0 : 16;
    const auto srd_b = make_srd(p.b + n0 * p.ldb, static_cast<uint64_t>(cols * p.ldb));
    const auto srd_a = make_srd(p.a, static_cast<uint64_t>(p.m * p.lda));
    const int per_wave = (p.steps + waves - 1) / waves;
    const int begin = wave * per_wave, end = min(begin + per_wave, p.steps);
    const uint32_t b_at = c < cols ? static_cast<uint32_t>(c * p.ldb + g * 16) : kOutOfRange;
    uint32_t a_at[RT];
    i32x4_t acc[RT] = {};
#pragma unroll
    for (int r = 0; r < RT; ++r) a_at[r] = r * 16 + c < p.m ? static_cast<uint32_t>((r * 16 + c) * p.lda + g * 16) : kOutOfRange;
#pragma unroll 2
    for (int t = begin; t < end; ++t) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint32_t k = static_cast<uint32_t>(t) * 128u + h * 64u;
            const i32x4_t b = __builtin_bit_cast(i32x4_t, load16(srd_b, b_at + k, 0));
#pragma unroll
            for (int r = 0; r < RT; ++r) acc[r] = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4_t, load16(srd_a, a_at[r] + k, 0)), b, acc[r], 0, 0, 0);
        }
    }
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int i = 0; i < 4; ++i) sums[wave][r * 4 + i][lane] = acc[r][i];
    __syncthreads();
    const int64_t col = n0 + c;
    if (c >= cols) return;
    const float sb = load_as_f32(p.b_scale, p.b_scale_dtype, col);
    for (int j = wave; j < RT * 4; j += waves) {
        const int64_t row = (j >> 2) * 16 + g * 4 + (j & 3);
        if (row >= p.m) continue;
        int32_t sum = 0;
        for (int w = 0; w < waves; ++w) sum += sums[w][j][lane];
        store_scaled(p, row, col, sum, p.a_scale[row], sb);
    }
}

// Tall calls: 128 x 128 tiles.
__global__ __launch_bounds__(256) void int8_tile_kernel(Int8Params p)
{
    __shared__ __attribute__((aligned(16))) uint8_t smem[2 * 128 * 144];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t m0 = static_cast<int64_t>(blockIdx.y) * 128, n0 = static_cast<int64_t>(blockIdx.x) * 128;
    const int64_t rows = p.m - m0 < 128 ? p.m - m0 : 128, cols = p.n - n0 < 128 ? p.n - n0 : 128;
    const auto srd_a = make_srd(p.a + m0 * p.lda, static_cast<uint64_t>(rows * p.lda));
    const auto srd_b = make_srd(p.b + n0 * p.ldb, static_cast<uint64_t>(cols * p.ldb));
    const int wm = (wave & 1) * 64, wn = (wave >> 1) * 64;
    i32x16_t acc[2][2] = {};
    for (int t = 0; t < p.steps; ++t) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int id = threadIdx.x + i * 256, r = id >> 3, ch = id & 7;
            const uint4 va = load16(srd_a, r < rows ? static_cast<uint32_t>(r * p.lda + ch * 16 + t * 128) : kOutOfRange, 0);
            const uint4 vb = load16(srd_b, r < cols ? static_cast<uint32_t>(r * p.ldb + ch * 16 + t * 128) : kOutOfRange, 0);
            *reinterpret_cast<uint4*>(smem + r * 144 + ch * 16) = va;
            *reinterpret_cast<uint4*>(smem + 128 * 144 + r * 144 + ch * 16) = vb;
        }
        __syncthreads();
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            i32x4_t a[2], b[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                a[i] = *reinterpret_cast<const i32x4_t*>(smem + (wm + i * 32 + (lane & 31)) * 144 + s * 32 + (lane >> 5) * 16);
                b[i] = *reinterpret_cast<const i32x4_t*>(smem + 128 * 144 + (wn + i * 32 + (lane & 31)) * 144 + s * 32 + (lane >> 5) * 16);
            }
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(a[i], b[j], acc[i][j], 0, 0, 0);
        }
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int64_t col = n0 + wn + j * 32 + (lane & 31);
        if (col >= p.n) continue;
        const float sb = load_as_f32(p.b_scale, p.b_scale_dtype, col);
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int64_t row = m0 + wm + i * 32 + (e >> 2) * 8 + (lane >> 5) * 4 + (e & 3);
                if (row < p.m) store_scaled(p, row, col, acc[i][j][e], p.a_scale[row], sb);
            }
    }
}

Int8Params params_of(const RocmInt8Args* a)
{
    Int8Params p{};
    p.a = a->a;
    p.a_scale = a->a_scale;
    p.b = a->b;
    p.b_scale = a->b_scale;
    p.bias = a->bias;
    p.y = a->y;
    p.m = a->m;
    p.n = a->n;
    p.lda = a->lda;
    p.ldb = a->ldb;
    p.steps = static_cast<int>((a->k + 127) / 128);
    p.b_scale_dtype = a->b_scale_dtype;
    p.bias_dtype = a->bias_dtype;
    p.y_dtype = a->y_dtype;
    return p;
}

}  // namespace
}  // namespace mnb

extern "C" int rocm_launch_quantize_rows(const void* a, int dtype, int64_t m, int64_t k, int8_t* codes, float* scales, rocm_stream_t stream)
{
    using namespace mnb;
    if (m <= 0 || k <= 0) return 0;
    if (m > 0x7fffffff || k >= ROCM_INT8_MAX_K) return static_cast<int>(hipErrorInvalidValue);
    const int64_t kp = (k + 127) / 128 * 128;
    hipStream_t s = static_cast<hipStream_t>(stream);
    auto go = [&](auto kernel, auto* x) {
        hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(m)), dim3(256), 0, s, x, k, kp, codes, scales);
        return static_cast<int>(hipGetLastError());
    };
    if (dtype == ROCM_DT_F32) return go(quantize_rows_kernel<float, false>, static_cast<const float*>(a));
    if (dtype == ROCM_DT_BF16) return go(quantize_rows_kernel<uint16_t, true>, static_cast<const uint16_t*>(a));
    return go(quantize_rows_kernel<uint16_t, false>, static_cast<const uint16_t*>(a));
}

extern "C" int rocm_launch_pad_codes(const int8_t* from, int64_t rows, int64_t k, int8_t* to, rocm_stream_t stream)
{
    using namespace mnb;
    const int64_t kp = (k + 127) / 128 * 128;
    for (int64_t r = 0; r < rows; r += 65535) {
        const unsigned part = static_cast<unsigned>(rows - r < 65535 ? rows - r : 65535);
        hipLaunchKernelGGL(pad_codes_kernel, dim3(static_cast<unsigned>((kp / 8 + 255) / 256), part), dim3(256), 0, static_cast<hipStream_t>(stream), from + r * k, k, kp, to + r * kp);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return static_cast<int>(e);
    }
    return 0;
}

extern "C" int rocm_int8_pads_b(const RocmInt8Args* args) { return args->k % 16 != 0; }
extern "C" uint64_t rocm_int8_scratch_bytes(const RocmInt8Args*) { return 0; }
extern "C" const char* rocm_int8_variant(const RocmInt8Args* args) { return args->m <= 64 ? "int8_rows" : "int8_tile"; }

extern "C" int rocm_launch_int8(const RocmInt8Args* args, rocm_stream_t stream)
{
    using namespace mnb;
    if (args->m <= 0 || args->n <= 0) return 0;
    hipStream_t s = static_cast<hipStream_t>(stream);
    const Int8Params p = params_of(args);
    if (args->m <= 64) {
        const unsigned grid = static_cast<unsigned>((p.n + 15) / 16), threads = 512;
        auto go = [&](auto kernel) {
            hipLaunchKernelGGL(kernel, dim3(grid), dim3(threads), 0, s, p);
            return static_cast<int>(hipGetLastError());
        };
        return p.m <= 16 ? go(int8_rows_kernel<1>) : p.m <= 32 ? go(int8_rows_kernel<2>) : go(int8_rows_kernel<4>);
    }
    hipLaunchKernelGGL(int8_tile_kernel, dim3(static_cast<unsigned>((p.n + 127) / 128), static_cast<unsigned>((p.m + 127) / 128)), dim3(256), 0, s, p);
    return static_cast<int>(hipGetLastError());
}
