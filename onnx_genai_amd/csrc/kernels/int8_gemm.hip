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

// One workgroup of WAVES waves a row: the largest magnitude, then the codes. The first HELD eights of a thread stay in registers, all loaded before any is looked
// at; what lies behind them is read again. Memory bounds it: 8192 rows of 4096 in bf16 take 26 us (3.9 TB/s), 500 of 18944 take 9 (3.2 TB/s; one read of the row
// after the other took 14).
template <typename T, bool BF16, int WAVES, int HELD>
__global__ __launch_bounds__(WAVES * 64) void quantize_rows_kernel(const T* __restrict__ a, int64_t k, int64_t kp, int8_t* __restrict__ codes, float* __restrict__ scales)
{
    using V8 = Eight<T, BF16>;
    constexpr int kThreads = WAVES * 64;
    __shared__ uint32_t slots[WAVES];
    const int64_t row = blockIdx.x;
    const T* const x = a + row * k;
    const int vectors = static_cast<int>(kp / 8), whole = static_cast<int>(k / 8), rest = static_cast<int>(k & 7);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    V8 held[HELD];
#pragma unroll
    for (int h = 0; h < HELD; ++h) {
        const int i = threadIdx.x + h * kThreads;
        held[h].zero();
        if (i < whole) held[h].load(x + i * 8);
    }
    if (rest)
#pragma unroll
        for (int h = 0; h < HELD; ++h)
            if (static_cast<int>(threadIdx.x) + h * kThreads == whole) held[h].load_first(x + whole * 8, rest);
    auto piece = [&](int i, float (&v)[8]) {
        V8 e;
        if (i < whole) e.load(x + i * 8);
        else if (i == whole && rest) e.load_first(x + i * 8, rest);
        else e.zero();
        e.get(v);
    };
    uint32_t amax = 0;
    float v[8];
    auto look = [&] {
#pragma unroll
        for (int e = 0; e < 8; ++e) amax = larger(amax, __float_as_uint(v[e]) & 0x7fffffffu);
    };
#pragma unroll
    for (int h = 0; h < HELD; ++h) {
        held[h].get(v);
        look();
    }
    for (int i = threadIdx.x + HELD * kThreads; i < vectors; i += kThreads) {
        piece(i, v);
        look();
    }
    const RowScale scale(over_workgroup(amax, slots, wave, WAVES, larger));
    if (threadIdx.x == 0) scales[row] = scale.scale;
    auto put = [&](int i) {
        uint32_t d[2] = {0, 0};
#pragma unroll
        for (int e = 0; e < 8; ++e) d[e >> 2] |= static_cast<uint32_t>(scale.code(v[e]) & 0xff) << (8 * (e & 3));
        *reinterpret_cast<uint2*>(codes + row * kp + i * 8) = make_uint2(d[0], d[1]);
    };
#pragma unroll
    for (int h = 0; h < HELD; ++h) {
        const int i = threadIdx.x + h * kThreads;
        if (i < vectors) {
            held[h].get(v);
            put(i);
        }
    }
    for (int i = threadIdx.x + HELD * kThreads; i < vectors; i += kThreads) {
        piece(i, v);
        put(i);
    }
}

// Rows of k bytes -> rows of kp bytes, zeros behind. Sixteen bytes a thread, from wherever they begin: the hardware takes such loads whole. (24 rows of 3585 -> 18944:
// 46 us a call, 71 with loads of a byte; 21 where K is 3584.)
__global__ __launch_bounds__(256) void pad_codes_kernel(const int8_t* __restrict__ from, int64_t k, int64_t kp, int8_t* __restrict__ to)
{
    struct __attribute__((packed, aligned(1))) Anywhere {
        uint32_t d[4];
    };
    const int64_t row = blockIdx.y;
    const int64_t i = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) * 16;
    if (i >= kp) return;
    const int8_t* const x = from + row * k + i;
    uint32_t d[4] = {0, 0, 0, 0};
    if (i + 16 <= k) {
        const Anywhere a = *reinterpret_cast<const Anywhere*>(x);
#pragma unroll
        for (int e = 0; e < 4; ++e) d[e] = a.d[e];
    } else {
#pragma unroll
        for (int e = 0; e < 16; ++e)
            if (i + e < k) d[e >> 2] |= static_cast<uint32_t>(static_cast<uint8_t>(x[e])) << (8 * (e & 3));
    }
    *reinterpret_cast<uint4*>(to + row * kp + i) = make_uint4(d[0], d[1], d[2], d[3]);
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
    int columns;               // of a workgroup: few rows
    int b_scale_dtype, bias_dtype, y_dtype;
};

__device__ __forceinline__ void store_scaled(const Int8Params& p, int64_t row, int64_t col, int32_t sum, float a_scale, float b_scale)
{
    const float v = static_cast<float>(sum) * a_scale * b_scale;
    store_from_f32(p.y, p.y_dtype, row * p.n + col, with_bias(v, p.bias, p.bias_dtype, row, p.n, col, p.y_dtype));
}

// Few rows: a workgroup has up to 16 CT columns, its waves split K; B's bytes bound it. v_mfma_i32_16x16x64_i8: lane l holds 16 bytes of k of row (or column) l % 16, k
// from (l / 16) * 16. RT: tiles of 16 rows; lanes whose row is not there load no codes (a CU's vector memory path is 64 bytes a cycle, and 16 rows are as many
// bytes as 16 columns). Two steps' loads are in flight.
// FUSED (up to three rows of at most 32 KiB of codes): a is [m, k] of type T, and every workgroup makes the codes for itself, in LDS, while its first weights are on
// their way: a launch of its own takes longer than a row's second and third trip from L2.
// Measured: one row of 4096 -> 6144 with the quantizer inside 8.2 us, three sets of operands in turn (25 MB: 3.1 TB/s, an empty launch is 2 of them); the same operands
// each time, which the last-level cache then holds, 8 rows of 4096 -> 28672 23.5 us (5.0 TB/s), 24 rows of 4096 -> 12288 13.7 us (3.7 TB/s).
template <int RT, int CT, typename T, bool BF16, bool FUSED>
__global__ __launch_bounds__(512) void int8_rows_kernel(const int8_t* b_base, const void* a_base, int m, int n, int k, int steps, Int8Params p)
{
    __shared__ int32_t sums[8][RT * CT * 4][64];
    extern __shared__ __attribute__((aligned(16))) uint8_t coded[];                     // FUSED: rows of kp codes
    __shared__ float row_scale[4];
    __shared__ uint32_t slots[16];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c = lane & 15, g = lane >> 4, kp = steps * 128;
    const int64_t n0 = static_cast<int64_t>(blockIdx.x) * p.columns;
    const int cols = static_cast<int>(n - n0 < p.columns ? n - n0 : p.columns);
    const auto srd_b = make_srd(b_base + n0 * p.ldb, static_cast<uint64_t>(cols * p.ldb));
    const auto srd_a = make_srd(a_base, FUSED ? 0 : static_cast<uint64_t>(m) * p.lda);
    const int begin = steps * wave >> 3, end = steps * (wave + 1) >> 3;                // (eight waves)
    uint32_t b_at[CT], a_at[RT];
    i32x4_t acc[RT][CT] = {};
#pragma unroll
    for (int j = 0; j < CT; ++j) b_at[j] = j * 16 + c < cols ? static_cast<uint32_t>((j * 16 + c) * p.ldb + g * 16) : kOutOfRange;
#pragma unroll
    for (int r = 0; r < RT; ++r) a_at[r] = r * 16 + c < m ? static_cast<uint32_t>((r * 16 + c) * p.lda + g * 16) : kOutOfRange;
    struct Step {
        uint4 b[CT][2], a[FUSED ? 1 : RT][2];
    };
    auto load = [&](int t, Step& s) {
        // (behind the wave's last step nothing is read, but asked for all the same: a branch would have every load waited for)
        const uint32_t at = t < end ? static_cast<uint32_t>(t) * 128u : 0u, off = t < end ? 0u : kOutOfRange;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int j = 0; j < CT; ++j) s.b[j][h] = load16(srd_b, off ? off : b_at[j] + at + h * 64, 0);
            if constexpr (!FUSED)
#pragma unroll
                for (int r = 0; r < RT; ++r) s.a[r][h] = load16(srd_a, off ? off : a_at[r] + at + h * 64, 0);
        }
    };
    auto multiply = [&](int t, const Step& s) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            i32x4_t fused = {};
            if constexpr (FUSED) {
                if (c < m) fused = *reinterpret_cast<const i32x4_t*>(coded + c * kp + t * 128 + h * 64 + g * 16);
            }
#pragma unroll
            for (int r = 0; r < RT; ++r)
#pragma unroll
                for (int j = 0; j < CT; ++j)
                    acc[r][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(FUSED ? fused : __builtin_bit_cast(i32x4_t, s.a[FUSED ? 0 : r][h]), __builtin_bit_cast(i32x4_t, s.b[j][h]), acc[r][j], 0, 0, 0);
        }
    };
    Step one, two;
    load(begin, one);
    load(begin + 1, two);
    if constexpr (FUSED) {
        using V8 = Eight<T, BF16>;
        const int pieces = kp / 8;
        constexpr int kHeld = 2;                                                       // pieces a thread holds between the two passes
        for (int t = 0; t < m; ++t) {
            const T* const x = static_cast<const T*>(a_base) + static_cast<int64_t>(t) * k;
            auto piece = [&](int i, V8& e) {
                const int left = k - i * 8;
                if (left >= 8) e.load(x + i * 8);
                else if (left > 0) e.load_first(x + i * 8, left);
                else e.zero();
            };
            V8 held[kHeld];
            uint32_t amax = 0;
            auto look = [&](const V8& e) {
                float v[8];
                e.get(v);
#pragma unroll
                for (int q = 0; q < 8; ++q) amax = larger(amax, __float_as_uint(v[q]) & 0x7fffffffu);
            };
#pragma unroll
            for (int j = 0; j < kHeld; ++j) {
                const int i = threadIdx.x + j * 512;
                if (i < pieces) piece(i, held[j]);
                else held[j].zero();
            }
#pragma unroll
            for (int j = 0; j < kHeld; ++j) look(held[j]);
            for (int i = threadIdx.x + kHeld * 512; i < pieces; i += 512) {
                V8 e;
                piece(i, e);
                look(e);
            }
            __syncthreads();                                                           // (the slots of the row before are read)
            const RowScale scale(over_workgroup(amax, slots, wave, 8, larger));
            if (threadIdx.x == 0) row_scale[t] = scale.scale;
            auto code = [&](int i, const V8& e) {
                float v[8];
                e.get(v);
                uint32_t d[2] = {0, 0};
#pragma unroll
                for (int q = 0; q < 8; ++q) d[q >> 2] |= static_cast<uint32_t>(scale.code(v[q]) & 0xff) << (8 * (q & 3));
                *reinterpret_cast<uint2*>(coded + t * kp + i * 8) = make_uint2(d[0], d[1]);
            };
#pragma unroll
            for (int j = 0; j < kHeld; ++j)
                if (static_cast<int>(threadIdx.x) + j * 512 < pieces) code(threadIdx.x + j * 512, held[j]);
            for (int i = threadIdx.x + kHeld * 512; i < pieces; i += 512) {
                V8 e;
                piece(i, e);
                code(i, e);
            }
        }
        __syncthreads();
    }
    for (int t = begin; t < end; t += 2) {
        multiply(t, one);
        load(t + 2, one);
        if (t + 1 < end) multiply(t + 1, two);
        load(t + 3, two);
    }
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int j = 0; j < CT; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) sums[wave][(r * CT + j) * 4 + i][lane] = acc[r][j][i];
    __syncthreads();
    for (int q = wave; q < RT * CT * 4; q += 8) {
        const int tile = q >> 2, r = tile / CT, j = tile % CT;
        const int64_t row = r * 16 + g * 4 + (q & 3), col = n0 + j * 16 + c;
        if (row >= m || j * 16 + c >= cols) continue;
        int32_t sum = 0;
#pragma unroll
        for (int w = 0; w < 8; ++w) sum += sums[w][q][lane];
        store_scaled(p, row, col, sum, FUSED ? row_scale[row] : p.a_scale[row], load_as_f32(p.b_scale, p.b_scale_dtype, col));
    }
}

// Tall calls: tiles of 64 W x 64 W, four waves of 32 W x 32 W each on v_mfma_i32_32x32x32_i8, BK bytes of K a step, both operands from memory straight into LDS.
//
// A step's pieces of 16 bytes lie in LDS in the order in which the loads leave them (a wave's 64 lanes side by side), rows of BK bytes; which piece of its row a lane
// asks for is turned round by its row, so that the 32 rows of an operand read meet each bank as often as it takes and no more.
// Four steps are in LDS or on their way. One barrier a step: before the step's last products the next step has arrived, its first operands are read while those
// products run, and the loads of the step four on go where this step's operands were, which all are in registers by then.
// W = 4 (256 x 256): 256 accumulators a lane, one wave a SIMD; a piece read from LDS meets four others. W = 2 (128 x 128): two workgroups a CU, for grids that would
// not cover the chip; with slices of K, which make one workgroup a CU, BK = 128 instead of 64, whole lines (500 rows of 18944 -> 3584: 50 us instead of 59).
// Measured: 8192 rows of 4096 -> 14336 520-540 us (1.8 POP/s; a product of twice the K reaches 2.0, so that some 130 us are the first loads and the last stores of
// seven rounds of tiles, one workgroup a CU), 500 rows of 18944 -> 3584 in two slices 50 us and 7.5 for their sum (1.2 POP/s).
template <int W, int BK>
struct Int8Tile {
    static constexpr int kStages = 4;
    static constexpr int kRows = 64 * W, kPieces = BK / 16, kStage = 2 * kRows * BK;     // bytes of a step: A, then B
    static constexpr int kLoads = kStage / 1024 / 4;                                     // of a wave
    static constexpr int kRowsPerLoad = 1024 / BK, kSteps = BK / 32;

    static __device__ __forceinline__ int turned(int row, int piece)
    {
        if constexpr (kPieces == 8) return piece ^ (row & 7);
        return piece ^ (row >> 1 & 3);
    }
};

typedef __attribute__((ext_vector_type(4))) uint32_t srd_t;
__device__ __forceinline__ srd_t plain_srd(const void* base, uint32_t bytes)
{
    const uint64_t at = reinterpret_cast<uint64_t>(base);
    srd_t s;
    s.x = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(at));
    s.y = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(at >> 32));
    s.z = __builtin_amdgcn_readfirstlane(bytes);
    s.w = 0x00020000u;
    return s;
}

template <int W, int BK, bool SLICED>
__global__ __launch_bounds__(256, W == 4 ? 1 : 2) void int8_tile_kernel(Int8Params p, unsigned tiles_m, unsigned tiles_n, unsigned slices)
{
    using Tile = Int8Tile<W, BK>;
    constexpr int kWave = 32 * W, kStage = Tile::kStage, kSteps = Tile::kSteps;
    extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];           // four steps
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = lane & 31, g = lane >> 5;

    // Workgroups go round the eight XCDs; each takes a run of one slice's tiles, eight row blocks by all columns at a time, so that its L2 sees an operand more than once.
    const unsigned of_slice = tiles_m * tiles_n, all = SLICED ? of_slice * slices : of_slice, per = (all + 7) / 8, linear = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
    if ((blockIdx.x >> 3) >= per || linear >= all) return;
    const unsigned slice = SLICED ? linear / of_slice : 0, tile = linear - slice * of_slice;
    const unsigned band = tile / (8 * tiles_n), in_band = tile - band * 8 * tiles_n, rows_here = min(8u, tiles_m - band * 8);
    const int64_t m0 = static_cast<int64_t>(band * 8 + in_band % rows_here) * Tile::kRows, n0 = static_cast<int64_t>(in_band / rows_here) * Tile::kRows;
    const int rows = static_cast<int>(p.m - m0 < Tile::kRows ? p.m - m0 : Tile::kRows), cols = static_cast<int>(p.n - n0 < Tile::kRows ? p.n - n0 : Tile::kRows);
    const int total = p.steps * (128 / BK), share = p.steps_per_slice * (128 / BK);
    const int begin = static_cast<int>(slice) * share, end = min(begin + share, total), count = end - begin;

    // Load i of a wave brings kRowsPerLoad rows; rows that are not there repeat the last. The range ends with the operand's last row, and moves on with K.
    uint32_t at[Tile::kLoads];
#pragma unroll
    for (int i = 0; i < Tile::kLoads; ++i) {
        const bool of_b = i >= Tile::kLoads / 2;
        const int row = (wave * (Tile::kLoads / 2) + i % (Tile::kLoads / 2)) * Tile::kRowsPerLoad + lane / Tile::kPieces;
        const int from = min(row, (of_b ? cols : rows) - 1);
        at[i] = static_cast<uint32_t>(from * static_cast<int>(of_b ? p.ldb : p.lda) + Tile::turned(row, lane % Tile::kPieces) * 16);
    }
    const int8_t* const a = p.a + m0 * p.lda;
    const int8_t* const b = p.b + n0 * p.ldb;
    const uint32_t a_bytes = static_cast<uint32_t>(rows * p.lda), b_bytes = static_cast<uint32_t>(cols * p.ldb);
    const uint32_t lds = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)smem;
    auto fetch = [&](int t) {                                    // step `begin + t` into its quarter of LDS
        const uint32_t k = static_cast<uint32_t>(begin + t) * BK, to = lds + (t & 3) * kStage + wave * (kStage / 8);
        // (behind the slice's last step: nothing, into a quarter that nobody reads any more)
        const bool is = t < count;
        // The compiler puts no wait states in front of what stands in an asm block. A load needs five behind a vector instruction that wrote one of its scalar registers:
        // the ranges' ends are differences cut off at zero as signed numbers, which scalar instructions make (unsigned, a vector one did), and the assembly is tested for it.
        // (s_nop 4 here instead: 8192 rows 1 % slower, 24 rows 4 %.) A load into LDS needs one behind the write of M0, a reserved register that the compiler keeps nothing in.
        const srd_t sa = plain_srd(a + k, is ? a_bytes - k : 0u), sb = plain_srd(b + k, is ? static_cast<uint32_t>(max(static_cast<int>(b_bytes) - static_cast<int>(k), 0)) : 0u);
#pragma unroll
        for (int i = 0; i < Tile::kLoads; ++i) {
            const bool of_b = i >= Tile::kLoads / 2;
            const uint32_t dst = __builtin_amdgcn_readfirstlane(to + (of_b ? kStage / 2 : 0) + i % (Tile::kLoads / 2) * 1024);
            asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(dst), "v"(at[i]), "s"(of_b ? sb : sa) : "memory");
        }
    };
    const int wm = (wave & 1) * kWave, wn = (wave >> 1) * kWave;
    i32x4_t fa[2][W], fb[2][W];
    auto operands = [&](int t, int s, i32x4_t (&xa)[W], i32x4_t (&xb)[W]) {
        const uint8_t* const half = smem + (t & 3) * kStage;
#pragma unroll
        for (int i = 0; i < W; ++i) {
            const int ra = wm + i * 32 + c, rb = wn + i * 32 + c;
            xa[i] = *reinterpret_cast<const i32x4_t*>(half + ra * BK + Tile::turned(ra, s * 2 + g) * 16);
            xb[i] = *reinterpret_cast<const i32x4_t*>(half + kStage / 2 + rb * BK + Tile::turned(rb, s * 2 + g) * 16);
        }
    };
    i32x16_t acc[W][W] = {};
    auto products = [&](const i32x4_t (&xa)[W], const i32x4_t (&xb)[W], int first, int last) {
#pragma unroll
        for (int i = 0; i < W; ++i)
            if (i >= first && i < last)
#pragma unroll
                for (int j = 0; j < W; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(xa[i], xb[j], acc[i][j], 0, 0, 0);
    };
    // A read of an operand after each product while there are any. (The compiler would put them where they are used, and wait.)
    auto interleave = [&] {
#pragma unroll
        for (int i = 0; i < 2 * W; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        }
    };
    // own loads but those of the steps behind the next are in, own reads done, and everyone's
    auto arrived = [&] {
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(2 * Tile::kLoads) : "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    fetch(0);                                                    // (no slice is empty)
    fetch(1);
    fetch(2);
    arrived();
    operands(0, 0, fa[0], fb[0]);
    fetch(3);
    for (int t = 0; t < count; ++t) {
#pragma unroll
        for (int s = 0; s < kSteps - 1; ++s) {
            operands(t, s + 1, fa[(s + 1) & 1], fb[(s + 1) & 1]);
            products(fa[s & 1], fb[s & 1], 0, W);
            interleave();
            __builtin_amdgcn_sched_barrier(0);
        }
        arrived();
        operands(t + 1, 0, fa[0], fb[0]);                        // (behind the last step: whatever lies there, for no product)
        products(fa[1], fb[1], 0, W / 2);
        __builtin_amdgcn_sched_barrier(0);
        fetch(t + 4);
        __builtin_amdgcn_sched_barrier(0);
        products(fa[1], fb[1], W / 2, W);
        __builtin_amdgcn_sched_barrier(0);
    }

    // A lane has column c and rows 8 (e / 4) + 4 g + e % 4 of each 32 x 32; 32 rows of all of the wave's columns are turned round in the wave's own piece of LDS, and
    // a lane leaves with eight columns, the same ones in all of its rows: whole lines of y. (One form takes the accumulators out, whatever becomes of them: with one
    // for each kind of result the compiler moves all 256 at once, and spills.)
    constexpr int kTurn = kWave + 8, kAcross = kWave / 8, kDown = 64 / kAcross;          // dwords from a row to the next; lanes to a row, rows of a wave
    static_assert(32 % kDown == 0 && 4 * (4 * 32 * kTurn) <= 4 * kStage);
    const int64_t first = n0 + wn + lane % kAcross * 8;
    const int64_t left = p.n - first;                            // columns from here on
    const int mine = lane / kAcross;
    float sb[8] = {}, bias[8] = {};
    bool wide = false;                                           // whole eights go out at once
    if constexpr (SLICED) {
        wide = (p.n & 3) == 0 && left >= 8;
    } else {
        const bool row_bias = p.bias && (p.bias_dtype & ROCM_BIAS_PER_ROW);
        wide = !row_bias && left >= 8 && (p.n & (p.y_dtype == ROCM_DT_F32 ? 3 : 7)) == 0 && (reinterpret_cast<uintptr_t>(p.y) & 15) == 0;
#pragma unroll
        for (int q = 0; q < 8; ++q) {
            const int64_t col = q < left ? first + q : p.n - 1;
            sb[q] = load_as_f32(p.b_scale, p.b_scale_dtype, col);
            if (p.bias && !row_bias) bias[q] = load_as_f32(p.bias, p.bias_dtype, col);
        }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");             // (what was fetched behind the end has to be in before LDS is used for something else)
    __syncthreads();
    int32_t* const turn = reinterpret_cast<int32_t*>(smem) + wave * (32 * kTurn);
#pragma unroll
    for (int i = 0; i < W; ++i) {
#pragma unroll
        for (int j = 0; j < W; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) turn[((e >> 2) * 8 + g * 4 + (e & 3)) * kTurn + j * 32 + c] = acc[i][j][e];
        lds_order();
#pragma unroll 2
        for (int d = 0; d < 32; d += kDown) {
            const int64_t row = m0 + wm + i * 32 + d + mine;
            if (row >= p.m || left <= 0) continue;
            const int32_t* const from = turn + (d + mine) * kTurn + lane % kAcross * 8;
            const int4 lo = *reinterpret_cast<const int4*>(from), hi = *reinterpret_cast<const int4*>(from + 4);
            if constexpr (SLICED) {
                int32_t* const part = p.partial + (static_cast<int64_t>(slice) * p.m + row) * p.n + first;
                if (wide) {
                    reinterpret_cast<int4*>(part)[0] = lo;
                    reinterpret_cast<int4*>(part)[1] = hi;
                } else {
#pragma unroll 1
                    for (int q = 0; q < 8 && q < left; ++q) part[q] = from[q];
                }
            } else {
                const float sa = p.a_scale[row];
                if (!wide) {
#pragma unroll 1
                    for (int q = 0; q < 8 && q < left; ++q) store_scaled(p, row, first + q, from[q], sa, load_as_f32(p.b_scale, p.b_scale_dtype, first + q));
                    continue;
                }
                const int32_t sum[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
                float v[8];
#pragma unroll
                for (int q = 0; q < 8; ++q) v[q] = static_cast<float>(sum[q]) * sa * sb[q] + bias[q];
                const int64_t at = row * p.n + first;
                if (p.y_dtype == ROCM_DT_F32) {
                    float4* const y = reinterpret_cast<float4*>(static_cast<float*>(p.y) + at);
                    y[0] = make_float4(v[0], v[1], v[2], v[3]);
                    y[1] = make_float4(v[4], v[5], v[6], v[7]);
                } else {
                    uint4* const y = reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.y) + at);
                    Eight<uint16_t, true> wide_range;
                    Eight<uint16_t, false> half;
                    if (p.y_dtype == ROCM_DT_BF16) {
                        wide_range.set(v);
                        *y = make_uint4(wide_range.raw.x, wide_range.raw.y, wide_range.raw.z, wide_range.raw.w);
                    } else {
                        half.set(v);
                        *y = make_uint4(half.raw.x, half.raw.y, half.raw.z, half.raw.w);
                    }
                }
            }
        }
        lds_order();
    }
}

// y from the sums of slices of K: four columns a thread where rows of n begin at a multiple of four.
template <int FOUR>
__global__ __launch_bounds__(256) void int8_reduce_kernel(Int8Params p, int slices)
{
    const int64_t row = static_cast<int64_t>(blockIdx.z) * gridDim.y + blockIdx.y, col = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) * FOUR;
    if (row >= p.m || col >= p.n) return;
    int32_t sum[FOUR] = {};
    for (int i = 0; i < slices; ++i) {
        const int32_t* const from = p.partial + (i * p.m + row) * p.n + col;
        if constexpr (FOUR == 4) {
            const int4 v = *reinterpret_cast<const int4*>(from);
            sum[0] += v.x, sum[1] += v.y, sum[2] += v.z, sum[3] += v.w;
        } else {
            sum[0] += *from;
        }
    }
#pragma unroll
    for (int q = 0; q < FOUR; ++q) store_scaled(p, row, col + q, sum[q], p.a_scale[row], load_as_f32(p.b_scale, p.b_scale_dtype, col + q));
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
    auto go = [&](auto kernel, unsigned threads, auto* x) {
        constexpr int64_t kMost = 1 << 21;                   // rows of a launch: a grid has fewer than 2^32 threads
        for (int64_t r = 0; r < m; r += kMost) {
            hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(m - r < kMost ? m - r : kMost)), dim3(threads), 0, s, x + r * k, k, kp, codes + r * kp, scales + r);
            const hipError_t e = hipGetLastError();
            if (e != hipSuccess) return static_cast<int>(e);
        }
        return 0;
    };
    // (rows of 4096 by 4 waves 39 us of a call, by 16 waves 55; of 18944, 500 rows, 29 and 26)
    auto held = [&](auto four_waves, auto sixteen_waves, auto* x) { return kp <= 8192 ? go(four_waves, 256u, x) : go(sixteen_waves, 1024u, x); };
    if (dtype == ROCM_DT_F32) return held(quantize_rows_kernel<float, false, 4, 4>, quantize_rows_kernel<float, false, 16, 3>, static_cast<const float*>(a));
    if (dtype == ROCM_DT_BF16) return held(quantize_rows_kernel<uint16_t, true, 4, 4>, quantize_rows_kernel<uint16_t, true, 16, 3>, static_cast<const uint16_t*>(a));
    return held(quantize_rows_kernel<uint16_t, false, 4, 4>, quantize_rows_kernel<uint16_t, false, 16, 3>, static_cast<const uint16_t*>(a));
}

extern "C" int rocm_launch_pad_codes(const int8_t* from, int64_t rows, int64_t k, int8_t* to, rocm_stream_t stream)
{
    using namespace mnb;
    const int64_t kp = (k + 127) / 128 * 128;
    for (int64_t r = 0; r < rows; r += 65535) {
        const unsigned part = static_cast<unsigned>(rows - r < 65535 ? rows - r : 65535);
        hipLaunchKernelGGL(pad_codes_kernel, dim3(static_cast<unsigned>((kp / 16 + 255) / 256), part), dim3(256), 0, static_cast<hipStream_t>(stream), from + r * k, k, kp, to + r * kp);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return static_cast<int>(e);
    }
    return 0;
}

namespace mnb {
namespace {

// Rows up to which a call streams B, and up to which it does if B is small: 24 rows of 4096 -> 8192 take 10.7 us so and 15.3 in tiles with a sum over slices,
// 24 rows of 18944 -> 3584 (65 MiB) 25 and 19, 60 rows of 4096 -> 14336 (56 MiB) 31 and 19.
constexpr int64_t kFewRows = 16, kSomeRows = 32, kSmallBytes = 52 << 20;

// What a call is launched as.
struct Int8Plan {
    int tile;                   // 0: rows
    int slices;
};
Int8Plan plan_of(const RocmInt8Args& a)
{
    Int8Plan p{0, 1};
    if (a.m <= kFewRows || (a.m <= kSomeRows && a.n * ((a.k + 127) / 128 * 128) <= kSmallBytes)) return p;
    auto tiles = [&](int64_t t) { return (a.m + t - 1) / t * ((a.n + t - 1) / t); };
    const int64_t cus = rocm_ffi_compute_units(), steps = (a.k + 127) / 128;
    // 256 x 256 from tiles for three quarters of the CUs on. K 4096, us in tiles of 256 and of 128: 1024 x 8192 (128 tiles of 256) 65 and 48, 1024 x 10240 (160) 67 and
    // 66, 1500 x 8192 (192) 69 and 74, 1024 x 14336 (224) 74 and 92.
    p.tile = tiles(256) >= cus * 3 / 4 ? 256 : 128;
    if (p.tile == 128) {
        // Slices of K until a workgroup for each CU is there, none of less than 16 steps. 500 rows of 18944 -> 3584 (112 tiles): 80 us without, 54 with two, 59 with four,
        // 64 with six; 100 rows of them (28 tiles): 76 without, 23 with nine or sixteen.
        int64_t s = cus / tiles(128);
        if (s > steps / 16) s = steps / 16;
        s = s < 1 ? 1 : s > 16 ? 16 : s;
        const int64_t share = (steps + s - 1) / s;
        p.slices = static_cast<int>((steps + share - 1) / share);
    }
    return p;
}
// Whether the product quantizes its rows itself. us of a call among others on the same operands (in the last-level cache: less than the kernel takes on others), with
// and without, 4096 -> 6144: 1 row 6.7 and 8.9, 2 7.7 and 9.2, 3 8.5 and 9.3, 4 9.5 and 9.4; 4096 -> 14336: 1 row 11.8
// and 15.0, 3 15.3 and 15.1, 4 17.0 and 15.8.
bool fuses(const RocmInt8Args& a) { return a.m <= 3 && (a.a_dtype == ROCM_DT_F16 || a.a_dtype == ROCM_DT_BF16) && a.m * ((a.k + 127) / 128 * 128) <= 32768; }

}  // namespace
}  // namespace mnb

extern "C" int rocm_int8_pads_b(const RocmInt8Args* args) { return args->k % 16 != 0; }
extern "C" uint64_t rocm_int8_scratch_bytes(const RocmInt8Args* args)
{
    const mnb::Int8Plan p = mnb::plan_of(*args);
    return p.slices > 1 ? static_cast<uint64_t>(p.slices) * args->m * args->n * 4 : 0;
}
extern "C" int rocm_int8_fuses_quantizer(const RocmInt8Args* args) { return mnb::fuses(*args); }
extern "C" const char* rocm_int8_variant(const RocmInt8Args* args)
{
    const mnb::Int8Plan p = mnb::plan_of(*args);
    if (p.tile == 0) return args->a_float ? "int8_rows_fused" : "int8_rows";
    return p.tile == 256 ? "int8_tile_256" : p.slices > 1 ? "int8_tile_128_sliced" : "int8_tile_128";
}

extern "C" int rocm_launch_int8(const RocmInt8Args* args, rocm_stream_t stream)
{
    using namespace mnb;
    if (args->m <= 0 || args->n <= 0) return 0;
    hipStream_t s = static_cast<hipStream_t>(stream);
    Int8Params p = params_of(args);
    const Int8Plan plan = plan_of(*args);
    if (plan.tile == 0) {
        // As many columns a workgroup, up to 48, as make the grid one, two ... times the CUs: tiles of whole 16s left 5 us of 24 to the few that came last
        // (24 rows of 3584 -> 18944), and more workgroups read the rows more often (24 rows of 4096 -> 8192: 13.4 us with 16 columns each, 10.7 with 32).
        const int64_t cus = rocm_ffi_compute_units(), most = 48;
        int64_t times = (p.n + cus * most - 1) / (cus * most);
        p.columns = static_cast<int>((p.n + cus * times - 1) / (cus * times));
        if (p.columns < 16) p.columns = 16;
        const unsigned grid = static_cast<unsigned>((p.n + p.columns - 1) / p.columns);
        auto go = [&](auto kernel, const void* a, size_t lds) {
            hipLaunchKernelGGL(kernel, dim3(grid), dim3(512), lds, s, p.b, a, static_cast<int>(p.m), static_cast<int>(p.n), static_cast<int>(args->k), p.steps, p);
            return static_cast<int>(hipGetLastError());
        };
        auto columns = [&](auto one, auto two, auto three, const void* a, size_t lds) { return p.columns <= 16 ? go(one, a, lds) : p.columns <= 32 ? go(two, a, lds) : go(three, a, lds); };
        if (args->a_float) {
            if (!fuses(*args)) return static_cast<int>(hipErrorInvalidValue);
            const size_t lds = static_cast<size_t>(p.m) * p.steps * 128;
            if (args->a_dtype == ROCM_DT_BF16)
                return columns(int8_rows_kernel<1, 1, uint16_t, true, true>, int8_rows_kernel<1, 2, uint16_t, true, true>, int8_rows_kernel<1, 3, uint16_t, true, true>, args->a_float, lds);
            return columns(int8_rows_kernel<1, 1, uint16_t, false, true>, int8_rows_kernel<1, 2, uint16_t, false, true>, int8_rows_kernel<1, 3, uint16_t, false, true>, args->a_float, lds);
        }
        if (p.m <= 16) return columns(int8_rows_kernel<1, 1, float, false, false>, int8_rows_kernel<1, 2, float, false, false>, int8_rows_kernel<1, 3, float, false, false>, p.a, 0);
        return columns(int8_rows_kernel<2, 1, float, false, false>, int8_rows_kernel<2, 2, float, false, false>, int8_rows_kernel<2, 3, float, false, false>, p.a, 0);
    }
    p.steps_per_slice = (p.steps + plan.slices - 1) / plan.slices;
    p.partial = plan.slices > 1 ? args->partial : nullptr;
    const unsigned tm = static_cast<unsigned>((p.m + plan.tile - 1) / plan.tile), tn = static_cast<unsigned>((p.n + plan.tile - 1) / plan.tile);
    const unsigned slices = static_cast<unsigned>(plan.slices);
    const dim3 grid((tm * tn * slices + 7) / 8 * 8);
    auto tiled = [&](auto kernel, size_t lds) {
        if (lds > 65536) {           // more than a kernel gets without asking
            const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(lds));
            if (e != hipSuccess) return e;
        }
        hipLaunchKernelGGL(kernel, grid, dim3(256), lds, s, p, tm, tn, slices);
        return hipGetLastError();
    };
    constexpr size_t kLds256 = 4 * Int8Tile<4, 64>::kStage, kLds128 = 4 * Int8Tile<2, 64>::kStage, kLdsSlices = 4 * Int8Tile<2, 128>::kStage;
    hipError_t e = plan.tile == 256 ? tiled(int8_tile_kernel<4, 64, false>, kLds256)
                   : p.partial      ? tiled(int8_tile_kernel<2, 128, true>, kLdsSlices)
                                    : tiled(int8_tile_kernel<2, 64, false>, kLds128);
    if (e == hipSuccess && p.partial) {
        const unsigned y = static_cast<unsigned>(p.m < 32768 ? p.m : 32768);
        const bool four = p.n % 4 == 0;
        const int64_t across = four ? p.n / 4 : p.n;
        hipLaunchKernelGGL(four ? int8_reduce_kernel<4> : int8_reduce_kernel<1>, dim3(static_cast<unsigned>((across + 255) / 256), y, static_cast<unsigned>((p.m + y - 1) / y)), dim3(256), 0, s, p, plan.slices);
        e = hipGetLastError();
    }
    return static_cast<int>(e);
}
