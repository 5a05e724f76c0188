// QMoE for up to four tokens, in two launches, each weight read once.
//
//   moe_few_up_kernel     every workgroup routes the tokens for itself; h = act(x Wg^T + bg, x Wu^T + bu) of one expert's columns for the rows that chose it
//   moe_few_down_kernel   y = base + sum over the active experts of weight * (h W2^T + bias)
//
// The weights' bytes bound it once there are enough of them, and before that the way to them: arguments, logits and weights are reached one after the other.
// A lane holds 32 elements of K of a row of x in registers, in 16 dot products of two with 32 nibbles of each of several columns (v_dot2_f32_f16, v_dot2_f32_bf16:
// 46 instructions for 16 bytes of weights and one row; the matrix core wants the nibbles turned between lanes and takes 71 with its corrections, for up to 16 rows).
// A nibble q is the 16-bit float magic + q (moe_dot.hiph), and the products' sum starts from -(magic + zp) times the lane's sum of x.
// LPC lanes stand side by side on K and read 16 LPC bytes of a column's row as the caller holds it; 64 / LPC columns are read at once.
#include "moe_dot.hiph"
#include "moe_route.hiph"

namespace mnb {
namespace {

typedef __attribute__((ext_vector_type(2))) _Float16 moe_half2_t;
typedef __attribute__((ext_vector_type(2))) __bf16 moe_bf16x2_t;

template <bool BF16>
__device__ __forceinline__ float dot2(uint32_t a, uint32_t b, float c)
{
    if constexpr (BF16) return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(moe_bf16x2_t, a), __builtin_bit_cast(moe_bf16x2_t, b), c, false);
    else return __builtin_amdgcn_fdot2(__builtin_bit_cast(moe_half2_t, a), __builtin_bit_cast(moe_half2_t, b), c, false);
}

// 32 elements of a row in the order of a dword's nibbles under a mask and shifts: 0 4 | 1 5 | 2 6 | 3 7 of each eight; and their sum.
template <bool BF16>
struct Elements32 {
    uint32_t v[16];
    float sum;

    // `count` of them are there (a multiple of 8), the rest is zero
    __device__ __forceinline__ void load(const uint16_t* x, int count)
    {
        constexpr uint32_t kOnes = BF16 ? 0x3f803f80u : 0x3c003c00u;
        sum = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            uint4 d = make_uint4(0, 0, 0, 0);
            if (j * 8 < count) d = *reinterpret_cast<const uint4*>(x + j * 8);
            v[4 * j] = __builtin_amdgcn_perm(d.z, d.x, 0x05040100u);           // 0 | 4
            v[4 * j + 1] = __builtin_amdgcn_perm(d.z, d.x, 0x07060302u);       // 1 | 5
            v[4 * j + 2] = __builtin_amdgcn_perm(d.w, d.y, 0x05040100u);
            v[4 * j + 3] = __builtin_amdgcn_perm(d.w, d.y, 0x07060302u);
#pragma unroll
            for (int i = 0; i < 4; ++i) sum = dot2<BF16>(v[4 * j + i], kOnes, sum);
        }
    }
};

template <bool BF16>
__device__ __forceinline__ void nibbles32(const uint4& w, uint32_t (&out)[16])
{
    constexpr uint32_t kMagic = BF16 ? 0x43004300u : 0x64006400u;
    uint32_t d[4] = {w.x, w.y, w.z, w.w};
    // unpacked for each row anew: kept for the next row, the nibbles of a wave's columns take 128 registers
    asm volatile("" : "+v"(d[0]), "+v"(d[1]), "+v"(d[2]), "+v"(d[3]));
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) out[4 * j + i] = ((d[j] >> (4 * i)) & 0x000f000fu) | kMagic;
}

// start + sum a (magic + q), in four chains
template <bool BF16>
__device__ __forceinline__ float dot32(const uint32_t (&a)[16], const uint32_t (&b)[16], float start)
{
    float s[4] = {start, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i & 3] = dot2<BF16>(a[i], b[i], s[i & 3]);
    return (s[0] + s[1]) + (s[2] + s[3]);
}

// The weights of NU times 64 / LPC columns: load u has column n0 + u (64 / LPC) + lane / LPC, bytes 16 (lane % LPC) on from a pass's begin.
template <typename ST, bool ZP, int NU, int LPC>
struct FewColumns {
    uint4 w[NU];
    typename ScaleIo<ST>::raw_t s[NU];
    uint8_t z[NU];

    __device__ __forceinline__ void load(const MoeMatrix& m, const MoeTile<1>& t, int live, int k, int kl)
    {
        const int group = (threadIdx.x & 63) / LPC;
        const uint32_t block = static_cast<uint32_t>(min(k / m.block_size, m.kb - 1));
#pragma unroll
        for (int u = 0; u < NU; ++u) {
            const int col = u * (64 / LPC) + group;
            const uint32_t row = static_cast<uint32_t>(col) * static_cast<uint32_t>(m.row_step);
            const bool is = col < live && kl >= 0;
            w[u] = load16(t.w[0], is ? row * static_cast<uint32_t>(m.row_bytes) + static_cast<uint32_t>(k) / 2 : kOutOfRange, 0);
            s[u] = ScaleIo<ST>::load_raw(t.s[0], is ? (row * static_cast<uint32_t>(m.kb) + block) * static_cast<uint32_t>(sizeof(ST)) : kOutOfRange, 0);
            if constexpr (ZP) z[u] = __builtin_amdgcn_raw_buffer_load_b8(t.z[0], static_cast<int>(is ? row * static_cast<uint32_t>(m.zp_row) + block / 2 : kOutOfRange), 0, 0);
        }
    }
};

// acc[u] += factor * scale * sum a (q - zp) for NH parts of a row
template <bool BF16, typename ST, bool ZP, int NU, int LPC, int NH>
__device__ __forceinline__ void few_multiply(const FewColumns<ST, ZP, NU, LPC>& c, const Elements32<BF16> (&a)[NH], int odd, float factor, float (&acc)[NU])
{
    constexpr float kMagic = BF16 ? 128.f : 1024.f;
    float sum = a[0].sum;
    if constexpr (NH == 2) sum += a[1].sum;
    const float plain = -(kMagic + 8.f) * sum;
#pragma unroll
    for (int u = 0; u < NU; ++u) {
        uint32_t q[16];
        nibbles32<BF16>(c.w[u], q);
        float start = plain;
        if constexpr (ZP) start = (-kMagic - static_cast<float>(odd ? c.z[u] >> 4 : c.z[u] & 15)) * sum;
        float d = dot32<BF16>(a[0].v, q, start);
        if constexpr (NH == 2) d += dot32<BF16>(a[1].v, q, 0.f);
        acc[u] = fmaf(factor * ScaleIo<ST>::to_f32(c.s[u], BF16), d, acc[u]);
    }
}

// The sum over the LPC lanes of a column, in each of them.
template <int LPC>
__device__ __forceinline__ float over_lanes(float v)
{
    auto add = [](float a, float b) { return a + b; };
    if constexpr (LPC == 64) return over_wave(v, add);
    v += __shfl_xor(v, 8, 64);
    v += __shfl_xor(v, 4, 64);
    v += __shfl_xor(v, 2, 64);
    v += __shfl_xor(v, 1, 64);
    if constexpr (LPC == 32) v += __shfl_xor(v, 16, 64);
    return v;
}

constexpr int kFewRows = 4;

// What is known before the call's other arguments are read: in scalar registers when a wave starts.
#define MOE_FEW_FIRST const void *logits, const uint16_t *x, int logits_dtype, int rows, int experts, int k, int normalize, unsigned col_tiles

// A wave has NU times 64 / LPC columns of gate and up, a workgroup four times as many.
template <bool BF16, typename ST, bool ZP, int LPC>
__global__ __launch_bounds__(256) void moe_few_up_kernel(MOE_FEW_FIRST, MoeUpCall p)
{
    constexpr int NU = 4, kCols = NU * 64 / LPC;
    __shared__ MoeFewRouting routing;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const unsigned slot = blockIdx.x / col_tiles;
    const int n0 = (static_cast<int>(blockIdx.x - slot * col_tiles) * 4 + wave) * kCols;
    route_few(routing, logits, logits_dtype, rows, experts, k, normalize);
    if (blockIdx.x == 0) write_table(routing, rows, k, p.table);
    if (static_cast<int>(slot) >= routing.active || n0 >= p.ip) return;
    const int expert = __builtin_amdgcn_readfirstlane(routing.chosen[slot]);
    const int live = min(p.m.n - n0, kCols);
    float g[kFewRows][NU] = {}, u[kFewRows][NU] = {};
    unsigned chose = 0;
    for (int t = 0; t < rows; ++t)
        for (int j = 0; j < k; ++j) chose |= static_cast<unsigned>(routing.expert[t * k + j] == expert) << t;
    chose = __builtin_amdgcn_readfirstlane(chose);
    if (live > 0) {
        MoeMatrix up = p.m;
        up.w[0] = p.m.w[1];
        const MoeTile<1> tg = moe_tile<ST, ZP, 1>(p.m, expert, n0, live), tu = moe_tile<ST, ZP, 1>(up, expert, n0, live);
        const int kl = lane % LPC, width = static_cast<int>(p.ldx);
        FewColumns<ST, ZP, NU, LPC> cg, cu;
        for (int k0 = 0; k0 < width; k0 += LPC * 32) {
            const int at = k0 + kl * 32, count = width - at;
            cg.load(p.m, tg, live, at, count > 0 ? kl : -1);
            cu.load(p.m, tu, live, at, count > 0 ? kl : -1);
            const int odd = (at / p.m.block_size) & 1;
#pragma unroll
            for (int t = 0; t < kFewRows; ++t) {
                if (!(chose >> t & 1)) continue;
                Elements32<BF16> a[1];
                a[0].load(x + t * p.ldx + at, count);
                few_multiply<BF16, ST, ZP, NU, LPC, 1>(cg, a, odd, 1.f, g[t]);
                few_multiply<BF16, ST, ZP, NU, LPC, 1>(cu, a, odd, 1.f, u[t]);
            }
        }
    }
    // lane u of a column's lanes keeps column u's result
    const int mine = lane % LPC, col = n0 + mine * (64 / LPC) + lane / LPC;
#pragma unroll
    for (int t = 0; t < kFewRows; ++t) {
        if (!(chose >> t & 1)) continue;
        float gate = 0.f, upv = 0.f;
#pragma unroll
        for (int i = 0; i < NU; ++i) {
            const float a = over_lanes<LPC>(g[t][i]), b = over_lanes<LPC>(u[t][i]);
            if (mine == i) {
                gate = a;
                upv = b;
            }
        }
        if (mine < NU && col < p.ip) store_h<BF16>(p, static_cast<int64_t>(slot) * kFewRows + t, col, col < p.m.n ? moe_gated(p, expert, col, gate, upv) : 0.f);
    }
}

// A wave has eight columns and a share of the experts' K; a workgroup's waves have the same columns.
template <bool BF16, typename ST, bool ZP, int LPC>
__global__ __launch_bounds__(512) void moe_few_down_kernel(MoeDownCall p)
{
    constexpr int NU = LPC / 8, kCols = 8;
    __shared__ float sums[8][kFewRows][kCols];
    __shared__ float weight[kFewPairs][kFewRows];
    __shared__ int32_t chosen[kFewPairs];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6, lane = threadIdx.x & 63;
    const int n0 = static_cast<int>(blockIdx.x) * kCols, live = min(p.m.n - n0, kCols);
    const int active = p.table->active;
    for (int i = threadIdx.x; i < active * kFewRows; i += blockDim.x) weight[i / kFewRows][i % kFewRows] = p.table->weight[i / kFewRows][i % kFewRows];
    for (int i = threadIdx.x; i < active; i += blockDim.x) chosen[i] = p.table->expert[i];
    __syncthreads();
    const int kl = lane % LPC, width = static_cast<int>(p.ip), passes = (width + LPC * 32 - 1) / (LPC * 32);
    float acc[kFewRows][NU] = {};
    for (int item = wave; item < active * passes; item += waves) {
        const int slot = item / passes, at = (item - slot * passes) * (LPC * 32) + kl * 32, count = width - at;
        const MoeTile<1> tile = moe_tile<ST, ZP, 1>(p.m, __builtin_amdgcn_readfirstlane(chosen[slot]), n0, live);
        FewColumns<ST, ZP, NU, LPC> c;
        c.load(p.m, tile, live, at, count > 0 ? kl : -1);
        const int odd = (at / p.m.block_size) & 1;
#pragma unroll
        for (int t = 0; t < kFewRows; ++t) {
            const float w = weight[slot][t];
            if (!(w > 0.f)) continue;
            const uint16_t* const h = p.h + (static_cast<int64_t>(slot) * kFewRows + t) * (2 * p.ip) + at;
            Elements32<BF16> a[2];
            a[0].load(h, count);
            a[1].load(h + p.ip, count);
            few_multiply<BF16, ST, ZP, NU, LPC, 2>(c, a, odd, w, acc[t]);
        }
    }
#pragma unroll
    for (int t = 0; t < kFewRows; ++t) {
        if (t >= p.rows) continue;
#pragma unroll
        for (int i = 0; i < NU; ++i) {
            const float v = over_lanes<LPC>(acc[t][i]);
            if (kl == i) sums[wave][t][i * (64 / LPC) + lane / LPC] = v;
        }
    }
    __syncthreads();
    const int row = threadIdx.x / kCols, c = threadIdx.x % kCols;
    if (row >= p.rows || c >= live) return;
    float v = p.table->base[row];
    for (int w = 0; w < waves; ++w) v += sums[w][row][c];
    const int64_t col = n0 + c;
    if (p.m.w[0].bias)
        for (int i = 0; i < active; ++i) {
            const float f = weight[i][row];
            if (f > 0.f) v = fmaf(f, load_as_f32(p.m.w[0].bias, p.m.bias_dtype, chosen[i] * p.m.expert_step + col), v);
        }
    store_from_f32(p.y, BF16 ? ROCM_DT_BF16 : ROCM_DT_F16, row * static_cast<int64_t>(p.m.n) + col, v);
}

// The lanes that a row of k elements keeps busiest; the longer read where that is equal.
int lanes_per_column(int64_t k)
{
    int best = 64;
    for (int lpc : {32, 16}) {
        auto taken = [&](int l) { return (k + l * 32 - 1) / (l * 32) * l; };
        if (taken(lpc) < taken(best)) best = lpc;
    }
    return best;
}

template <typename F>
int few_build(const RocmMoeArgs& a, bool zp, int lpc, F go)
{
    auto laned = [&](auto bf, auto st, auto z) {
        if (lpc == 64) return go(bf, st, z, std::integral_constant<int, 64>{});
        if (lpc == 32) return go(bf, st, z, std::integral_constant<int, 32>{});
        return go(bf, st, z, std::integral_constant<int, 16>{});
    };
    auto scaled = [&](auto bf) {
        if (a.scale_dtype == ROCM_DT_F32) return zp ? laned(bf, float{}, std::true_type{}) : laned(bf, float{}, std::false_type{});
        return zp ? laned(bf, uint16_t{}, std::true_type{}) : laned(bf, uint16_t{}, std::false_type{});
    };
    return a.dtype == ROCM_DT_BF16 ? scaled(std::true_type{}) : scaled(std::false_type{});
}

}  // namespace

int launch_moe_few(const RocmMoeArgs& a, const MoeUpCall& up, const MoeDownCall& down, int slots, hipStream_t s)
{
    int rc = few_build(a, a.gate.zp != nullptr, lanes_per_column(up.ldx), [&](auto bf, auto st, auto zp, auto lanes) {
        constexpr int LPC = decltype(lanes)::value;
        const unsigned col_tiles = static_cast<unsigned>((up.ip + 1024 / LPC - 1) / (1024 / LPC));
        hipLaunchKernelGGL((moe_few_up_kernel<decltype(bf)::value, decltype(st), decltype(zp)::value, LPC>), dim3(col_tiles * static_cast<unsigned>(slots)), dim3(256), 0, s, up.logits, up.x,
                           up.logits_dtype, up.rows, up.experts, up.k, up.normalize, col_tiles, up);
        return static_cast<int>(hipGetLastError());
    });
    if (rc != 0) return rc;
    return few_build(a, a.down.zp != nullptr, lanes_per_column(down.ip), [&](auto bf, auto st, auto zp, auto lanes) {
        hipLaunchKernelGGL((moe_few_down_kernel<decltype(bf)::value, decltype(st), decltype(zp)::value, decltype(lanes)::value>), dim3(static_cast<unsigned>(down.m.n + 7) / 8), dim3(512), 0, s, down);
        return static_cast<int>(hipGetLastError());
    });
}

}  // namespace mnb
