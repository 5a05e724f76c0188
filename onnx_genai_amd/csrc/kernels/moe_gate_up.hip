// QMoE, first half: h = act(x Wg^T + bg, x Wu^T + bu) of each expert for the rows that chose it,
//   act(g, u) = g sigmoid(alpha g) (u + beta),  g <= limit, |u| <= limit.
// h is held as a 16-bit value and the 16-bit rounding of what that left, so that the second half's matrix product loses nothing of it.
#include "moe_dot.hiph"

namespace mnb {
namespace {

// Up to 16 tokens: every active expert has a row for each, zero where the token did not choose it. A workgroup has 16 columns of gate and of up, K split over
// its waves.
template <bool BF16, int BS, typename ST, bool ZP>
__global__ __launch_bounds__(256) void moe_gate_up_kernel(MoeUpCall p)
{
    using Dot = MoeDot<BF16, BS, ST, ZP, 2, 1>;
    __shared__ float sums[4][2][256];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int slot = static_cast<int>(blockIdx.y), n0 = static_cast<int>(blockIdx.x) * 16;
    if (slot >= p.table->active) return;
    const int expert = p.table->expert[slot];
    const int64_t h_row = static_cast<int64_t>(slot) * kFewTokens;
    const int live = min(p.m.n - n0, 16);
    if (live > 0) {
        f32x4_t total[2] = {};
        const Dot dot(p.m, live);
        const MoeTile<2> tile = moe_tile<ST, ZP, 2>(p.m, expert, n0, live);
        const bool has = p.table->weight[slot][dot.col] > 0.f;
        const uint16_t* const x = p.x + (has ? dot.col : 0) * p.ldx;
        const int steps = static_cast<int>((p.ldx + 127) / 128), whole = static_cast<int>(p.ldx / 128);
        const int begin = steps * wave / 4, end = steps * (wave + 1) / 4;
        moe_pipeline<typename Dot::Step>(begin, min(end, whole), [&](typename Dot::Step& s, int t) { dot.template load<false>(s, tile, t, x, has, 0, 0); },
                                         [&](const typename Dot::Step& s, int) { dot.multiply(s, total); });
        if (whole < steps && end == steps && begin < end) {
            typename Dot::Step s = {};
            dot.template load<true>(s, tile, whole, x, has, 0, static_cast<int>(p.ldx));
            dot.multiply(s, total);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            sums[wave][0][(dot.g * 4 + i) * 16 + dot.col] = total[0][i];
            sums[wave][1][(dot.g * 4 + i) * 16 + dot.col] = total[1][i];
        }
    }
    __syncthreads();
    const int row = threadIdx.x >> 4, col = n0 + (threadIdx.x & 15);
    float v = 0.f;
    if (p.table->weight[slot][row] > 0.f && col < p.m.n) {
        float g = 0.f, u = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            g += sums[w][0][threadIdx.x];
            u += sums[w][1][threadIdx.x];
        }
        v = moe_gated(p, expert, col, g, u);
    }
    store_h<BF16>(p, h_row + row, col, v);
}

}  // namespace

int launch_moe_gate_up(const RocmMoeArgs& a, const MoeUpCall& p, int slots, hipStream_t s)
{
    return moe_build(a, a.gate.zp != nullptr, [&](auto bf, auto bs, auto st, auto zp) {
        constexpr bool BF16 = decltype(bf)::value, ZP = decltype(zp)::value;
        constexpr int BS = decltype(bs)::value;
        using ST = decltype(st);
        hipLaunchKernelGGL((moe_gate_up_kernel<BF16, BS, ST, ZP>), dim3(static_cast<unsigned>(p.ip / 16), static_cast<unsigned>(slots)), dim3(256), 0, s, p);
        return static_cast<int>(hipGetLastError());
    });
}

}  // namespace mnb
