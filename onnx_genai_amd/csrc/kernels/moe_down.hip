// QMoE, second half: the experts' down projections and their weighted sum.
#include "moe_dot.hiph"

namespace mnb {
namespace {

// Up to 16 tokens: y = base + sum over the active experts of weight * (h W2^T + bias), a product over all experts' K one behind the other. A workgroup has
// 16 columns; its waves share the steps of all experts evenly, and what they have is added up in one order.
template <bool BF16, int BS, typename ST, bool ZP>
__global__ __launch_bounds__(512) void moe_down_few_kernel(MoeDownCall p)
{
    constexpr int kRows = kFewTokens;
    using Dot = MoeDot<BF16, BS, ST, ZP, 1, 2>;
    __shared__ float sums[8][256];
    __shared__ float weight[kFewPairs][kRows];
    __shared__ int32_t experts[kFewPairs];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const int n0 = static_cast<int>(blockIdx.x) * kRows, live = min(p.m.n - n0, kRows);
    const int active = p.table->active;
    for (int i = threadIdx.x; i < active * kRows; i += blockDim.x) weight[i / kRows][i % kRows] = p.table->weight[i / kRows][i % kRows];
    for (int i = threadIdx.x; i < active; i += blockDim.x) experts[i] = p.table->expert[i];
    __syncthreads();

    const Dot dot(p.m, live);
    const int steps = static_cast<int>(p.ip / 128), items = active * steps;
    const int begin = static_cast<int>(static_cast<int64_t>(items) * wave / waves), end = static_cast<int>(static_cast<int64_t>(items) * (wave + 1) / waves);
    f32x4_t total[1] = {}, y = {0.f, 0.f, 0.f, 0.f};
    int slot = -1;
    auto flush = [&] {
        if (slot < 0) return;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float w = weight[slot][dot.g * 4 + i];
            y[i] += w > 0.f ? w * total[0][i] : 0.f;                       // (a row of h that is not finite is another token's)
            total[0][i] = 0.f;
        }
    };
    moe_pipeline<typename Dot::Step>(begin, end,
                                     [&](typename Dot::Step& s, int item) {
                                         const int at = static_cast<int>(static_cast<unsigned>(item) / static_cast<unsigned>(steps));
                                         const MoeTile<1> tile = moe_tile<ST, ZP, 1>(p.m, __builtin_amdgcn_readfirstlane(experts[at]), n0, live);
                                         dot.template load<false>(s, tile, item - at * steps, p.h + (static_cast<int64_t>(at) * kRows + dot.col) * (2 * p.ip), dot.col < p.rows, p.ip, 0);
                                     },
                                     [&](const typename Dot::Step& s, int item) {
                                         if (item / steps != slot) {
                                             flush();
                                             slot = item / steps;
                                         }
                                         dot.multiply(s, total);
                                     });
    flush();
#pragma unroll
    for (int i = 0; i < 4; ++i) sums[wave][(dot.g * 4 + i) * 16 + dot.col] = y[i];
    __syncthreads();
    const int row = threadIdx.x / kRows, c = threadIdx.x % kRows;
    if (row >= kRows || row >= p.rows || c >= live) return;
    float v = p.table->base[row];
    for (int w = 0; w < waves; ++w) v += sums[w][threadIdx.x];
    const int64_t col = n0 + c;
    if (p.m.w[0].bias)
        for (int i = 0; i < active; ++i) v = fmaf(weight[i][row], load_as_f32(p.m.w[0].bias, p.m.bias_dtype, experts[i] * p.m.expert_step + col), v);
    store_from_f32(p.y, BF16 ? ROCM_DT_BF16 : ROCM_DT_F16, row * static_cast<int64_t>(p.m.n) + col, v);
}

}  // namespace

int launch_moe_down(const RocmMoeArgs& a, const MoeDownCall& p, hipStream_t s)
{
    return moe_build(a, a.down.zp != nullptr, [&](auto bf, auto bs, auto st, auto zp) {
        constexpr bool BF16 = decltype(bf)::value, ZP = decltype(zp)::value;
        constexpr int BS = decltype(bs)::value;
        using ST = decltype(st);
        const unsigned n = static_cast<unsigned>(p.m.n);
        hipLaunchKernelGGL((moe_down_few_kernel<BF16, BS, ST, ZP>), dim3((n + 15) / 16), dim3(512), 0, s, p);
        return static_cast<int>(hipGetLastError());
    });
}

}  // namespace mnb
