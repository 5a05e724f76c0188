// QMoE over few rows an expert: the weights stream once through v_mfma_f32_16x16x32_{f16,bf16}, 16 columns by 16 rows of pairs.
//
//   h = act(x Wg^T + bg, x Wu^T + bu),  act(g, u) = g sigmoid(alpha g) (u + beta), g <= limit, |u| <= limit           (moe_gate_up_kernel)
//   out = h W2^T                                                                                                       (moe_down_kernel)
//
// The weights' bytes bound it. A lane reads 16 bytes of one column's packed row as the caller holds them. A nibble q becomes the 16-bit float magic + q with
// one permutation and one and-or for two (magic = 1024 in f16, 128 in bf16: exact), and the matrix core sums a (magic + q) over a block; with S the
// block's sum of a, from a product with ones,
//   sum a (q - zp) scale = scale (sum a (magic + q) - (magic + zp) S).
// The f32 sums hold magic + q next to q - zp, which costs at most eight of their 24 bits: 2^-16 of the largest terms, a sixteenth of an f16 result's half step.
// h is rounded to the activations' type, as a graph of separate nodes has it and as the matrix core needs it: half a step of the type, as the result's own.
#include "moe.hiph"

namespace mnb {
namespace {

typedef __attribute__((ext_vector_type(8))) _Float16 half8_t;
typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8_t;
typedef __attribute__((ext_vector_type(4))) float f32x4_t;

template <bool BF16>
__device__ __forceinline__ f32x4_t mfma16(const uint4& a, const uint4& b, f32x4_t c)
{
    if constexpr (BF16) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, a), __builtin_bit_cast(half8_t, b), c, 0, 0, 0);
}

template <bool BF16>
__device__ __forceinline__ uint4 magic_nibbles(uint32_t w)
{
    constexpr uint32_t kMagic = BF16 ? 0x43004300u : 0x64006400u;
    const uint32_t w4 = w >> 4;
    auto pair = [&](uint32_t sel) { return (__builtin_amdgcn_perm(w4, w, sel) & 0x000f000fu) | kMagic; };
    return make_uint4(pair(0x0c040c00u), pair(0x0c050c01u), pair(0x0c060c02u), pair(0x0c070c03u));
}

struct MoeRowsParams {
    const uint16_t* x;       // rows of ldx elements (a multiple of 8), zeros from k on
    int64_t ldx;
    const int32_t* token;    // row of a pair -> row of x; NULL: the same
    const int4* tiles;
    MoeWeights w[2];
    int64_t expert_step;     // rows of w from one expert to the next
    int row_step;            // and from one column to the next
    int n, kb, block_size;
    unsigned col_tiles;
    int64_t row_bytes, zp_row;
    int chunks;              // of 128 k
    int scale_dtype, bias_dtype;
    void* out;
    int64_t ldo;
    float alpha, beta, limit;
};

// Sums of one 16 x 16 tile of NM products over chunks [begin, end) of K: lane l has column l % 16 and rows 4 (l / 16) + i.
// BS: the block size, 128 for those above, too.
template <bool BF16, int BS, int NM>
__device__ __forceinline__ void moe_dot(const MoeRowsParams& p, int expert, int n0, const uint16_t* x_row, int begin, int end, f32x4_t (&total)[NM])
{
    constexpr bool kTranspose = BS < 128;
    constexpr int kBlocks = 128 / BS, kSteps = 4 / kBlocks;
    const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
    const bool live = n0 + c < p.n;
    const uint8_t* b[NM];
    int64_t at[NM];
#pragma unroll
    for (int m = 0; m < NM; ++m) {
        at[m] = expert * p.expert_step + static_cast<int64_t>(live ? n0 + c : 0) * p.row_step;
        b[m] = p.w[m].b + at[m] * p.row_bytes;
    }
    const uint4 ones = BF16 ? make_uint4(0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u) : make_uint4(0x3c003c00u, 0x3c003c00u, 0x3c003c00u, 0x3c003c00u);
    for (int t = begin; t < end; ++t) {
        uint4 w[NM], a[4];
        const int64_t byte = static_cast<int64_t>(t) * 64 + g * 16;
#pragma unroll
        for (int m = 0; m < NM; ++m) {
            w[m] = byte < p.row_bytes ? *reinterpret_cast<const uint4*>(b[m] + byte) : make_uint4(0, 0, 0, 0);
            if constexpr (kTranspose) transpose_groups(w[m]);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int64_t k = static_cast<int64_t>(t) * 128 + (kTranspose ? j * 32 + g * 8 : g * 32 + j * 8);
            a[j] = x_row && k < p.ldx ? *reinterpret_cast<const uint4*>(x_row + k) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int q = 0; q < kBlocks; ++q) {
            f32x4_t s = {0.f, 0.f, 0.f, 0.f}, sum[NM] = {};
#pragma unroll
            for (int j = q * kSteps; j < (q + 1) * kSteps; ++j) {
                s = mfma16<BF16>(a[j], ones, s);
#pragma unroll
                for (int m = 0; m < NM; ++m) {
                    const uint32_t d = j == 0 ? w[m].x : j == 1 ? w[m].y : j == 2 ? w[m].z : w[m].w;
                    sum[m] = mfma16<BF16>(a[j], magic_nibbles<BF16>(d), sum[m]);
                }
            }
            const int block = BS < 128 ? t * kBlocks + q : static_cast<int>(static_cast<int64_t>(t) * 128 / p.block_size);
#pragma unroll
            for (int m = 0; m < NM; ++m) {
                const float scale = block < p.kb ? load_as_f32(p.w[m].scales, p.scale_dtype, at[m] * p.kb + block) : 0.f;
                const int z = block < p.kb ? zero_point_of(p.w[m].zp ? p.w[m].zp + at[m] * p.zp_row : nullptr, block) : 8;
                const float off = -static_cast<float>((BF16 ? 128 : 1024) + z);
#pragma unroll
                for (int i = 0; i < 4; ++i) total[m][i] = fmaf(scale, fmaf(off, s[i], sum[m][i]), total[m][i]);
            }
        }
    }
}

template <bool BF16, int BS, int NM>
__device__ __forceinline__ bool moe_tile_sums(const MoeRowsParams& p, const int4& tile, int n0, float (*sums)[NM * 4][64], f32x4_t (&total)[NM])
{
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const int r = lane & 15;
    const uint16_t* x_row = nullptr;
    if (r < tile.z) {
        const int64_t row = p.token ? p.token[tile.y + r] : tile.y + r;
        x_row = p.x + row * p.ldx;
    }
    const int per_wave = (p.chunks + waves - 1) / waves;
    const int begin = wave * per_wave, end = min(begin + per_wave, p.chunks);
    moe_dot<BF16, BS, NM>(p, tile.x, n0, x_row, begin, end, total);
#pragma unroll
    for (int m = 0; m < NM; ++m)
#pragma unroll
        for (int i = 0; i < 4; ++i) sums[wave][m * 4 + i][lane] = total[m][i];
    __syncthreads();
    if (wave != 0) return false;
#pragma unroll
    for (int m = 0; m < NM; ++m)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float v = sums[0][m * 4 + i][lane];
            for (int w = 1; w < waves; ++w) v += sums[w][m * 4 + i][lane];
            total[m][i] = v;
        }
    return true;
}

template <bool BF16, int BS>
__global__ __launch_bounds__(256) void moe_gate_up_kernel(MoeRowsParams p)
{
    __shared__ float sums[4][8][64];
    const int4 tile = p.tiles[blockIdx.x / p.col_tiles];
    if (tile.z == 0) return;
    const int n0 = static_cast<int>(blockIdx.x % p.col_tiles) * 16;
    f32x4_t total[2] = {};
    if (!moe_tile_sums<BF16, BS, 2>(p, tile, n0, sums, total)) return;
    const int lane = threadIdx.x & 63, col = n0 + (lane & 15);
    float bg = 0.f, bu = 0.f;
    if (p.w[0].bias && col < p.n) {
        const int64_t at = tile.x * p.expert_step + static_cast<int64_t>(col) * p.row_step;
        bg = load_as_f32(p.w[0].bias, p.bias_dtype, at);
        bu = load_as_f32(p.w[1].bias, p.bias_dtype, at);
    }
    uint16_t* const out = static_cast<uint16_t*>(p.out);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = (lane >> 4) * 4 + i;
        if (r >= tile.z) continue;
        const float v = col < p.n ? moe_activation(total[0][i] + bg, total[1][i] + bu, p.alpha, p.beta, p.limit) : 0.f;
        out[(tile.y + r) * p.ldo + col] = BF16 ? f32_to_bf16_bits(v) : f32_to_f16_bits(v);
    }
}

template <bool BF16, int BS>
__global__ __launch_bounds__(256) void moe_down_kernel(MoeRowsParams p)
{
    __shared__ float sums[4][4][64];
    const int4 tile = p.tiles[blockIdx.x / p.col_tiles];
    if (tile.z == 0) return;
    const int n0 = static_cast<int>(blockIdx.x % p.col_tiles) * 16;
    f32x4_t total[1] = {};
    if (!moe_tile_sums<BF16, BS, 1>(p, tile, n0, sums, total)) return;
    const int lane = threadIdx.x & 63, col = n0 + (lane & 15);
    if (col >= p.n) return;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = (lane >> 4) * 4 + i;
        if (r < tile.z) static_cast<float*>(p.out)[(tile.y + r) * p.ldo + col] = total[0][i];
    }
}

MoeWeights weights_of(const RocmMoeWeights& w) { return MoeWeights{w.b, w.scales, w.zp, w.bias}; }

// The workspace of a call, part by part.
struct MoeLayout {
    int64_t kp, ip, pairs;
    int max_tiles;
    uint64_t expert, weight, pair_row, token, base, tiles, x, act, out, total;
};
constexpr int kTileRows = 16;

MoeLayout layout_of(const RocmMoeArgs& a)
{
    MoeLayout l{};
    l.pairs = a.rows * a.k;
    l.kp = (a.hidden + 7) / 8 * 8;
    l.ip = (a.inter + 15) / 16 * 16;
    l.max_tiles = static_cast<int>(l.pairs / kTileRows + (l.pairs < a.experts ? l.pairs : a.experts));
    uint64_t at = 0;
    auto part = [&](uint64_t bytes) {
        const uint64_t here = at;
        at += (bytes + 255) / 256 * 256;
        return here;
    };
    l.expert = part(l.pairs * 4);
    l.weight = part(l.pairs * 4);
    l.pair_row = part(l.pairs * 4);
    l.token = part(l.pairs * 4);
    l.base = part(a.rows * 4);
    l.tiles = part(static_cast<uint64_t>(l.max_tiles) * 16);
    l.x = part(l.kp != a.hidden ? a.rows * l.kp * 2 : 0);
    l.act = part(l.pairs * l.ip * 2);
    l.out = part(l.pairs * a.hidden * 4);
    l.total = at;
    return l;
}

}  // namespace
}  // namespace mnb

extern "C" uint64_t rocm_moe_workspace_bytes(const RocmMoeArgs* args) { return mnb::layout_of(*args).total; }
extern "C" const char* rocm_moe_variant(const RocmMoeArgs*) { return "moe_rows"; }

extern "C" int rocm_launch_moe(const RocmMoeArgs* args, void* workspace, rocm_stream_t stream)
{
    using namespace mnb;
    const RocmMoeArgs& a = *args;
    if (a.rows <= 0) return 0;
    hipStream_t s = static_cast<hipStream_t>(stream);
    const MoeLayout l = layout_of(a);
    uint8_t* const ws = static_cast<uint8_t*>(workspace);
    const MoeRoute route{reinterpret_cast<int32_t*>(ws + l.expert), reinterpret_cast<float*>(ws + l.weight), reinterpret_cast<int32_t*>(ws + l.pair_row),
                         reinterpret_cast<int32_t*>(ws + l.token), reinterpret_cast<float*>(ws + l.base), reinterpret_cast<int4*>(ws + l.tiles)};
    int rc = launch_moe_top_k(a, route, s);
    if (rc == 0) rc = launch_moe_plan(a, kTileRows, l.max_tiles, route, s);
    const void* x = a.x;
    if (rc == 0 && l.kp != a.hidden) {
        rc = launch_moe_pad_rows(a.x, a.rows, a.hidden, l.kp, ws + l.x, s);
        x = ws + l.x;
    }
    if (rc != 0) return rc;
    auto shaped = [&](MoeRowsParams& p, int64_t k, int64_t n) {
        p.tiles = route.tiles;
        p.n = static_cast<int>(n);
        p.col_tiles = static_cast<unsigned>((n + 15) / 16);
        p.kb = static_cast<int>((k + a.block_size - 1) / a.block_size);
        p.block_size = a.block_size;
        p.row_bytes = static_cast<int64_t>(p.kb) * a.block_size / 2;
        p.zp_row = (p.kb + 1) / 2;
        p.chunks = static_cast<int>((k + 127) / 128);
        p.scale_dtype = a.scale_dtype;
        p.bias_dtype = a.bias_dtype;
    };
    MoeRowsParams up{}, down{};
    shaped(up, a.hidden, a.inter);
    up.x = static_cast<const uint16_t*>(x);
    up.ldx = l.kp;
    up.token = route.token;
    up.w[0] = weights_of(a.gate);
    up.w[1] = weights_of(a.up);
    up.expert_step = a.up_expert_step;
    up.row_step = a.up_row_step;
    up.out = ws + l.act;
    up.ldo = l.ip;
    up.alpha = a.alpha;
    up.beta = a.beta;
    up.limit = a.limit;
    shaped(down, a.inter, a.hidden);
    down.x = reinterpret_cast<const uint16_t*>(ws + l.act);
    down.ldx = l.ip;
    down.w[0] = weights_of(a.down);
    down.expert_step = a.hidden;
    down.row_step = 1;
    down.out = ws + l.out;
    down.ldo = a.hidden;
    auto both = [&](auto bf, auto bs) {
        constexpr bool BF16 = decltype(bf)::value;
        constexpr int BS = decltype(bs)::value;
        hipLaunchKernelGGL((moe_gate_up_kernel<BF16, BS>), dim3(up.col_tiles * static_cast<unsigned>(l.max_tiles)), dim3(256), 0, s, up);
        hipLaunchKernelGGL((moe_down_kernel<BF16, BS>), dim3(down.col_tiles * static_cast<unsigned>(l.max_tiles)), dim3(256), 0, s, down);
        return static_cast<int>(hipGetLastError());
    };
    auto sized = [&](auto bf) {
        return a.block_size == 32 ? both(bf, std::integral_constant<int, 32>{}) : a.block_size == 64 ? both(bf, std::integral_constant<int, 64>{}) : both(bf, std::integral_constant<int, 128>{});
    };
    rc = a.dtype == ROCM_DT_BF16 ? sized(std::true_type{}) : sized(std::false_type{});
    return rc != 0 ? rc : launch_moe_combine(a, route, reinterpret_cast<const float*>(ws + l.out), s);
}
