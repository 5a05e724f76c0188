// QMoE for up to four tokens, in two launches, each weight read once.
//
//   moe_few_up_kernel     every workgroup routes the tokens for itself; h = act(x Wg^T + bg, x Wu^T + bu) of one expert's columns for the rows that chose it
//   moe_few_down_kernel   y = base + sum over the active experts of weight * (h W2^T + bias)
//
// The weights' bytes bound it once there are enough of them, and before that the way to them: arguments, logits and weights are reached one after the other.
// A lane holds 32 elements of K of a row of x in registers and multiplies them with 32 nibbles of each of several columns: f16 in 16 dot products of two (v_dot2_f32_f16),
// bf16 in f32 by 32 mixed-precision multiply-adds (v_fma_mix_f32). A weight enters as the f16 q - zp, which is exact, so that one of zero adds nothing however large its x
// is. (As magic + q, with -(magic + zp) times the sum of x in front, a pair of weights takes one instruction less in f16 and two in bf16, and what is left of magic * x
// shows: an x of 60000 at weights of zero put y off by 15 %. One token 17.7 us and 18.4 now, three tokens of 4096 and 14336 131 and 133.)
// Measured: one token, 8 of 64 experts of 2048 and 1024 in bf16, 12.6 us up and 7.4 down (28 MB; an empty launch is 2 us, and routing 3 more before the first weights),
// three tokens of 4096 and 14336 over 8 experts in f16 with zero points 82 and 58 us (3.8 and 2.7 TB/s).
// LPC lanes stand side by side on K and read 16 LPC bytes of a column's row as the caller holds it; 64 / LPC columns are read at once.
#include "moe_route.hiph"

namespace mnb {
namespace {

// What a step reads of its tile of columns: wave-uniform.
template <int NM>
struct MoeTile {
    __amdgpu_buffer_rsrc_t w[NM], s[NM], z[NM];
};

// Columns [n0, n0 + live) of an expert; with none, every load reads as zeros and goes to no memory.
template <typename ST, bool ZP, int NM>
__device__ __forceinline__ MoeTile<NM> moe_tile(const MoeMatrix& m, int expert, int n0, int live)
{
    MoeTile<NM> t;
    const int64_t row = expert * m.expert_step + static_cast<int64_t>(n0) * m.row_step;
    const uint64_t rows = live > 0 ? static_cast<uint64_t>(live - 1) * m.row_step + 1 : 0;
#pragma unroll
    for (int i = 0; i < NM; ++i) {
        t.w[i] = make_srd(m.w[i].b + row * m.row_bytes, rows * m.row_bytes);
        t.s[i] = make_srd(static_cast<const ST*>(m.w[i].scales) + row * m.kb, rows * m.kb * sizeof(ST));
        t.z[i] = ZP ? make_srd(m.w[i].zp + row * m.zp_row, rows * m.zp_row) : t.w[i];
    }
    return t;
}

// 32 elements of a row in the order of a dword's nibbles under a mask and shifts: 0 4 | 1 5 | 2 6 | 3 7 of each eight.
struct Elements32 {
    uint32_t v[16];

    // `count` of them are there (a multiple of 8), the rest is zero
    __device__ __forceinline__ void load(const uint16_t* x, int count)
    {
#pragma unroll
        for (int j = 0; j < 4; ++j) put(j, j * 8 < count ? *reinterpret_cast<const uint4*>(x + j * 8) : make_uint4(0, 0, 0, 0));
    }
    __device__ __forceinline__ void put(int j, const uint4& d)
    {
        v[4 * j] = d.x;
        v[4 * j + 1] = d.y;
        v[4 * j + 2] = d.z;
        v[4 * j + 3] = d.w;
    }
    __device__ __forceinline__ void order()
    {
#pragma unroll
        for (int j = 0; j < 4; ++j) put(j, ordered(make_uint4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3])));
    }
    static __device__ __forceinline__ uint4 ordered(const uint4& d)
    {
        return make_uint4(__builtin_amdgcn_perm(d.z, d.x, 0x05040100u), __builtin_amdgcn_perm(d.z, d.x, 0x07060302u), __builtin_amdgcn_perm(d.w, d.y, 0x05040100u),
                          __builtin_amdgcn_perm(d.w, d.y, 0x07060302u));
    }
};

// 32 nibbles as f16 pairs q - z, exact. A nibble in the low four bits of an f16's ten is 1024 + q, in the next four 1024 + 16 q, which one packed multiply-add takes
// to q - z: two of a dword's four pairs need no shift of their own.
// What that takes, in registers: masks in vector ones and the magic in a scalar one make and, or one instruction.
struct Unpacking {
    uint32_t low = 0x000f000fu, high = 0x00f000f0u, magic = opaque_scalar(0x64006400u);
    __device__ __forceinline__ Unpacking() { asm volatile("" : "+v"(low), "+v"(high)); }
};
__device__ __forceinline__ void weights32(const Unpacking& by, const uint4& w, uint32_t z, half2p_t (&out)[16])
{
    uint32_t d[4] = {w.x, w.y, w.z, w.w};
    // unpacked for each row anew: kept for the next row, the nibbles of a wave's columns take 128 registers
    asm volatile("" : "+v"(d[0]), "+v"(d[1]), "+v"(d[2]), "+v"(d[3]));
    // -(1024 + z) and -(64 + z): f16's steps there are 1 and 1/16
    const half2p_t off = __builtin_bit_cast(half2p_t, 0xE400E400u + z * 0x00010001u), off_high = __builtin_bit_cast(half2p_t, 0xD400D400u + z * 0x00100010u);
    const half2p_t sixteenth = __builtin_bit_cast(half2p_t, 0x2C002C00u);
    auto pair = [&](uint32_t bits, uint32_t mask) { return __builtin_bit_cast(half2p_t, (bits & mask) | by.magic); };
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const uint32_t upper = d[j] >> 8;
        out[4 * j] = pair(d[j], by.low) + off;
        out[4 * j + 1] = __builtin_elementwise_fma(pair(d[j], by.high), sixteenth, off_high);
        out[4 * j + 2] = pair(upper, by.low) + off;
        out[4 * j + 3] = __builtin_elementwise_fma(pair(upper, by.high), sixteenth, off_high);
    }
}

// A row's 32 elements as they are multiplied, and their product with 32 weights, in four chains. f16: dot products of two, for each part of a value.
template <bool BF16, int NH>
struct Factors32 {
    uint32_t v[NH][16];
    __device__ __forceinline__ explicit Factors32(const Elements32 (&a)[NH])
    {
#pragma unroll
        for (int h = 0; h < NH; ++h)
#pragma unroll
            for (int i = 0; i < 16; ++i) v[h][i] = a[h].v[i];
    }
    __device__ __forceinline__ float dot(const half2p_t (&q)[16]) const
    {
        float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int h = 0; h < NH; ++h)
#pragma unroll
            for (int i = 0; i < 16; ++i) s[i & 3] = __builtin_amdgcn_fdot2(__builtin_bit_cast(half2p_t, v[h][i]), q[i], s[i & 3], false);
        return (s[0] + s[1]) + (s[2] + s[3]);
    }
};
// bf16: in f32, the parts of a value joined, with the f16 weights in mixed-precision multiply-adds. (Weights widened to bf16 for dot products of two take a quarter
// more instructions: one token of 8 of 64 experts 19.3 us, 18.4 so.)
template <int NH>
struct Factors32<true, NH> {
    float v[32];
    __device__ __forceinline__ explicit Factors32(const Elements32 (&a)[NH])
    {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            v[2 * i] = __uint_as_float(a[0].v[i] << 16);
            v[2 * i + 1] = __uint_as_float(a[0].v[i] & 0xffff0000u);
            if constexpr (NH == 2) {
                v[2 * i] += __uint_as_float(a[1].v[i] << 16);
                v[2 * i + 1] += __uint_as_float(a[1].v[i] & 0xffff0000u);
            }
        }
    }
    __device__ __forceinline__ float dot(const half2p_t (&q)[16]) const
    {
        float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            s[i & 1] = fmaf(static_cast<float>(q[i].x), v[2 * i], s[i & 1]);
            s[2 + (i & 1)] = fmaf(static_cast<float>(q[i].y), v[2 * i + 1], s[2 + (i & 1)]);
        }
        return (s[0] + s[1]) + (s[2] + s[3]);
    }
};

// The weights of NU times 64 / LPC columns: load u has column n0 + u (64 / LPC) + lane / LPC, bytes 16 (lane % LPC) on from a pass's begin.
template <typename ST, bool ZP, int NU, int LPC>
struct FewColumns {
    uint4 w[NU];
    typename ScaleIo<ST>::raw_t s[NU];
    uint32_t z[NU];

    // k: the lane's first element. Columns that are not there lie beyond the tile's range and read as zeros; so may, or may not, what lies behind a row, whose
    // activations are zero.
    __device__ __forceinline__ void load(const MoeMatrix& m, const MoeTile<1>& t, int k, int shift)
    {
        const int group = (threadIdx.x & 63) / LPC;
        const uint32_t block = static_cast<uint32_t>(min(k >> shift, m.kb - 1));
        const uint32_t first = static_cast<uint32_t>(group * m.row_step), step = static_cast<uint32_t>(64 / LPC * m.row_step);
        const uint32_t row_bytes = static_cast<uint32_t>(m.row_bytes), kb = static_cast<uint32_t>(m.kb), zp_row = static_cast<uint32_t>(m.zp_row);
        const uint32_t w_at = first * row_bytes + static_cast<uint32_t>(k) / 2, s_at = (first * kb + block) * static_cast<uint32_t>(sizeof(ST)), z_at = first * zp_row + block / 2;
#pragma unroll
        for (int u = 0; u < NU; ++u) {
            w[u] = load16(t.w[0], w_at + u * (step * row_bytes), 0);
            s[u] = ScaleIo<ST>::load_raw(t.s[0], s_at + u * (step * kb * static_cast<uint32_t>(sizeof(ST))), 0);
            if constexpr (ZP) z[u] = __builtin_amdgcn_raw_buffer_load_b8(t.z[0], static_cast<int>(z_at + u * (step * zp_row)), 0, 0);
        }
    }
};

// acc[u] += factor * scale * sum a (q - zp) for NH parts of a row
template <bool BF16, typename ST, bool ZP, int NU, int LPC, int NH>
__device__ __forceinline__ void few_multiply(const Unpacking& by, const FewColumns<ST, ZP, NU, LPC>& c, const Factors32<BF16, NH>& a, int odd, float factor, float (&acc)[NU])
{
#pragma unroll
    for (int u = 0; u < NU; ++u) {
        half2p_t q[16];
        weights32(by, c.w[u], ZP ? (c.z[u] >> odd) & 15u : 8u, q);
        acc[u] = fmaf(factor * ScaleIo<ST>::to_f32(c.s[u], BF16), a.dot(q), acc[u]);
    }
}

// The sum over the LPC lanes of a column, in each of them.
template <int LPC>
__device__ __forceinline__ float over_lanes(float v)
{
    auto add = [](float a, float b) { return a + b; };
    if constexpr (LPC == 64) return over_wave(v, add);
    v = over_row(v, add);
    if constexpr (LPC == 32) {
        const uint32_t bits = __float_as_uint(v);
        const auto s = __builtin_amdgcn_permlane16_swap(bits, bits, false, false);
        v = __uint_as_float(s[0]) + __uint_as_float(s[1]);
    }
    return v;
}

constexpr int kFewRows = 4;

// What is known before the call's other arguments are read: in scalar registers when a wave starts.
#define MOE_FEW_FIRST const void *logits, const uint16_t *x, int logits_dtype, int rows, int experts, int k, int normalize, int width

// A wave has NU times 64 / LPC columns of gate and up of one expert at a time; the tiles of all active experts, one behind the other, go round the waves of the
// grid. The rows of x lie in LDS, in the order of the nibbles, a pass's first eight elements of each lane side by side, then the second eight ..., so that a read
// meets every bank once.
template <bool BF16, typename ST, bool ZP, int LPC>
__global__ __launch_bounds__(256) void moe_few_up_kernel(MOE_FEW_FIRST, MoeUpCall p)
{
    constexpr int NU = 4, kCols = NU * 64 / LPC, kPass = LPC * 32;
    using Columns = FewColumns<ST, ZP, NU, LPC>;
    __shared__ MoeFewRouting routing;
    __shared__ int32_t chose_of[kFewPairs];                              // bit t: token t chose it
    extern __shared__ __attribute__((aligned(16))) uint4 staged[];      // [rows][pass][4][LPC]
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, kl = lane % LPC;
    const int passes = static_cast<unsigned>(width + kPass - 1) / kPass;
    const unsigned pieces = passes * (kPass / 8);
    const bool ranks = ranks_few(rows, experts);
    const float logit = ranks ? few_logit(logits, logits_dtype, rows, experts) : 0.f;
    for (int t = 0; t < rows; ++t)
        for (unsigned piece = threadIdx.x; piece < pieces; piece += 256) {
            const unsigned l = piece / 4;
            const uint4 d = piece * 8 < static_cast<unsigned>(width) ? *reinterpret_cast<const uint4*>(x + static_cast<int64_t>(t) * width + piece * 8) : make_uint4(0, 0, 0, 0);
            staged[((t * passes + l / LPC) * 4 + piece % 4) * LPC + l % LPC] = Elements32::ordered(d);
        }
    if (ranks) rank_few(routing, logit, rows, experts, k, normalize);
    else route_few<4>(routing, logits, logits_dtype, rows, experts, k, normalize);
    if (blockIdx.x == 0) write_table(routing, rows, k, p.table);
    if (rows > 1) {
        for (int i = threadIdx.x; i < routing.active; i += 256) {
            int bits = 0;
            for (int t = 0; t < rows; ++t)
                for (int j = 0; j < k; ++j) bits |= (routing.expert[t * k + j] == routing.chosen[i]) << t;
            chose_of[i] = bits;
        }
        __syncthreads();
    }

    const Unpacking by;
    const int shift = 31 - __builtin_clz(p.m.block_size);
    MoeMatrix up = p.m;
    up.w[0] = p.m.w[1];
    // A unit is a pass over a tile's K. No division: a wave counts its way through units, and an integer division is forty instructions.
    const int tiles = static_cast<int>((static_cast<unsigned>(p.ip) + kCols - 1) / kCols), step = static_cast<int>(gridDim.x) * 4, active = routing.active;
    struct Place {
        int slot, tile, pass;
    };
    auto settle = [&](Place& at) {
        while (at.tile >= tiles) {
            at.tile -= tiles;
            ++at.slot;
        }
    };
    auto next = [&](Place& at) {
        if (++at.pass < passes) return;
        at.pass = 0;
        at.tile += step;
        settle(at);
    };
    Place ahead{0, static_cast<int>(blockIdx.x) * 4 + wave, 0};
    settle(ahead);
    Place now = ahead;
    float g[kFewRows][NU] = {}, u[kFewRows][NU] = {};
    Columns cg[2], cu[2];
    auto load = [&](Columns& to_g, Columns& to_u) {
        const int at = ahead.pass * kPass + kl * 32;
        const bool is = ahead.slot < active;
        const int expert = __builtin_amdgcn_readfirstlane(routing.chosen[is ? ahead.slot : 0]);
        // (a tile of columns behind the last, whose h is zero, reads the last column)
        const int n0 = is ? min(ahead.tile * kCols, p.m.n - 1) : 0, live = is ? min(p.m.n - n0, kCols) : 0;
        to_g.load(p.m, moe_tile<ST, ZP, 1>(p.m, expert, n0, live), at, shift);
        to_u.load(p.m, moe_tile<ST, ZP, 1>(up, expert, n0, live), at, shift);
        next(ahead);
    };
    auto multiply = [&](const Columns& of_g, const Columns& of_u) {
        const int pass = now.pass, slot = now.slot, odd = ((pass * kPass + kl * 32) >> shift & 1) * 4;
        const int chose = rows > 1 ? __builtin_amdgcn_readfirstlane(chose_of[slot]) : 1;
#pragma unroll
        for (int t = 0; t < kFewRows; ++t) {
            if (!(chose >> t & 1)) continue;
            Elements32 a[1];
#pragma unroll
            for (int j = 0; j < 4; ++j) a[0].put(j, staged[((t * passes + pass) * 4 + j) * LPC + kl]);
            const Factors32<BF16, 1> factors(a);
            few_multiply<BF16, ST, ZP, NU, LPC, 1>(by, of_g, factors, odd, 1.f, g[t]);
            few_multiply<BF16, ST, ZP, NU, LPC, 1>(by, of_u, factors, odd, 1.f, u[t]);
        }
        if (pass != static_cast<int>(passes) - 1) return next(now);
        // the tile's sums; lane i of a column's lanes keeps column i's
        const int expert = __builtin_amdgcn_readfirstlane(routing.chosen[slot]), col = now.tile * kCols + kl * (64 / LPC) + lane / LPC;
#pragma unroll
        for (int t = 0; t < kFewRows; ++t) {
            if (!(chose >> t & 1)) continue;
            float gate = 0.f, upv = 0.f;
#pragma unroll
            for (int i = 0; i < NU; ++i) {
                const float a = over_lanes<LPC>(g[t][i]), b = over_lanes<LPC>(u[t][i]);
                if (kl == i) {
                    gate = a;
                    upv = b;
                }
                g[t][i] = u[t][i] = 0.f;
            }
            if (kl < NU && col < p.ip) store_h<BF16>(p, static_cast<int64_t>(slot) * kFewRows + t, col, col < p.m.n ? moe_gated(p, expert, col, gate, upv) : 0.f);
        }
        next(now);
    };
    // two units' loads in flight; those behind the last read nothing (a tile of no columns), but are asked for all the same: a branch would have every load waited for
    if (now.slot >= active) return;
    load(cg[0], cu[0]);
    while (true) {
        load(cg[1], cu[1]);
        multiply(cg[0], cu[0]);
        if (now.slot >= active) break;
        load(cg[0], cu[0]);
        multiply(cg[1], cu[1]);
        if (now.slot >= active) break;
    }
}

// A wave has eight columns and a share of the experts' K; a workgroup's waves have the same columns. An item is one pass over one expert's K; its weights and
// the first row that it meets are asked for one item ahead.
template <bool BF16, typename ST, bool ZP, int LPC>
__global__ __launch_bounds__(512) void moe_few_down_kernel(const MoeFewTable* table, int slots, MoeDownCall p)
{
    constexpr int NU = LPC / 8, kCols = 8, kPass = LPC * 32;
    struct Item {
        FewColumns<ST, ZP, NU, LPC> c;
        Elements32 a[2];
    };
    __shared__ float sums[8][kFewRows][kCols];
    __shared__ float weight[kFewPairs][kFewRows];
    __shared__ int32_t chosen[kFewPairs];
    __shared__ float base[kFewRows];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6, lane = threadIdx.x & 63, kl = lane % LPC;
    if (threadIdx.x < kFewRows) base[threadIdx.x] = table->base[threadIdx.x];
    for (int i = threadIdx.x; i < slots * kFewRows; i += blockDim.x) weight[i / kFewRows][i % kFewRows] = table->weight[i / kFewRows][i % kFewRows];
    for (int i = threadIdx.x; i < slots; i += blockDim.x) chosen[i] = table->expert[i];
    const int active = table->active;
    __syncthreads();
    const Unpacking by;
    const int n0 = static_cast<int>(blockIdx.x) * kCols, live = min(p.m.n - n0, kCols);
    const int shift = 31 - __builtin_clz(p.m.block_size), width = static_cast<int>(p.ip), passes = static_cast<int>(static_cast<unsigned>(width + kPass - 1) / kPass);
    struct Place {
        int slot, pass;
    };
    auto settle = [&](Place& at) {
        while (at.pass >= passes) {
            at.pass -= passes;
            ++at.slot;
        }
    };
    Place ahead{0, wave};
    settle(ahead);
    Place now = ahead;
    float acc[kFewRows][NU] = {};
    auto first_row = [&](int slot) {
        int t = 0;
        while (t < kFewRows - 1 && !(weight[slot][t] > 0.f)) ++t;
        return __builtin_amdgcn_readfirstlane(t);
    };
    auto rows_of = [&](int slot, int t, int at, Elements32 (&a)[2]) {
        const uint16_t* const h = p.h + (static_cast<int64_t>(slot) * kFewRows + t) * (2 * p.ip) + at;
        a[0].load(h, width - at);
        a[1].load(h + p.ip, width - at);
    };
    auto load = [&](Item& to) {
        const bool is = ahead.slot < active;
        const int slot = is ? ahead.slot : 0, at = ahead.pass * kPass + kl * 32;
        to.c.load(p.m, moe_tile<ST, ZP, 1>(p.m, __builtin_amdgcn_readfirstlane(chosen[slot]), n0, is ? live : 0), at, shift);
        rows_of(slot, p.rows > 1 ? first_row(slot) : 0, at, to.a);
        ahead.pass += waves;
        settle(ahead);
    };
    auto multiply = [&](Item& of) {
        const int slot = now.slot, at = now.pass * kPass + kl * 32, odd = (at >> shift & 1) * 4, first = p.rows > 1 ? first_row(slot) : 0;
        now.pass += waves;
        settle(now);
#pragma unroll
        for (int t = 0; t < kFewRows; ++t) {
            const float w = weight[slot][t];
            if (!(w > 0.f)) continue;
            if (t != first) rows_of(slot, t, at, of.a);
            of.a[0].order();
            of.a[1].order();
            few_multiply<BF16, ST, ZP, NU, LPC, 2>(by, of.c, Factors32<BF16, 2>(of.a), odd, w, acc[t]);
        }
    };
    if (now.slot < active) {
        Item one, two;
        load(one);
        while (true) {
            load(two);
            multiply(one);
            if (now.slot >= active) break;
            load(one);
            multiply(two);
            if (now.slot >= active) break;
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
    const int row = static_cast<int>(threadIdx.x) / kCols, col_in = static_cast<int>(threadIdx.x) % kCols;
    if (row >= p.rows || col_in >= live) return;
    float v = base[row];
#pragma unroll
    for (int w = 0; w < 8; ++w) v += w < waves ? sums[w][row][col_in] : 0.f;
    const int64_t col = n0 + col_in;
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
        // each workgroup routes first, which takes it 3 us: no more of them than run at once
        const int64_t waves = slots * ((up.ip + 256 / LPC - 1) / (256 / LPC));
        const unsigned grid = static_cast<unsigned>((waves + 3) / 4 < 2 * rocm_ffi_compute_units() ? (waves + 3) / 4 : 2 * rocm_ffi_compute_units());
        const size_t lds = static_cast<size_t>(up.rows) * ((up.ldx + LPC * 32 - 1) / (LPC * 32)) * (LPC * 64);
        auto kernel = moe_few_up_kernel<decltype(bf)::value, decltype(st), decltype(zp)::value, LPC>;
        hipLaunchKernelGGL(kernel, dim3(grid), dim3(256), lds, s, up.logits, up.x, up.logits_dtype, up.rows, up.experts, up.k, up.normalize,
                           static_cast<int>(up.ldx), up);
        return static_cast<int>(hipGetLastError());
    });
    if (rc != 0) return rc;
    return few_build(a, a.down.zp != nullptr, lanes_per_column(down.ip), [&](auto bf, auto st, auto zp, auto lanes) {
        // (4 tokens, 2048 columns: 47 us with 512 threads, 51 with 256; 1 token, 4096 columns: 56 and 51)
        const unsigned grid = static_cast<unsigned>(down.m.n + 7) / 8, threads = grid <= static_cast<unsigned>(rocm_ffi_compute_units()) ? 512 : 256;
        auto kernel = moe_few_down_kernel<decltype(bf)::value, decltype(st), decltype(zp)::value, decltype(lanes)::value>;
        hipLaunchKernelGGL(kernel, dim3(grid), dim3(threads), 0, s, down.table, slots, down);
        return static_cast<int>(hipGetLastError());
    });
}

}  // namespace mnb
