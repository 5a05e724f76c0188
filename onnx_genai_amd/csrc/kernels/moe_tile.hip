// QMoE over tiles of pairs sorted by expert, on v_mfma_f32_32x32x16_{f16,bf16}: 32 TM rows by 64 columns of gate and of up, or by 128 of down.
//
// A wave has all rows of the tile and 32 columns of weights that no other wave has (16 of gate beside 16 of up), so that it unpacks them for itself, from
// registers into the matrix core; only activations go through LDS, in the order in which a dword's nibbles come out (0 4 1 5 2 6 3 7 of each eight).
// Weights enter the matrix core as q - zp, which is exact in 16 bits, and each block's sum is scaled in f32: no weight is rounded.
// TM = 4 (prompts): 64 vector instructions scale a block's sums and 44 (bf16: 76) unpack 64 k beside 512 cycles of products. Neither unit is at its limit: of the SIMDs'
// cycles vector instructions take 59 % up and 47 % down in bf16 with blocks of 128, products 39 and 34 %; in f16 with blocks of 32, 63 and 53 %, 32 and 29 %. The shares
// add up to 81 to 98 %: two waves a SIMD, which meet at a barrier every 64 k, overlap the two little. TM = 1 (a few rows an expert): the weights' bytes, and a CU's path to memory, where 64 columns' scales take as long as
// their weights.
// Measured: TM = 1, 48 tokens of 8 out of 64 experts of 2048 and 1024, blocks of 64, 52 us up and 28 down (2.7 TB/s); TM = 4, 4096 tokens of those, blocks of 128, 405 us
// up and 222 down (0.68 and 0.62 PFLOP/s at 1.9 GHz), 777 tokens of 4 out of 16 experts of 2880, f16,
// blocks of 32, 230 us up and 121 down (0.45 and 0.43 PFLOP/s; its tiles are 128 and 66 rows, a quarter of them absent). With a step's reads and unpacking in front of
// its products, as the compiler places them, those were 414, 223, 252 and 142.
// Weights rounded to 16 bits before the product save the scaling and half of the accumulators, so that a wave has 64 columns (777 tokens: 191 us up and 124 down; 4096
// tokens in bf16: 349 and 188), and put y off by up to twice its own rounding: they stay exact.
// h is rounded to the activations' type here (as a graph of separate nodes has it): a second part of it would be half again as many products in the second half.
#include "moe.hiph"
#include "prefill_common.hiph"
#include "rows.hiph"

namespace mnb {
namespace {

// Nibbles 0 and 4 of `bits` as q - zp: plain_nibbles for two of its eight.
template <bool BF16>
__device__ __forceinline__ uint32_t tile_pair(uint32_t bits, uint32_t z, uint32_t mask, uint32_t magic)
{
    const half2p_t h = __builtin_bit_cast(half2p_t, (bits & mask) | magic);
    if constexpr (BF16) {
        const float off = -1024.0f - static_cast<float>(z);
        float one = 1.0f;
        asm("" : "+v"(one));                                   // (a factor the compiler knows to be one would make it a conversion and an add)
        return __builtin_amdgcn_perm(__float_as_uint(fmaf(static_cast<float>(h.y), one, off)), __float_as_uint(fmaf(static_cast<float>(h.x), one, off)), 0x07060302u);
    } else {
        return __builtin_bit_cast(uint32_t, h + __builtin_bit_cast(half2p_t, 0xE400E400u | (z * 0x00010001u)));
    }
}

template <bool BF16, int BS, typename ST, bool UP, int TM>
__global__ __launch_bounds__(256, TM == 4 ? 2 : 4) void moe_tile_kernel(MoeTileCall p)
{
    constexpr int kPitch = 9;                                            // pieces of 16 bytes from a row of 64 elements in LDS to the next
    __shared__ uint4 staged[2][TM * 32 * kPitch];
    // (slices of down's K along z; without them z goes on where y ends)
    const unsigned slice = !UP && p.slices > 1 ? blockIdx.z : 0u, index = (slice ? 0u : blockIdx.z) * gridDim.y + blockIdx.y;
    if (index >= p.count) return;
    const int4 tile = p.tiles[index];
    if (tile.z == 0) return;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = lane & 31, g = lane >> 5;
    const int col = UP ? static_cast<int>(blockIdx.x) * 64 + wave * 16 + (c & 15) : static_cast<int>(blockIdx.x) * 128 + wave * 32 + c;
    const int which = UP ? c >> 4 : 0;
    const int64_t at = tile.x * p.m.expert_step + static_cast<int64_t>(min(col, p.m.n - 1)) * p.m.row_step;       // (columns that are not there repeat the last)
    const uint8_t* const b = (which ? p.m.w[1].b : p.m.w[0].b) + at * p.m.row_bytes;
    const ST* const s = static_cast<const ST*>(which ? p.m.w[1].scales : p.m.w[0].scales) + at * p.m.kb;
    const uint8_t* const z = (which ? p.m.w[1].zp : p.m.w[0].zp) + at * p.m.zp_row;
    const int from = UP ? 0 : static_cast<int>(slice) * p.steps_per_slice, all_steps = static_cast<int>(p.ldx) >> 6;
    const int steps = UP || p.slices == 1 ? all_steps : min(from + p.steps_per_slice, all_steps);             // where the slice ends
    const int shift = 31 - __builtin_clz(p.m.block_size), row_bytes = static_cast<int>(p.m.row_bytes), last_block = p.m.kb - 1;

    const int piece = threadIdx.x & 7;
    const uint16_t* x[TM];
#pragma unroll
    for (int i = 0; i < TM; ++i) {
        const int64_t row = tile.y + min(static_cast<int>(threadIdx.x >> 3) + i * 32, tile.z - 1);                // (nor are rows)
        x[i] = p.x + (p.token ? p.token[row] : row) * p.ldx + piece * 8;
    }
    auto load_w = [&](int t, uint4& to) {
        const int byte = t * 32 + g * 16;
        to = *reinterpret_cast<const uint4*>(b + (byte < row_bytes ? byte : 0));                                  // (behind a row's end its activations are zero)
    };
    // Scales of two blocks at once, one in each lane group, and their zero points: 32 columns' scales take a CU's path to memory as long as their weights of a step,
    // however few bytes they are. (Two steps are one block of 128.)
    struct Scales {
        ST s;
        uint16_t z;
    };
    auto load_s = [&](int t, Scales& to) {
        const int block = t * 64 >> shift;
        to.s = s[min(block + (BS == 128 ? 0 : g), last_block)];
        to.z = z[min(block, last_block) >> 1];
    };
    uint4 ahead[TM];
    auto load_x = [&](int t) {
#pragma unroll
        for (int i = 0; i < TM; ++i) ahead[i] = *reinterpret_cast<const uint4*>(x[i] + t * 64);
    };
    auto stage = [&](int t, int i) {
        const uint4 d = ahead[i];
        staged[t & 1][((threadIdx.x >> 3) + i * 32) * kPitch + piece] = make_uint4(__builtin_amdgcn_perm(d.z, d.x, 0x05040100u), __builtin_amdgcn_perm(d.z, d.x, 0x07060302u),
                                                                                   __builtin_amdgcn_perm(d.w, d.y, 0x05040100u), __builtin_amdgcn_perm(d.w, d.y, 0x07060302u));
    };
    uint32_t mask = 0x000f000fu;
    asm volatile("" : "+v"(mask));
    const uint32_t magic = opaque_scalar(0x64006400u);

    float16_t total[TM] = {}, sum[TM] = {};
    const float16_t none = {};
    // (The instructions that first touch what was loaded are pinned: the compiler would widen it, and wait for it, a step before.)
    float scale[2];
    uint32_t zero[2];
    auto take = [&](int t, const Scales& from) {
        uint32_t v;
        if constexpr (sizeof(ST) == 4) v = __float_as_uint(from.s);
        else if constexpr (BF16) asm volatile("v_lshlrev_b32 %0, 16, %1" : "=v"(v) : "v"(from.s));
        else asm volatile("v_cvt_f32_f16 %0, %1" : "=v"(v) : "v"(from.s));
        if constexpr (BS == 128) {
            scale[0] = scale[1] = __uint_as_float(v);
            asm volatile("v_bfe_u32 %0, %1, %2, 4" : "=v"(zero[0]) : "v"(from.z), "s"((min(t * 64 >> shift, last_block) & 1) * 4));
            zero[1] = zero[0];
        } else {
            const auto both = __builtin_amdgcn_permlane32_swap(v, v, false, false);
            scale[0] = __uint_as_float(both[0]);
            scale[1] = __uint_as_float(both[1]);
            asm volatile("v_bfe_u32 %0, %1, 0, 4" : "=v"(zero[0]) : "v"(from.z));
            asm volatile("v_bfe_u32 %0, %1, 4, 4" : "=v"(zero[1]) : "v"(from.z));
        }
    };
    // A step is four parts of 16 k. Behind a part's product of 32 rows come the next part's read of them and a share of its weights' unpacking, so that they run beside
    // the products; the last part's come from the next step, whose activations all waves have staged by then: the step's only barrier. A block's sum is scaled where
    // the next block's first product overwrites it.
    uint4 rows[TM];
    uint32_t weights[2][4];
    float pending = 0.f;                                                 // the scale of the block whose sum this is
    auto read = [&](int t, int part, int i) { return staged[t & 1][(i * 32 + c) * kPitch + (BS == 32 ? part * 2 + g : g * 4 + part)]; };
    // BS 32: lane group h has block h; afterwards x and y hold block 0 of both groups, z and w block 1
    auto arrange = [&](uint4& w) {
        if constexpr (BS == 32) {
            const auto lo = __builtin_amdgcn_permlane32_swap(w.x, w.y, false, false), hi = __builtin_amdgcn_permlane32_swap(w.z, w.w, false, false);
            w = make_uint4(lo[0], hi[0], lo[1], hi[1]);
        }
    };
    auto unpack = [&](const uint4& w, int part, int two, uint32_t zp) {
        const uint32_t q = part == 0 ? w.x : part == 1 ? w.y : part == 2 ? w.z : w.w;
        return tile_pair<BF16>(q >> (4 * two), zp, mask, magic);
    };
    // FIRST: the step begins a block (of 64 or more). which: its scale, next_which: that of the next step, whose scales are taken before the last part.
    auto step = [&](int t, uint4& now, uint4& next, int which, int next_which, bool first, auto take_next) {
        float of_block[2] = {BS == 32 ? scale[0] : scale[which], scale[1]};
        uint32_t zp = BS == 32 ? zero[0] : zero[which], zp1 = zero[1];
#pragma unroll
        for (int part = 0; part < 4; ++part) {
            if (part == 3) {
                take_next();
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                __builtin_amdgcn_s_barrier();
                asm volatile("" ::: "memory");
                load_w(min(t + 2, steps - 1), now);
                arrange(next);
            }
            if (part == 1) load_x(min(t + 2, steps - 1));
            __builtin_amdgcn_sched_barrier(0);
            const bool begins = BS == 32 ? part % 2 == 0 : part == 0 && first;
            const float done = pending;
            if (begins) pending = of_block[part / 2];
            const int coming = (part + 1) & 3;
            const uint32_t coming_zp = part == 3 ? (BS == 32 ? zero[0] : zero[next_which]) : BS == 32 && part >= 1 ? zp1 : zp;
#pragma unroll
            for (int i = 0; i < TM; ++i) {
                if (begins)
#pragma unroll
                    for (int e = 0; e < 16; ++e) total[i][e] = fmaf(done, sum[i][e], total[i][e]);
                const uint32_t(&w)[4] = weights[part & 1];
                sum[i] = mfma32<BF16>(rows[i], make_uint4(w[0], w[1], w[2], w[3]), begins ? none : sum[i]);
                rows[i] = read(part == 3 ? t + 1 : t, coming, i);
#pragma unroll
                for (int two = i * 4 / TM; two < (i + 1) * 4 / TM; ++two) weights[(part + 1) & 1][two] = unpack(part == 3 ? next : now, coming, two, coming_zp);
                if (part == 0) stage(t + 1, i);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    };

    uint4 one, two_w;
    Scales sa, sb;                                                       // (blocks of 32: of a step each; else sa of both)
    load_x(from);
    load_s(from, sa);
    load_w(from, one);
    if (BS == 32) load_s(from + 1, sb);
    load_w(min(from + 1, steps - 1), two_w);
#pragma unroll
    for (int i = 0; i < TM; ++i) stage(from, i);
    load_x(min(from + 1, steps - 1));
    __syncthreads();
    take(from, sa);
    load_s(from + 2, sa);
    arrange(one);
#pragma unroll
    for (int i = 0; i < TM; ++i) rows[i] = read(from, 0, i);
#pragma unroll
    for (int two = 0; two < 4; ++two) weights[0][two] = unpack(one, 0, two, zero[0]);
    auto none_taken = [] {};
    int t = from;                                                        // (even)
    for (; t + 2 <= steps; t += 2) {                                     // (with a branch between the two the compiler waits for all loads there)
        if constexpr (BS == 32) {
            step(t, one, two_w, 0, 0, true, [&] {
                take(t + 1, sb);
                load_s(t + 3, sb);
            });
        } else {
            step(t, one, two_w, 0, 1, true, none_taken);
        }
        step(t + 1, two_w, one, 1, 0, BS != 128, [&] {
            take(t + 2, sa);
            load_s(t + 4, sa);
        });
    }
    if (t < steps) step(t, one, two_w, 0, 0, true, none_taken);
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) total[i][e] = fmaf(pending, sum[i][e], total[i][e]);

    // a lane has column c and rows 8 (e / 4) + 4 g + e % 4 of each 32
    auto row_of = [&](int i, int e) { return i * 32 + (e >> 2) * 8 + g * 4 + (e & 3); };
    if constexpr (UP) {
        float bias_g = 0.f, bias_u = 0.f;
        const bool is = col < p.m.n;
        if (p.m.w[0].bias && is) {
            bias_g = load_as_f32(p.m.w[0].bias, p.m.bias_dtype, at);
            bias_u = load_as_f32(p.m.w[1].bias, p.m.bias_dtype, at);
        }
        // lanes with gate take the even rows, lanes with up the odd ones
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int e = 0; e < 16; e += 2) {
                const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(total[i][e]), __float_as_uint(total[i][e]), false, false);
                const auto o = __builtin_amdgcn_permlane16_swap(__float_as_uint(total[i][e + 1]), __float_as_uint(total[i][e + 1]), false, false);
                const float gate = __uint_as_float(which ? o[0] : a[0]) + bias_g, up = __uint_as_float(which ? o[1] : a[1]) + bias_u;
                const int row = row_of(i, e + which);
                if (row >= tile.z || col >= p.ldh) continue;
                const float v = is ? moe_activation(gate, up, p.alpha, p.beta, p.limit) : 0.f;
                p.h[(tile.y + row) * p.ldh + col] = BF16 ? f32_to_bf16_bits(v) : f32_to_f16_bits(v);
            }
    } else {
        if (col >= p.m.n) return;
        float* const out = p.out + slice * p.slice_elements;
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int row = row_of(i, e);
                if (row < tile.z) out[static_cast<int64_t>(tile.y + row) * p.m.n + col] = total[i][e];
            }
    }
}

}  // namespace

int launch_moe_tile(const RocmMoeArgs& a, const MoeTileCall& p, bool up, int tile_rows, hipStream_t s)
{
    auto go = [&](auto bf, auto bs, auto st, auto half) {
        constexpr bool BF16 = decltype(bf)::value, UP = decltype(half)::value;
        constexpr int BS = decltype(bs)::value;
        using ST = decltype(st);
        dim3 grid = moe_grid(UP ? static_cast<unsigned>((p.ldh + 63) / 64) : static_cast<unsigned>(p.m.n + 127) / 128, static_cast<int>(p.count));
        if (!UP && p.slices > 1) grid.z = static_cast<unsigned>(p.slices);
        if (tile_rows == 128) hipLaunchKernelGGL((moe_tile_kernel<BF16, BS, ST, UP, 4>), grid, dim3(256), 0, s, p);
        else hipLaunchKernelGGL((moe_tile_kernel<BF16, BS, ST, UP, 1>), grid, dim3(256), 0, s, p);
        return static_cast<int>(hipGetLastError());
    };
    auto halved = [&](auto bf, auto bs, auto st) { return up ? go(bf, bs, st, std::true_type{}) : go(bf, bs, st, std::false_type{}); };
    auto scaled = [&](auto bf, auto bs) { return a.scale_dtype == ROCM_DT_F32 ? halved(bf, bs, float{}) : halved(bf, bs, uint16_t{}); };
    auto typed = [&](auto bf) {
        if (a.block_size == 32) return scaled(bf, std::integral_constant<int, 32>{});
        if (a.block_size == 64) return scaled(bf, std::integral_constant<int, 64>{});
        return scaled(bf, std::integral_constant<int, 128>{});
    };
    return a.dtype == ROCM_DT_BF16 ? typed(std::true_type{}) : typed(std::false_type{});
}

}  // namespace mnb
