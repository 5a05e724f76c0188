// QMoE over tiles of 128 pairs of one expert, on v_mfma_f32_32x32x16_f16: by 128 columns of gate and of up, or by 256 of down. For prompts in f16, where the matrix
// cores bound it.
//
// A wave has all rows of the tile and 64 columns of weights that no other wave has (32 of gate beside the same 32 of up), so that it unpacks them for itself, from
// registers into the matrix core; only activations go through LDS, in the order in which a dword's nibbles come out (0 4 1 5 2 6 3 7 of each eight).
// A weight is s (q - zp) in f16, rounded once (and infinite beyond 65504, as it is wherever weights are dequantized to f16). Scaling each block's sum in f32 instead,
// as the other tiles do, takes 64 instructions for each 32 columns of a block beside 64 cycles (blocks of 32) to 256 (of 128) of products, and twice the
// accumulators, which leaves a wave 32 columns and so half as many products for every operand read from LDS. What it costs: y is off by 2.4e-4 of its norm instead
// of 2.2e-4. (In bf16 it would be 3.4e-3 instead of 2.3e-3: those calls keep exact weights.) h is rounded to f16 too, as a graph of separate nodes has it.
//
// A step of 64 k is four parts of 16. While a part's products run, the next one's rows are read and its weights unpacked, the next step's first part among them: its
// activations have been staged by all waves before the last part, the step's only barrier. Loads are a step (activations) or nearly two (weights) ahead.
#include "moe.hiph"
#include "prefill_common.hiph"
#include "rows.hiph"

namespace mnb {
namespace {

constexpr int kTm = 4, kCt = 2;                                          // tiles of 32 rows, and of 32 columns, of a wave

// Elements 0 and 4 of the eight whose nibbles are `bits`: 1024 + q is what a nibble makes of 0x6400, taking 1024 + zp away is exact, the product with s is rounded.
struct Scaled {
    half2p_t scale, off;
    // (The instructions that first touch what was loaded are pinned: the compiler would widen it, and wait for it, a step before.)
    __device__ __forceinline__ void set(uint16_t raw, uint16_t two_zeros, int which)
    {
        uint32_t z, bits;
        asm volatile("v_bfe_u32 %0, %1, %2, 4" : "=v"(z) : "v"(two_zeros), "v"(which));
        asm volatile("v_perm_b32 %0, %1, %1, %2" : "=v"(bits) : "v"(raw), "s"(0x01000100));
        scale = __builtin_bit_cast(half2p_t, bits);
        off = __builtin_bit_cast(half2p_t, 0xE400E400u | (z * 0x00010001u));
    }
    __device__ __forceinline__ uint32_t pair(uint32_t bits, uint32_t mask, uint32_t magic) const
    {
        return __builtin_bit_cast(uint32_t, (__builtin_bit_cast(half2p_t, (bits & mask) | magic) + off) * scale);
    }
};

template <bool UP>
__global__ __launch_bounds__(256, 2) void moe_tall_kernel(MoeTileCall p)
{
    constexpr int kPitch = 9;                                            // pieces of 16 bytes from a row of 64 elements in LDS to the next
    __shared__ uint4 staged[2][kTm * 32 * kPitch];
    const unsigned index = blockIdx.z * gridDim.y + blockIdx.y;
    if (index >= p.count) return;
    const int4 tile = p.tiles[index];
    if (tile.z == 0) return;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = lane & 31, g = lane >> 5;
    const int first_col = UP ? static_cast<int>(blockIdx.x) * 128 + wave * 32 + c : static_cast<int>(blockIdx.x) * 256 + wave * 64 + c;
    const int steps = static_cast<int>(p.ldx) >> 6, last_block = p.m.kb - 1, shift = 31 - __builtin_clz(p.m.block_size), row_bytes = static_cast<int>(p.m.row_bytes);
    const int64_t expert = tile.x * p.m.expert_step;

    // Addresses are scalar bases and 32 bits a lane (the host sees to that); rows and columns that are not there repeat the last.
    const uint8_t *b[kCt], *z[kCt];
    const uint16_t* s[kCt];
    uint32_t column[kCt];
#pragma unroll
    for (int j = 0; j < kCt; ++j) {
        const RocmMoeWeights& w = p.m.w[UP ? j : 0];
        b[j] = w.b + expert * p.m.row_bytes;
        s[j] = static_cast<const uint16_t*>(w.scales) + expert * p.m.kb;
        z[j] = w.zp + expert * p.m.zp_row;
        column[j] = static_cast<uint32_t>(min(UP ? first_col : first_col + j * 32, p.m.n - 1)) * static_cast<uint32_t>(p.m.row_step);
    }
    const int piece = threadIdx.x & 7;
    const uint8_t* const x = reinterpret_cast<const uint8_t*>(p.token ? p.x : p.x + tile.y * p.ldx);
    uint32_t row_at[kTm];
#pragma unroll
    for (int i = 0; i < kTm; ++i) {
        const int row = min(static_cast<int>(threadIdx.x >> 3) + i * 32, tile.z - 1);
        row_at[i] = static_cast<uint32_t>(p.token ? p.token[tile.y + row] : row) * static_cast<uint32_t>(p.ldx * 2) + piece * 16;
    }
    struct Weights {
        uint4 w[kCt];
        uint16_t s[kCt], z[kCt];
    };
    const uint32_t zp_row = static_cast<uint32_t>(p.m.zp_row), kb = static_cast<uint32_t>(p.m.kb);
    auto block_of = [&](int t) { return min((t * 64 + g * 32) >> shift, last_block); };
    auto load_w = [&](int t, Weights& to) {
        const int byte = t * 32 + g * 16;                                // (behind a row's end its activations are zero)
        const uint32_t from = byte < row_bytes ? byte : 0, block = block_of(t);
#pragma unroll
        for (int j = 0; j < kCt; ++j) {
            to.w[j] = *reinterpret_cast<const uint4*>(b[j] + (column[j] * static_cast<uint32_t>(row_bytes) + from));
            to.s[j] = *reinterpret_cast<const uint16_t*>(reinterpret_cast<const uint8_t*>(s[j]) + (column[j] * kb + block) * 2u);
            to.z[j] = z[j][column[j] * zp_row + (block >> 1)];
        }
    };
    uint4 ahead[kTm];
    auto load_x = [&](int t) {
#pragma unroll
        for (int i = 0; i < kTm; ++i) ahead[i] = *reinterpret_cast<const uint4*>(x + (row_at[i] + static_cast<uint32_t>(t) * 128u));
    };
    auto stage = [&](int t, int i) {
        const uint4 d = ahead[i];
        staged[t & 1][((threadIdx.x >> 3) + i * 32) * kPitch + piece] = make_uint4(__builtin_amdgcn_perm(d.z, d.x, 0x05040100u), __builtin_amdgcn_perm(d.z, d.x, 0x07060302u),
                                                                                   __builtin_amdgcn_perm(d.w, d.y, 0x05040100u), __builtin_amdgcn_perm(d.w, d.y, 0x07060302u));
    };
    uint32_t mask = 0x000f000fu;
    asm volatile("" : "+v"(mask));
    const uint32_t magic = opaque_scalar(0x64006400u);

    float16_t total[kTm][kCt] = {};
    uint4 rows[kTm];
    uint32_t weights[2][kCt][4];
    Scaled scaled[kCt];
    auto read = [&](int t, int part, int i) { return staged[t & 1][(i * 32 + c) * kPitch + g * 4 + part]; };
    auto scale = [&](int t, const Weights& from) {
        const int odd = (block_of(t) & 1) * 4;
#pragma unroll
        for (int j = 0; j < kCt; ++j) scaled[j].set(from.s[j], from.z[j], odd);
    };
    auto unpack = [&](int part, int j, int two, const Weights& from) {
        const uint32_t q = part == 0 ? from.w[j].x : part == 1 ? from.w[j].y : part == 2 ? from.w[j].z : from.w[j].w;
        return scaled[j].pair(q >> (4 * two), mask, magic);
    };
    auto step = [&](int t, Weights& now, Weights& next) {
#pragma unroll
        for (int part = 0; part < 4; ++part) {
            if (part == 3) {
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                __builtin_amdgcn_s_barrier();
                asm volatile("" ::: "memory");
                load_w(min(t + 2, steps - 1), now);
                scale(t + 1, next);
            }
            if (part == 1) load_x(min(t + 2, steps - 1));
            __builtin_amdgcn_sched_barrier(0);
            const int coming = (part + 1) & 3;
#pragma unroll
            for (int i = 0; i < kTm; ++i) {
#pragma unroll
                for (int j = 0; j < kCt; ++j) {
                    const uint32_t(&w)[4] = weights[part & 1][j];
                    total[i][j] = mfma32<false>(rows[i], make_uint4(w[0], w[1], w[2], w[3]), total[i][j]);
                }
                rows[i] = read(part == 3 ? t + 1 : t, coming, i);
#pragma unroll
                for (int two = i % 2 * 2; two < i % 2 * 2 + 2; ++two) weights[(part + 1) & 1][i / 2][two] = unpack(coming, i / 2, two, part == 3 ? next : now);
                if (part == 0) stage(t + 1, i);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    };

    Weights one, two;
    load_x(0);
    load_w(0, one);
#pragma unroll
    for (int i = 0; i < kTm; ++i) stage(0, i);
    load_x(min(1, steps - 1));
    load_w(min(1, steps - 1), two);
    __syncthreads();
    scale(0, one);
#pragma unroll
    for (int i = 0; i < kTm; ++i) {
        rows[i] = read(0, 0, i);
#pragma unroll
        for (int q = i % 2 * 2; q < i % 2 * 2 + 2; ++q) weights[0][i / 2][q] = unpack(0, i / 2, q, one);
    }
    for (int t = 0; t + 1 < steps; t += 2) {                             // (a branch between the two would let the compiler move the unpacking behind it)
        step(t, one, two);
        step(t + 1, two, one);
    }
    if (steps & 1) step(steps - 1, one, two);

    // a lane has column c and rows 8 (e / 4) + 4 g + e % 4 of each 32
    auto row_of = [&](int i, int e) { return i * 32 + (e >> 2) * 8 + g * 4 + (e & 3); };
    if constexpr (UP) {
        float bias_g = 0.f, bias_u = 0.f;
        const bool is = first_col < p.m.n;
        if (p.m.w[0].bias && is) {
            const int64_t at = expert + static_cast<int64_t>(column[0]);
            bias_g = load_as_f32(p.m.w[0].bias, p.m.bias_dtype, at);
            bias_u = load_as_f32(p.m.w[1].bias, p.m.bias_dtype, at);
        }
        if (first_col >= p.ldh) return;
#pragma unroll
        for (int i = 0; i < kTm; ++i)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int row = row_of(i, e);
                if (row >= tile.z) continue;
                const float v = is ? moe_activation(total[i][0][e] + bias_g, total[i][1][e] + bias_u, p.alpha, p.beta, p.limit) : 0.f;
                p.h[(tile.y + row) * p.ldh + first_col] = f32_to_f16_bits(v);
            }
    } else {
#pragma unroll
        for (int j = 0; j < kCt; ++j) {
            const int col = first_col + j * 32;
            if (col >= p.m.n) return;
#pragma unroll
            for (int i = 0; i < kTm; ++i)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const int row = row_of(i, e);
                    if (row < tile.z) p.out[static_cast<int64_t>(tile.y + row) * p.m.n + col] = total[i][j][e];
                }
        }
    }
}

}  // namespace

int launch_moe_tall(const MoeTileCall& p, bool up, hipStream_t s)
{
    auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, moe_grid(up ? static_cast<unsigned>((p.ldh + 127) / 128) : static_cast<unsigned>(p.m.n + 255) / 256, static_cast<int>(p.count)), dim3(256), 0, s, p);
        return static_cast<int>(hipGetLastError());
    };
    return up ? go(moe_tall_kernel<true>) : go(moe_tall_kernel<false>);
}

}  // namespace mnb
