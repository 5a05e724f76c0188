// CacheAttention over many rows: prompts and chunks of them.
//
// A workgroup has 128 rows, or 256, 32 a wave, and goes through the tokens 64 at a time: the codes are read once for all rows, become f16 on their way into LDS
// (exactly), and are read from there as operands. As over few rows the scores are taken transposed, S^T = K Q^T, 32 tokens by 32 rows an instruction, with the tokens of a
// key tile in the order in which a lane's scores are the weights that it has to hand in for O^T = V^T P^T: row m of the instruction is token 16 (m / 16) + 8 ((m / 4) % 2) +
// 4 ((m / 8) % 2) + m % 4. Keys lie in LDS a token a row, values an element a row, rows 16 bytes apart more than their data, which spreads 16 rows over all banks.
// While a step is computed, the next one's codes are on their way into registers; they go to the other half of LDS behind it.
//
// A page's scales are numbers of 16 tokens each here, and stay out of the products over single scores: key scales enter a score's one multiply-add, value scales its exponent,
// operand = 2^(score + log2(scale) - reference), and their inverse the sum of 8 operands. The reference is the largest score + log2(scale) that a row has seen, so operands are rounded as over few rows.
//
// 8192 tokens, 32 query heads by 8 of 128, each token after those before it: 595 to 605 us, 910 to 925 TFLOP/s; the library's product of f16 matrices reaches 1150. What is left are the vector
// instructions of the softmax, about as many cycles as the products and hardly overlapped with them, since a wave's products wait for its own weights: their issue alone is four fifths of the time.
// On the way: 16 rows a workgroup 1891 us, 128 rows 926, a path of its own for steps without masks 700, table entries a step ahead 688, reads out of LDS six products ahead 650, 256 rows 587;
// operands relative to what a row sees, and not to pages that it does not, 597.
#include "cache_attention.hiph"

namespace mnb {
namespace {

constexpr int kWaveRows = 32;
constexpr float kLeastShare = 60.f;          // bits by which a page's largest operands may lie below the reference: what is further below, and so 0 in f16, counts as this, for the sum's sake
constexpr float kLeastBits = -1000.f;        // log2 of a scale of 0

typedef __attribute__((ext_vector_type(16))) float float16_t;
typedef __attribute__((ext_vector_type(4))) float float4_t;

// The order of N matrix instructions and the reads out of LDS of an operand each: reads stay kAhead in front, which covers what a read takes.
constexpr int kAhead = 6;
template <int N>
__device__ __forceinline__ void reads_ahead()
{
    constexpr int kMatrix = 0x008, kRead = 0x100, kFirst = N < kAhead ? N : kAhead;
    __builtin_amdgcn_sched_group_barrier(kRead, kFirst, 0);
#pragma unroll
    for (int i = 0; i < N - kFirst; ++i) {
        __builtin_amdgcn_sched_group_barrier(kMatrix, 1, 0);
        __builtin_amdgcn_sched_group_barrier(kRead, 1, 0);
    }
    __builtin_amdgcn_sched_group_barrier(kMatrix, kFirst, 0);
}

template <int D>
struct Tile {
    static constexpr int kKeyPitch = D * 2 + 16, kValuePitch = kGroup * 2 + 16, kValueRows = (D + 31) / 32 * 32;
    alignas(16) uint8_t k[kGroup * kKeyPitch];
    alignas(16) uint8_t v[kValueRows * kValuePitch];
    float key_scale[4], value_bits[4];       // of 16 tokens each; log2 of the values' scale
    int there[4];
};

// WIDE: pages of 64 tokens or more, so that a step lies in one.
// TEAMS 2: two teams of waves over the same rows, each every other step, their results joined in LDS: where there are few workgroups, half as many steps follow one another.
template <int D, bool E4M3, bool WIDE, int WAVES, int TEAMS>
__global__ __launch_bounds__(64 * WAVES * TEAMS, D <= 128 ? 8 / (WAVES * TEAMS) : 1) void attention_rows_kernel(AttentionParams p)
{
    constexpr int kThreads = 64 * WAVES, kRows = WAVES * kWaveRows;
    constexpr int kSteps = D / 16, kOut = (D + 31) / 32, kPieces = 4 * D, kEach = (kPieces + kThreads - 1) / kThreads;
    constexpr int kPages = WIDE ? 1 : 4;                         // that a step's scales are of
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    Tile<D>* const tiles = reinterpret_cast<Tile<D>*>(lds);
    const RocmCache& c = p.a.cache;
    Piece w;
    if (!piece_at(p, blockIdx.x, &w)) return;
    const int head = w.head;
    const int team = TEAMS > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x / kThreads) : 0, thread = threadIdx.x - team * kThreads;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(thread >> 6);
    const int n = lane & 31, h = lane >> 5;
    const int context = context_of(c, w.s);
    const bool bf16 = p.a.dtype == ROCM_DT_BF16;

    // the lane's query row: half h has the elements 16 i + 8 h of it
    const int first_row = w.tile * kRows + wave * kWaveRows, left = w.s.rows * p.group - first_row, rows = left < kWaveRows ? left : kWaveRows;
    const int token = p.by_group.of(first_row + n), member = first_row + n - token * p.group;
    const int own = w.s.past + token, last_seen = own < context ? own : context - 1;
    Bytes16 raw[kSteps];
    {
        const uint16_t* const row = static_cast<const uint16_t*>(p.a.q) + static_cast<int64_t>(w.s.first + token) * p.a.q_step + (head * p.group + member) * D + 8 * h;
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            raw[i] = Bytes16{0, 0, 0, 0};
            if (n < rows) raw[i] = *reinterpret_cast<const Bytes16*>(row + 16 * i);
        }
    }
    // tokens that every row of the wave sees, and those that some row does
    const int first_own = w.s.past + p.by_group.of(first_row), last_own = w.s.past + p.by_group.of(first_row + (rows > 0 ? rows : 1) - 1);
    const int window = p.a.window;

    const int page_bits = __builtin_ctz(c.page);
    const int64_t page_bytes = static_cast<int64_t>(c.page) * D;
    // A thread's 16-byte pieces of a step. Keys: piece i is 16 elements of token i / (D / 16). Values: 16 tokens of an element; of a wide page piece i is of element i / 4 and tokens
    // 16 (i % 4) on, 64 bytes of an element together; else of element i % D and tokens 16 (i / D) on, so that a piece of keys and one of values are of the same 16 tokens, and
    // with D a multiple of 64, all of a wave's pieces.
    constexpr bool kOneOfWave = WIDE || D % 64 == 0;
    uint4 keys[kEach], values[kEach];
    const int32_t* const table = c.table + static_cast<int64_t>(w.b) * c.width;
    int entries[kEach], scale_entry = 0;                         // of the table, for the step to be loaded next: asked for a step ahead, looked at when it begins
    int pages[kEach], scale_page = -1;                           // -1: none
    float key_scale = 0.f, value_scale = 0.f;
    auto sub_of = [&](int j) {
        const int i = thread + j * kThreads;
        if constexpr (WIDE) return static_cast<int>(thread & 3);
        else if constexpr (kOneOfWave) return (wave * 64 + j * kThreads) / D;
        else return i / D & 3;
    };
    auto ask = [&](int group) {
        if constexpr (!WIDE) {
#pragma unroll
            for (int j = 0; j < kEach; ++j) entries[j] = entry_of(c, table, page_bits, group * kGroup + sub_of(j) * 16);
        }
        scale_entry = entry_of(c, table, page_bits, group * kGroup + (WIDE ? 0 : thread & 3) * 16);
    };
    auto find_pages = [&](int group) {
        scale_page = page_from(c, scale_entry, group * kGroup + (WIDE ? 0 : thread & 3) * 16, context);
        if constexpr (WIDE) {
            scale_page = __builtin_amdgcn_readfirstlane(scale_page);
        } else {
#pragma unroll
            for (int j = 0; j < kEach; ++j) {
                pages[j] = page_from(c, entries[j], group * kGroup + sub_of(j) * 16, context);
                if constexpr (kOneOfWave) pages[j] = __builtin_amdgcn_readfirstlane(pages[j]);
            }
        }
    };
    auto load = [&](int group) {
#pragma unroll
        for (int j = 0; j < kEach; ++j) {
            const int i = thread + j * kThreads;
            if (kPieces % kThreads == 0 || i < kPieces) {
                const int page = WIDE ? scale_page : pages[j], sub = WIDE ? 0 : sub_of(j), skip = (group * kGroup + sub * 16) & (c.page - 1);
                const int64_t at = (static_cast<int64_t>(page < 0 ? 0 : page) * c.kv_heads + head) * page_bytes;
                const uint32_t within = static_cast<uint32_t>(i - sub * D);
                keys[j] = *reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(c.k) + at + skip * D + within * 16);
                values[j] = *reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(c.v) + at + skip + (WIDE ? (within >> 2) * static_cast<uint32_t>(c.page) + (within & 3) * 16 : within * static_cast<uint32_t>(c.page)));
            }
        }
        if (thread < kPages) {
            const int64_t at = static_cast<int64_t>(scale_page < 0 ? 0 : scale_page) * c.kv_heads + head;
            key_scale = c.k_scale[at];
            value_scale = c.v_scale[at];
        }
    };
    // `there`: bit j, the page of the thread's pieces j was one; of_scale: that of its scales was
    auto store = [&](int group, Tile<D>& tile, uint32_t there, bool of_scale) {
#pragma unroll
        for (int j = 0; j < kEach; ++j) {
            const int i = thread + j * kThreads, sub = sub_of(j);
            const int live = (there >> j) & 1 ? clamped(context - (group * kGroup + sub * 16), 0, 16) : 0;
            if (WIDE ? !(there & 1) || (group + 1) * kGroup > context : __ballot(live < 16) != 0) {
                // what lies behind the context may be anything
                uint32_t* const d = &values[j].x;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int l = live - 4 * e;
                    d[e] &= l >= 4 ? 0xffffffffu : l <= 0 ? 0u : 0xffffffffu >> (32 - 8 * l);
                }
            }
            if (kPieces % kThreads == 0 || i < kPieces) {
                const int t = i / (D / 16), col = i - t * (D / 16);
                half8_t lo, hi;
                widen<E4M3>(keys[j], lo, hi);
                half8_t* const k = reinterpret_cast<half8_t*>(tile.k + t * Tile<D>::kKeyPitch + col * 32);
                k[0] = lo;
                k[1] = hi;
                widen<E4M3>(values[j], lo, hi);
                half8_t* const v = reinterpret_cast<half8_t*>(tile.v + (WIDE ? i >> 2 : i - sub * D) * Tile<D>::kValuePitch + sub * 32);
                v[0] = lo;
                v[1] = hi;
            }
        }
        if (thread < kPages) {
            tile.key_scale[thread] = key_scale;
            // (the logarithm knows normal numbers only; one of NaN stays one)
            const bool low = value_scale < 5.42101086e-20f;
            const float bits = __builtin_amdgcn_logf(low ? value_scale * 18446744073709551616.f : value_scale) - (low ? 64.f : 0.f);
            tile.value_bits[thread] = !of_scale || bits < kLeastBits ? kLeastBits : bits;
            tile.there[thread] = of_scale;
        }
    };
    auto are_there = [&]() {
        if constexpr (WIDE) return scale_page >= 0 ? ~0u : 0u;
        uint32_t bits = 0;
#pragma unroll
        for (int j = 0; j < kEach; ++j) bits |= pages[j] >= 0 ? 1u << j : 0u;
        return bits;
    };

    // the first step's codes are on their way while the queries become operands
    Tile<D>* const mine = tiles + 2 * team;
    const int begin = w.span.lo + team;
    if (begin < w.span.hi) {
        ask(begin);
        find_pages(begin);
        load(begin);
    }
    half8_t q[kSteps];
    float row_scale;
    {
        auto get = [&](int i, float (&x)[8]) {
            const uint32_t d[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                x[2 * j] = bf16 ? __uint_as_float(d[j] << 16) : f16_bits_to_f32(static_cast<uint16_t>(d[j]));
                x[2 * j + 1] = bf16 ? __uint_as_float(d[j] & 0xffff0000u) : f16_bits_to_f32(static_cast<uint16_t>(d[j] >> 16));
            }
        };
        float most = 0.f;
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            float x[8];
            get(i, x);
#pragma unroll
            for (int j = 0; j < 8; ++j) most = fmaxf(most, fabsf(x[j]));
        }
        most = fmaxf(most, __shfl_xor(most, 32, 64));
        const QueryScale scale(most);
        row_scale = scale.undo * p.scale;
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            float x[8];
            get(i, x);
#pragma unroll
            for (int j = 0; j < 8; ++j) q[i][j] = static_cast<_Float16>(x[j] * scale.factor);
        }
    }

    float16_t o[kOut];
#pragma unroll
    for (int u = 0; u < kOut; ++u)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[u][i] = 0.f;
    float top = kNone, sum = 0.f, reference = kNone;

    if (begin < w.span.hi) {
        ask(begin + TEAMS);
        store(begin, mine[0], are_there(), scale_page >= 0);
    }
    for (int at = begin, turn = 0; at - team < w.span.hi; at += TEAMS, turn ^= 1) {
        __syncthreads();
        const Tile<D>& tile = mine[turn];
        const bool more = at + TEAMS < w.span.hi;
        if (more) {
            find_pages(at + TEAMS);
            load(at + TEAMS);
            ask(at + 2 * TEAMS);
        }
        const int t0 = at * kGroup;
        const bool skipped = rows <= 0 || at >= w.span.hi || t0 > last_own || (window > 0 && t0 + kGroup - 1 <= first_own - window);
        if (!skipped) {
            // scores: lane (n, h) gets token 16 s + 8 h + j of row n in score[s / 2][8 (s % 2) + j]
            float16_t score[2];
            const int order = 16 * (n >> 4) + 8 * ((n >> 2) & 1) + 4 * ((n >> 3) & 1) + (n & 3);
            const uint8_t* const key = tile.k + order * Tile<D>::kKeyPitch + h * 16;
#pragma unroll
            for (int i = 0; i < 16; ++i) score[0][i] = score[1][i] = 0.f;
#pragma unroll
            for (int i = 0; i < kSteps; ++i)
#pragma unroll
                for (int b = 0; b < 2; ++b)
                    score[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(*reinterpret_cast<const half8_t*>(key + b * 32 * Tile<D>::kKeyPitch + i * 32), q[i], score[b], 0, 0, 0);
            reads_ahead<2 * kSteps>();
            float ks[kPages], bits[kPages];
            int there = 15;
#pragma unroll
            for (int s = 0; s < kPages; ++s) {
                ks[s] = tile.key_scale[s] * row_scale;
                bits[s] = tile.value_bits[s];
                there &= tile.there[s] ? 15 : WIDE ? 0 : 15 ^ (1 << s);
            }
            if (p.a.softcap > 0.f) {
#pragma unroll
                for (int s = 0; s < 4; ++s)
#pragma unroll
                    for (int j = 0; j < 8; ++j) score[s >> 1][8 * (s & 1) + j] = capped(score[s >> 1][8 * (s & 1) + j] * ks[s % kPages], p.a.softcap, p.cap_inverse);
#pragma unroll
                for (int s = 0; s < kPages; ++s) ks[s] = 1.f;
            }
            // where some row of the wave does not see some token: bit 8 s + j of `seen` for the lane's row and its tokens
            const bool masked = there != 15 || t0 + kGroup - 1 > first_own || t0 + kGroup > context || (window > 0 && t0 <= last_own - window);
            uint32_t seen = 0;
            if (masked) {
                const int hi = last_seen - t0 - 8 * h, lo = window > 0 ? own - window + 1 - t0 - 8 * h : -8;
#pragma unroll
                for (int s = 0; s < 4; ++s) {
                    const int end = clamped(hi + 1 - 16 * s, 0, 8), begin = clamped(lo - 16 * s, 0, 8);
                    if ((there >> s) & 1) seen |= (((1u << end) - 1u) & ~((1u << begin) - 1u)) << (8 * s);
                }
#pragma unroll
                for (int e = 0; e < 32; ++e) score[e >> 4][e & 15] = (seen >> e) & 1 ? score[e >> 4][e & 15] : kNone;
            }
            float most = top, next = reference;
#pragma unroll
            for (int s = 0; s < 4; s += 4 / kPages) {
                float m = score[s >> 1][8 * (s & 1)];
#pragma unroll
                for (int e = 8 * s + 1; e < 8 * s + 32 / kPages; ++e) m = fmaxf(m, score[e >> 4][e & 15]);
                most = fmaxf(most, m * ks[s % kPages]);
                next = fmaxf(next, fmaf(m, ks[s % kPages], bits[s % kPages]));
            }
            {
                const uint32_t a = __float_as_uint(most), b = __float_as_uint(next);
                const auto r = __builtin_amdgcn_permlane32_swap(a, a, false, false), q = __builtin_amdgcn_permlane32_swap(b, b, false, false);
                most = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
                next = fmaxf(__uint_as_float(q[0]), __uint_as_float(q[1]));
            }
            // What sums and operands are relative to stays until something is kSlack bits above it: sums and values are seldom scaled again.
            if (__ballot(most > top + kSlack || next > reference + kSlack)) {
                const float shrink = __builtin_amdgcn_exp2f(top - (most == kNone ? 0.f : most));
                const float again = __builtin_amdgcn_exp2f(reference - (next == kNone ? 0.f : next));
                sum *= shrink;
                top = most;
                reference = next;
#pragma unroll
                for (int u = 0; u < kOut; ++u) o[u] *= again;
            }
            const float zero = top == kNone ? 0.f : top, behind = reference == kNone ? 0.f : zero - reference;          // (a row that has seen nothing yet)
            half8_t weights[4];
            auto weigh = [&](auto some) {
#pragma unroll
                for (int s = 0; s < 4; s += 4 / kPages) {
                    // (a NaN scale stays one)
                    const float all = bits[s % kPages] + behind, share = all < -kLeastShare ? -kLeastShare : all;
                    const float off = zero - kWeightBits - share;
                    float part = 0.f;
#pragma unroll
                    for (int e = 8 * s; e < 8 * s + 32 / kPages; ++e) {
                        float y = __builtin_amdgcn_exp2f(fmaf(score[e >> 4][e & 15], ks[s % kPages], -off));
                        if constexpr (decltype(some)::value) y = (seen >> e) & 1 ? y : 0.f;
                        part += y;
                        weights[e >> 3][e & 7] = static_cast<_Float16>(y);
                    }
                    sum = fmaf(part, fminf(__builtin_amdgcn_exp2f(-share), 1152921504606846976.f), sum);          // (no row's sum is NaN for a page that it does not see)
                }
            };
            if (masked) weigh(std::true_type{});
            else weigh(std::false_type{});
            const uint8_t* const from = tile.v + n * Tile<D>::kValuePitch + h * 16;
#pragma unroll
            for (int s = 0; s < 4; ++s)
#pragma unroll
                for (int u = 0; u < kOut; ++u)
                    o[u] = __builtin_amdgcn_mfma_f32_32x32x16_f16(*reinterpret_cast<const half8_t*>(from + u * 32 * Tile<D>::kValuePitch + s * 32), weights[s], o[u], 0, 0, 0);
            reads_ahead<4 * kOut>();
        }
        if (more) store(at + TEAMS, mine[turn ^ 1], are_there(), scale_page >= 0);
    }

    // o[u][4 a + i] is element 32 u + 8 a + 4 h + i of row n; from here on a mean of what the row has seen, which no value is beyond. A row that sees nothing is zero.
    sum += __shfl_xor(sum, 32, 64);
    {
        const float inverse = sum == 0.f ? 0.f : 1.0f / sum, back = reference == kNone ? 0.f : __builtin_amdgcn_exp2f(0.5f * (reference - top));          // (by halves: either may be beyond f32)
#pragma unroll
        for (int u = 0; u < kOut; ++u) o[u] = o[u] * inverse * back * back;
    }
    if constexpr (TEAMS > 1) {
        // the second team's results through LDS, where its tiles were: four elements a lane, lanes side by side
        float* const other = reinterpret_cast<float*>(tiles) + wave * (kOut * 16 + 2) * 64 + lane;
        __syncthreads();
        if (team == 1) {
#pragma unroll
            for (int u = 0; u < kOut; ++u)
#pragma unroll
                for (int i = 0; i < 16; ++i) other[(u * 16 + i) * 64] = o[u][i];
            other[kOut * 16 * 64] = top;
            other[(kOut * 16 + 1) * 64] = sum;
        }
        __syncthreads();
        if (team == 1) return;
        const float their_top = other[kOut * 16 * 64], most = fmaxf(top, their_top), zero = most == kNone ? 0.f : most;
        float ours = sum * __builtin_amdgcn_exp2f(top - zero), theirs = other[(kOut * 16 + 1) * 64] * __builtin_amdgcn_exp2f(their_top - zero);
        sum = ours + theirs;
        top = most;
        const float inverse = sum == 0.f ? 0.f : 1.0f / sum;
        ours *= inverse;
        theirs *= inverse;
#pragma unroll
        for (int u = 0; u < kOut; ++u)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[u][i] = o[u][i] * ours + other[(u * 16 + i) * 64] * theirs;
    }
    if (n >= rows) return;
    if (w.slot >= 0) {
        const int64_t place = (static_cast<int64_t>(w.slot) * c.kv_heads + head) * kRows + wave * kWaveRows + n;
#pragma unroll
        for (int u = 0; u < kOut; ++u)
#pragma unroll
            for (int a = 0; a < 4; ++a) {
                const int e = u * 32 + a * 8 + h * 4;
                if (D % 32 == 0 || e < D) *reinterpret_cast<float4_t*>(p.partial + place * D + e) = float4_t{o[u][4 * a], o[u][4 * a + 1], o[u][4 * a + 2], o[u][4 * a + 3]};
            }
        if (h == 0) p.partial_sums[place] = make_float2(top, sum);
    } else {
        uint16_t* const to = static_cast<uint16_t*>(p.a.y) + (static_cast<int64_t>(w.s.first + token) * p.a.heads + head * p.group + member) * D;
#pragma unroll
        for (int u = 0; u < kOut; ++u)
#pragma unroll
            for (int a = 0; a < 4; ++a) {
                const int e = u * 32 + a * 8 + h * 4;
                if (D % 32 == 0 || e < D) store_four(to + e, o[u][4 * a], o[u][4 * a + 1], o[u][4 * a + 2], o[u][4 * a + 3], p.a.dtype);
            }
    }
}

template <int D, bool E4M3, bool WIDE, int WAVES, int TEAMS>
hipError_t launch(const AttentionParams& p, dim3 grid, hipStream_t s)
{
    constexpr size_t kLds = 2 * TEAMS * sizeof(Tile<D>);
    static_assert(TEAMS == 1 || kLds >= static_cast<size_t>(WAVES) * ((D + 31) / 32 * 16 + 2) * 256, "room for a team's results");
    const auto kernel = attention_rows_kernel<D, E4M3, WIDE, WAVES, TEAMS>;
    if (kLds > 65536) {              // more than a kernel gets without asking
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kLds));
        if (e != hipSuccess) return e;
    }
    hipLaunchKernelGGL(kernel, grid, dim3(64 * WAVES * TEAMS), kLds, s, p);
    return hipGetLastError();
}

template <bool E4M3, bool WIDE>
hipError_t launch_of(const AttentionParams& p, dim3 grid, hipStream_t s)
{
    const bool most = p.tile_rows == kMostRows;
    if ((!most && p.tile_rows != kManyRows) || (p.teams != 1 && (most || p.teams != 2))) return hipErrorInvalidValue;
    auto sized = [&](auto size) {
        constexpr int D = decltype(size)::value;
        return most ? launch<D, E4M3, WIDE, 8, 1>(p, grid, s) : p.teams == 2 ? launch<D, E4M3, WIDE, 4, 2>(p, grid, s) : launch<D, E4M3, WIDE, 4, 1>(p, grid, s);
    };
    switch (p.a.cache.head_size) {
        case 64: return sized(std::integral_constant<int, 64>{});
        case 80: return sized(std::integral_constant<int, 80>{});
        case 96: return sized(std::integral_constant<int, 96>{});
        case 128: return sized(std::integral_constant<int, 128>{});
        case 256: return most || p.teams == 2 ? hipErrorInvalidValue : launch<256, E4M3, WIDE, 4, 1>(p, grid, s);
        default: return hipErrorInvalidValue;
    }
}

}  // namespace

hipError_t launch_attention_rows(const AttentionParams& p, dim3 grid, hipStream_t stream)
{
    const bool wide = p.a.cache.page >= kGroup;
    if (p.a.cache.code_dtype == ROCM_DT_E4M3) return wide ? launch_of<true, true>(p, grid, stream) : launch_of<true, false>(p, grid, stream);
    return wide ? launch_of<false, true>(p, grid, stream) : launch_of<false, false>(p, grid, stream);
}

}  // namespace mnb
