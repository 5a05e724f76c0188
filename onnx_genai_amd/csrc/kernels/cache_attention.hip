// CacheAttention over few rows: o = softmax(scale q k^T) v of a sequence's new tokens over its pages, where a key head has up to a few dozen query rows.
//
// The cache's bytes bound it: each is read once for all rows of a tile. A wave takes 64 tokens at a time on its own, straight from memory into the operands of the
// matrix instructions, without LDS. Scores are taken transposed, S^T = K Q^T: 16 tokens (rows) by 16 queries (columns) an instruction, over any order of tokens and of
// head elements as long as both operands agree. So row m of key tile t is token 16 (m / 4) + 4 t + m % 4: a lane then holds the scores of 16 tokens in a row, which is
// what it needs of them as the second operand of O^T = V^T P^T, with 16 tokens of one element a 16-byte load of the values' page. Nothing moves between lanes but
// the maximum of a row. The 16 tokens lie in one page, which holds 16 at least, and their page's scale is one number a lane.
//
// Codes are exact in f16, as 8-bit integers and as e4m3. Queries go to f16 with their row's largest at 2^8 (what falls below f16's range is less than 2^-22 of it).
// Weights p = exp(s - max) become operands as p times the scale of the values' page, relative to the largest such product that the row has seen, in f16: rounded to 11 bits, below 2^-25 of the
// largest to 2^-36 of it. Sums of p itself and all products are in f32.
//
// One token each of 64 sequences of up to 8192, 32 query heads by 8 of 128 (538 MB): 119 to 124 us, 4.3 to 4.5 TB/s. One token after 131071 (268 MB): 55 us with its join, 4.9 TB/s; a GPU-wide copy reaches
// 5.2 TB/s. With little to read the trips to memory count: lengths, table, keys and scales; one token after 1000 takes 9 to 10 us. A tile of 32 rows, which would read a code once for twice the
// rows, was built for heads of up to 128 and left out: it needs more than the 256 registers that two waves a SIMD leave it (32 rows after up to 4000 tokens: 145 us against 99).
#include "cache_attention.hiph"

namespace mnb {
namespace {

constexpr int kWaves = 4, kThreads = 64 * kWaves, kRows = 16;
constexpr int kWhole = 32;                           // groups of 64 tokens below which a context stays whole

// The largest of the four lanes 16 apart, in each of them.
__device__ __forceinline__ float over_groups_max(float v)
{
    const uint32_t a = __float_as_uint(v);
    const auto s = __builtin_amdgcn_permlane16_swap(a, a, false, false);
    v = fmaxf(__uint_as_float(s[0]), __uint_as_float(s[1]));
    const uint32_t b = __float_as_uint(v);
    const auto t = __builtin_amdgcn_permlane32_swap(b, b, false, false);
    return fmaxf(__uint_as_float(t[0]), __uint_as_float(t[1]));
}
__device__ __forceinline__ float over_groups_sum(float v)
{
    const uint32_t a = __float_as_uint(v);
    const auto s = __builtin_amdgcn_permlane16_swap(a, a, false, false);
    v = __uint_as_float(s[0]) + __uint_as_float(s[1]);
    const uint32_t b = __float_as_uint(v);
    const auto t = __builtin_amdgcn_permlane32_swap(b, b, false, false);
    return __uint_as_float(t[0]) + __uint_as_float(t[1]);
}

template <int D>
struct Queries {
    static constexpr int kChunks = (D + 63) / 64;
    half8_t q[kChunks][2];
    float undo;                      // what a score is multiplied by for the row's own scale
    Bytes16 raw[kChunks][2];

    // Row n of lane n, 16 elements from 64 c + 16 g of it in q[c]: asked for first, and looked at when the first keys are on their way.
    __device__ __forceinline__ void ask(const uint16_t* row, int g)
    {
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
            raw[c][0] = raw[c][1] = Bytes16{0, 0, 0, 0};
            if (row && c * 64 + g * 16 < D) {
                raw[c][0] = *reinterpret_cast<const Bytes16*>(row + c * 64 + g * 16);
                raw[c][1] = *reinterpret_cast<const Bytes16*>(row + c * 64 + g * 16 + 8);
            }
        }
    }
    __device__ __forceinline__ void convert(bool bf16)
    {
        float x[kChunks][16];
        float most = 0.f;
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
            const uint32_t d[8] = {raw[c][0].x, raw[c][0].y, raw[c][0].z, raw[c][0].w, raw[c][1].x, raw[c][1].y, raw[c][1].z, raw[c][1].w};
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                x[c][2 * i] = bf16 ? __uint_as_float(d[i] << 16) : f16_bits_to_f32(static_cast<uint16_t>(d[i]));
                x[c][2 * i + 1] = bf16 ? __uint_as_float(d[i] & 0xffff0000u) : f16_bits_to_f32(static_cast<uint16_t>(d[i] >> 16));
                most = fmaxf(most, fmaxf(fabsf(x[c][2 * i]), fabsf(x[c][2 * i + 1])));
            }
        }
        const QueryScale scale(over_groups_max(most));
        undo = scale.undo;
#pragma unroll
        for (int c = 0; c < kChunks; ++c)
#pragma unroll
            for (int i = 0; i < 16; ++i) q[c][i >> 3][i & 7] = static_cast<_Float16>(x[c][i] * scale.factor);
    }
};

template <int D, bool E4M3, int WAVES>
__global__ __launch_bounds__(64 * WAVES, D <= 128 ? 8 / WAVES : 1) void attention_few_kernel(AttentionParams p)
{
    constexpr int kWaves = WAVES, kThreads = 64 * WAVES;
    constexpr int kChunks = (D + 63) / 64, kTiles = D / 16;
    extern __shared__ __attribute__((aligned(16))) float lds[];
    float (*const results)[kRows][D + 4] = reinterpret_cast<float (*)[kRows][D + 4]>(lds);                    // [kWaves]
    float2 (*const sums)[kRows] = reinterpret_cast<float2 (*)[kRows]>(lds + kWaves * kRows * (D + 4));         // [kWaves]
    const RocmCache& c = p.a.cache;
    Piece w;
    if (!piece_at(p, blockIdx.x, &w)) return;
    const int head = w.head;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n = lane & 15, g = lane >> 4;
    const int context = context_of(c, w.s);

    // the lane's query row
    const int first_row = w.tile * kRows, rows = w.s.rows * p.group - first_row < kRows ? w.s.rows * p.group - first_row : kRows;
    const int token = p.by_group.of(first_row + n), member = first_row + n - token * p.group;
    const int own = w.s.past + token;                                        // the row's own slot
    const bool row_there = n < rows;
    const uint16_t* const q_row = static_cast<const uint16_t*>(p.a.q) + static_cast<int64_t>(w.s.first + token) * p.a.q_step + (head * p.group + member) * D;
    Queries<D> q;
    // tokens that every row of the tile sees, and those that some row does
    const int first_own = w.s.past + p.by_group.of(first_row), last_own = w.s.past + p.by_group.of(first_row + rows - 1);
    const int window = p.a.window;

    float4_t o[kTiles];
#pragma unroll
    for (int u = 0; u < kTiles; ++u) o[u] = float4_t{0.f, 0.f, 0.f, 0.f};
    float top = kNone, sum = 0.f, reference = kNone;         // reference: log2 of the product that operands are relative to

    // The page of 16 tokens of a step: sub-block n / 4 for the lane's keys, g for its values and scales. A step's entries of the table are asked for a step before its keys.
    const int page_bits = __builtin_ctz(c.page);
    const int32_t* const table = c.table + static_cast<int64_t>(w.b) * c.width;
    int key_entry = 0, value_entry = 0;
    auto ask = [&](int group) {
        key_entry = entry_of(c, table, page_bits, group * kGroup + (n >> 2) * 16);
        value_entry = entry_of(c, table, page_bits, group * kGroup + g * 16);
    };
    struct Step {
        uint4 k[4][kChunks], v[kTiles];
        float ks, vs;
        int live;                                    // tokens of sub-block g that there are
    };
    const int64_t page_bytes = static_cast<int64_t>(c.page) * D;
    const uint8_t *const k_base = static_cast<const uint8_t*>(c.k), *const v_base = static_cast<const uint8_t*>(c.v);
    auto load_keys = [&](int group, int page, Step& s) {
        const int64_t at = (static_cast<int64_t>(page < 0 ? 0 : page) * c.kv_heads + head) * page_bytes;
        const int slot = ((group * kGroup + (n >> 2) * 16) & (c.page - 1)) + (n & 3);
        const uint8_t* const from = k_base + at + slot * D + g * 16;
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int i = 0; i < kChunks; ++i) {
                s.k[t][i] = make_uint4(0, 0, 0, 0);
                if (D % 64 == 0 || i * 64 + g * 16 < D) s.k[t][i] = *reinterpret_cast<const uint4*>(from + t * 4 * D + i * 64);
            }
    };
    auto load_values = [&](int group, int page, Step& s) {
        const int64_t index = static_cast<int64_t>(page < 0 ? 0 : page) * c.kv_heads + head;
        const uint8_t* const from = v_base + index * page_bytes + n * c.page + ((group * kGroup + g * 16) & (c.page - 1));
#pragma unroll
        for (int u = 0; u < kTiles; ++u) s.v[u] = *reinterpret_cast<const uint4*>(from + u * 16 * c.page);
    };
    auto load_scales = [&](int group, int page, Step& s) {
        const int64_t index = static_cast<int64_t>(page < 0 ? 0 : page) * c.kv_heads + head;
        s.ks = c.k_scale[index];
        s.vs = c.v_scale[index];
        s.live = page < 0 ? 0 : clamped(context - (group * kGroup + g * 16), 0, 16);
    };

    Step s;
    int at = w.span.lo + wave, value_page = -1;
    auto find = [&](int group) {
        value_page = page_from(c, value_entry, group * kGroup + g * 16, context);
        return page_from(c, key_entry, group * kGroup + (n >> 2) * 16, context);
    };
    if (at < w.span.hi) ask(at);
    q.ask(row_there ? q_row : nullptr, g);
    if (at < w.span.hi) {
        load_keys(at, find(at), s);
        load_scales(at, value_page, s);
        ask(at + kWaves);
        load_values(at, value_page, s);
    }
    q.convert(p.a.dtype == ROCM_DT_BF16);
    const float row_scale = q.undo * p.scale;
    for (; at < w.span.hi; at += kWaves) {
        const int t0 = at * kGroup;
        // scores: lane (n, g) gets token t0 + 16 g + 4 t + i of row n in score[t][i]
        float4_t score[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            score[t] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < kChunks; ++i) {
                half8_t lo, hi;
                widen<E4M3>(s.k[t][i], lo, hi);
                score[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(lo, q.q[i][0], score[t], 0, 0, 0);
                score[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(hi, q.q[i][1], score[t], 0, 0, 0);
            }
        }
        const int live = s.live;
        const float key_scale = s.ks * row_scale, value_scale = s.vs;
        // the next step's keys, scales and page numbers while this one goes on
        const bool more = at + kWaves < w.span.hi;
        if (more) {
            load_keys(at + kWaves, find(at + kWaves), s);
            load_scales(at + kWaves, value_page, s);
            ask(at + 2 * kWaves);
        }
        float x[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) x[e] = score[e >> 2][e & 3] * key_scale;
        if (p.a.softcap > 0.f) {
#pragma unroll
            for (int e = 0; e < 16; ++e) x[e] = capped(x[e], p.a.softcap, p.cap_inverse);
        }
        // where some row does not see some token: bit e of `seen` for the lane's row and token e of its
        const bool partial = __ballot(live < 16) != 0, masked = partial || t0 + kGroup - 1 > first_own || (window > 0 && t0 <= last_own - window);
        uint32_t seen = 0;
        if (masked) {
            const int here = t0 + g * 16;
            const int end = clamped(own - here + 1, 0, live), begin = window > 0 ? clamped(own - window + 1 - here, 0, 16) : 0;
            seen = ((1u << end) - 1u) & ~((1u << begin) - 1u);
#pragma unroll
            for (int e = 0; e < 16; ++e) x[e] = (seen >> e) & 1 ? x[e] : kNone;
        }
        float most = x[0];
#pragma unroll
        for (int e = 1; e < 16; ++e) most = fmaxf(most, x[e]);
        // (the scale's power of two, which is below it by less than a bit, will do; a scale of 0 or NaN, and what the row does not see, have no part in it)
        const float product = value_scale > 0.f ? most + static_cast<float>(__builtin_amdgcn_frexp_expf(value_scale) - 1) : kNone;
        most = fmaxf(top, over_groups_max(most));
        const float next = fmaxf(reference, over_groups_max(product));
        // What weights and operands are relative to stays until something is kSlack bits above it: sums and values are seldom scaled again.
        if (__ballot(most > top + kSlack || next > reference + (kSlack - 1.f))) {
            const float shrink = __builtin_amdgcn_exp2f(top - (most == kNone ? 0.f : most));
            const float again = __builtin_amdgcn_exp2f(reference - (next == kNone ? 0.f : next));
            sum *= shrink;
            top = most;
            reference = next;
#pragma unroll
            for (int u = 0; u < kTiles; ++u) o[u] *= again;
        }
        const float zero = top == kNone ? 0.f : top;                            // (a row that has seen nothing yet)
        // what makes a weight an operand; a NaN stays one. In two steps, as 2^(zero - reference) alone may be beyond f32, and the whole of it for a page whose weights are next to nothing
        const float step = __builtin_amdgcn_exp2f(reference == kNone ? 0.f : fminf(0.5f * (zero - reference), 120.f)), product_of_one = value_scale * step * step;
        const float relative = product_of_one > 3e38f ? 3e38f : product_of_one;
        half8_t weights[2];
        auto weigh = [&](auto some) {
            float part = 0.f;
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                float y = __builtin_amdgcn_exp2f(x[e] - (zero - kWeightBits)), weight = y * relative;
                if constexpr (decltype(some)::value) {
                    y = (seen >> e) & 1 ? y : 0.f;
                    weight = (seen >> e) & 1 ? weight : 0.f;
                }
                part += y;
                weights[e >> 3][e & 7] = static_cast<_Float16>(weight);
            }
            sum += part;
        };
        if (masked) weigh(std::true_type{});
        else weigh(std::false_type{});
        if (partial) {
            // what lies behind the context may be anything
            uint32_t keep[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int left = live - 4 * j;
                keep[j] = left >= 4 ? 0xffffffffu : left <= 0 ? 0u : 0xffffffffu >> (32 - 8 * left);
            }
#pragma unroll
            for (int u = 0; u < kTiles; ++u) s.v[u] = make_uint4(s.v[u].x & keep[0], s.v[u].y & keep[1], s.v[u].z & keep[2], s.v[u].w & keep[3]);
        }
#pragma unroll
        for (int u = 0; u < kTiles; ++u) {
            half8_t lo, hi;
            widen<E4M3>(s.v[u], lo, hi);
            o[u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(lo, weights[0], o[u], 0, 0, 0);
            o[u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(hi, weights[1], o[u], 0, 0, 0);
        }
        if (more) load_values(at + kWaves, value_page, s);
    }

    // the waves' results, means of what each has seen, which no value is beyond: o[u][i] is element 16 u + 4 g + i of row n
    sum = over_groups_sum(sum);
    const float own_inverse = sum == 0.f ? 0.f : 1.0f / sum, back = reference == kNone ? 0.f : __builtin_amdgcn_exp2f(0.5f * (reference - top));
#pragma unroll
    for (int u = 0; u < kTiles; ++u) *reinterpret_cast<float4_t*>(&results[wave][n][u * 16 + g * 4]) = o[u] * own_inverse * back * back;
    if (g == 0) sums[wave][n] = make_float2(top, sum);
    __syncthreads();
    constexpr int kQuads = D / 4;
    const int64_t out_step = static_cast<int64_t>(p.a.heads) * D;
    for (int i = threadIdx.x; i < rows * kQuads; i += kThreads) {
        const int row = i / kQuads, e = (i - row * kQuads) * 4;
        float most = kNone;
#pragma unroll
        for (int j = 0; j < kWaves; ++j) most = fmaxf(most, sums[j][row].x);
        const float zero = most == kNone ? 0.f : most;
        float total = 0.f, share[kWaves];
#pragma unroll
        for (int j = 0; j < kWaves; ++j) {
            share[j] = sums[j][row].y * __builtin_amdgcn_exp2f(sums[j][row].x - zero);
            total += share[j];
        }
        // a row that sees nothing is zero
        const float inverse = total == 0.f ? 0.f : 1.0f / total;
        float4_t all = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < kWaves; ++j) all += *reinterpret_cast<const float4_t*>(&results[j][row][e]) * (share[j] * inverse);
        if (w.slot >= 0) {
            const int64_t place = (static_cast<int64_t>(w.slot) * c.kv_heads + head) * kRows + row;
            *reinterpret_cast<float4_t*>(p.partial + place * D + e) = all;
            if (e == 0) p.partial_sums[place] = make_float2(most, total);
        } else {
            const int r = first_row + row, tk = p.by_group.of(r);
            uint16_t* const to = static_cast<uint16_t*>(p.a.y) + static_cast<int64_t>(w.s.first + tk) * out_step + (head * p.group + r - tk * p.group) * D + e;
            store_four(to, all[0], all[1], all[2], all[3], p.a.dtype);
        }
    }
}

// The pieces of a tile joined, in an order that is always the same. A workgroup has some rows of it; what a piece counts for in a row is found first, by a wave over the pieces
// of a row, so that the sums over the pieces wait for nothing but their loads.
constexpr int kMostPieces = 1025;                    // of a tile: the target and one more
__global__ __launch_bounds__(kThreads, 6) void attention_join_kernel(AttentionParams p, int d, int rows_at_once)
{
    extern __shared__ __attribute__((aligned(16))) float shares[];      // [rows_at_once][pieces], then [threads][4]
    const RocmCache& c = p.a.cache;
    const int head = blockIdx.x % c.kv_heads;
    Piece w;
    if (!tile_to_join(p, p.by_heads.of(blockIdx.x), &w)) return;
    const int first_row = w.tile * p.tile_rows, left = w.s.rows * p.group - first_row, rows = left < p.tile_rows ? left : p.tile_rows;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t piece_step = static_cast<int64_t>(c.kv_heads) * p.tile_rows, first = (static_cast<int64_t>(w.slot) * c.kv_heads + head) * p.tile_rows;
    // a group of d / 4 threads has a row's elements, four each, over every so many pieces; the first of them are on their way before anything is known of their shares
    const int quads = d / 4, groups = kThreads / quads, each = groups / rows_at_once;
    const int group = threadIdx.x / quads, quad = threadIdx.x - group * quads, r = group / each, part = group - r * each;
    float4_t* const sums = reinterpret_cast<float4_t*>(shares + (rows_at_once * w.pieces + 3) / 4 * 4);
    for (int row0 = blockIdx.y * rows_at_once; row0 < rows; row0 += gridDim.y * rows_at_once) {
        const bool busy = r < rows_at_once && row0 + r < rows;
        const float* const from = p.partial + (first + row0 + (busy ? r : 0)) * d + quad * 4;
        constexpr int kEarly = 4;
        float4_t early[kEarly];
#pragma unroll
        for (int j = 0; j < kEarly; ++j) {
            const int i = part + j * each;
            early[j] = float4_t{0.f, 0.f, 0.f, 0.f};
            if (busy && i < w.pieces) early[j] = *reinterpret_cast<const float4_t*>(from + i * piece_step * d);
        }
        for (int k = wave; k < rows_at_once; k += kWaves) {
            const int row = row0 + k < rows ? row0 + k : rows - 1;
            float most = kNone;
            for (int i = lane; i < w.pieces; i += 64) most = fmaxf(most, p.partial_sums[first + i * piece_step + row].x);
            most = over_wave(most, [](float x, float y) { return fmaxf(x, y); });
            const float zero = most == kNone ? 0.f : most;
            float sum = 0.f;
            for (int i = lane; i < w.pieces; i += 64) {
                const float2 s = p.partial_sums[first + i * piece_step + row];
                const float share = s.y * __builtin_amdgcn_exp2f(s.x - zero);
                sum += share;
                shares[k * w.pieces + i] = share;
            }
            sum = over_wave(sum, [](float x, float y) { return x + y; });
            const float inverse = sum == 0.f ? 0.f : 1.0f / sum;
            for (int i = lane; i < w.pieces; i += 64) shares[k * w.pieces + i] *= inverse;
        }
        __syncthreads();
        float4_t all = {0.f, 0.f, 0.f, 0.f};
        if (busy) {
            const float* const share = shares + r * w.pieces;
#pragma unroll
            for (int j = 0; j < kEarly; ++j)
                if (part + j * each < w.pieces) all += early[j] * share[part + j * each];
#pragma unroll 4
            for (int i = part + kEarly * each; i < w.pieces; i += each) {
                const float4_t v = *reinterpret_cast<const float4_t*>(from + i * piece_step * d);
                const float f = share[i];
                all += v * f;
            }
        }
        sums[threadIdx.x] = all;
        __syncthreads();
        if (busy && part == 0) {
            for (int i = 1; i < each; ++i) all += sums[threadIdx.x + i * quads];
            const int row = first_row + row0 + r, tk = p.by_group.of(row);
            store_four(static_cast<uint16_t*>(p.a.y) + (static_cast<int64_t>(w.s.first + tk) * p.a.heads + head * p.group + row - tk * p.group) * d + quad * 4, all[0], all[1], all[2], all[3], p.a.dtype);
        }
    }
}

struct Plan {
    bool ok, many;
    int tile_rows, target, least, whole, teams, most;
    int64_t tiles, pieces;          // most that a call of these sizes has, for one key head
    uint64_t sums_at, bytes;
};

Plan plan_of(const RocmCacheAttentionArgs& a)
{
    Plan plan{};
    const RocmCache& c = a.cache;
    if (a.rows <= 0 || c.sequences <= 0 || c.kv_heads < 1 || a.heads < c.kv_heads || a.heads % c.kv_heads != 0 || !rocm_cache_attention_supports(c.head_size) || a.rows >= (1 << 30) || c.page < 16 ||
        c.page > ROCM_CACHE_MAX_PAGE || (c.page & (c.page - 1)) != 0 || c.width < 1 || static_cast<int64_t>(c.width) * c.page >= (1 << 30))
        return plan;
    const int group = a.heads / c.kv_heads;
    if (a.rows * group >= (1 << 30)) return plan;
    const int64_t cus = rocm_ffi_compute_units(), per_head = a.rows * group, capacity = static_cast<int64_t>(c.width) * c.page;
    const bool small = c.head_size <= 128;
    // Beyond 64 rows a sequence, on average, tiles of many rows share what they read of the cache through LDS, (16 sequences of up to 4000 tokens, 64 rows a key head: 48 us in tiles of
    // 16, 65 us in one of 128; 64 such sequences with 128 rows: 139 and 117 us), unless there is little to do: where contexts are short or tiles few, a tile's own steps are what a call
    // waits for, and tiles of 16 deal them out to more waves. That holds for up to four tiles of 16 for each CU (two with heads of 256, one of which fills a CU) where contexts stay whole,
    // and for so much work in all where they are cut. (Prompts of 256 tokens, 32 heads by 8: 11 us in tiles of 16, 17 us in tiles of 128; 1000 tokens in a window of 1024, 14 heads of 64 by 2:
    // 20 and 32 us; but 1024 tokens, 32 by 8: 49 and 32 us. 128 tokens after 3000: 25 and 36 us, after 6000: 45 and 38 us, after 16000: 95 and 59 us. Heads of 256, 64 tokens after 5000: 44 and
    // 72 us, 256 tokens: 107 and 78 us.)
    const int64_t fine = (per_head + kRows - 1) / kRows * c.kv_heads, seen = a.window > 0 && a.window < capacity ? a.window : capacity, busy = (small ? 2 : 1) * cus;
    const bool little = fine <= 2 * busy && (seen <= kGroup * kWhole || fine * seen <= 3000 * busy);
    plan.many = per_head > 64 * static_cast<int64_t>(c.sequences) && !little;
    plan.tile_rows = plan.many ? kManyRows : kRows;
    // 256 rows a tile, which halves what a row costs of the codes' way into LDS, once that gives two tiles for each CU; 128 rows with two teams of waves, which halves the steps that follow one
    // another, where there is no more than one tile for each CU. (4096 tokens over 32 heads by 8: 175 us, in tiles of 128 206 us; 2400 new tokens, 28 by 4: 54 us, with two teams
    // 68 us; 700 tokens, 32 by 32 heads of 80: 32 us with two teams, 43 us with one.)
    if (plan.many && small && per_head * c.kv_heads >= 2 * kMostRows * cus) plan.tile_rows = kMostRows;
    plan.tiles = per_head / plan.tile_rows + (a.rows < c.sequences ? a.rows : c.sequences);
    // Few rows: eight waves a tile instead of four, by the same rule. (16 sequences, 16 rows a key head, 8 of them: 31 us, with four waves 33 us; with 64 rows, four tiles a head: 57 and 48 us.)
    const int64_t busy_sequences = a.rows < c.sequences ? a.rows : c.sequences, full_tiles = per_head / plan.tile_rows, filled = full_tiles > busy_sequences ? full_tiles : busy_sequences;
    plan.teams = small && filled * c.kv_heads <= cus ? 2 : 1;
    // Pieces until there are as many workgroups as fit on the GPU at once: two for each CU, or one of 512 threads or heads of 256. None is shorter than 512 tokens, or 1024 in tiles of
    // many rows, and contexts below 2048 stay whole: joining pieces costs about what so many tokens take. (One token after 1000: 9 us whole, 13 us in two pieces; four tokens after 4000
    // with heads of 256: 31 us in pieces of 512 and more, 44 us in pieces of 1024 and more.)
    const int64_t at_once = plan.teams == 2 || plan.tile_rows == kMostRows || !small ? cus : 2 * cus;
    int64_t wanted = at_once / c.kv_heads;
    if (wanted > kMostPieces - 1) wanted = kMostPieces - 1;
    plan.least = plan.many ? 16 : 8;
    plan.whole = kWhole;
    // what a window lets the rows of a tile see (one more token than its rows have: it may begin inside a token's heads)
    const int64_t tokens = (plan.tile_rows + group - 1) / group + 1;
    plan.most = a.window > 0 ? static_cast<int>((a.window + tokens + kGroup - 2) / kGroup + 1) : 1 << 24;
    if (filled < wanted && capacity > kGroup * (kWhole - 1) && plan.most >= kWhole) plan.target = static_cast<int>(wanted);
    plan.pieces = plan.tiles + plan.target;
    const uint64_t places = 2 * static_cast<uint64_t>(plan.target) * c.kv_heads * plan.tile_rows;
    plan.sums_at = (places * c.head_size * 4 + 255) / 256 * 256;
    plan.bytes = plan.target ? plan.sums_at + (places * 8 + 255) / 256 * 256 : 0;
    plan.ok = plan.pieces * c.kv_heads < (1 << 23);          // (a grid has fewer than 2^32 threads, a workgroup up to 512)
    return plan;
}

template <int D, bool E4M3, int WAVES>
hipError_t launch_tiles(const AttentionParams& p, dim3 grid, hipStream_t s)
{
    constexpr size_t kLds = WAVES * kRows * ((D + 4) * 4 + 8);
    const auto kernel = attention_few_kernel<D, E4M3, WAVES>;
    if (kLds > 65536) {              // more than a kernel gets without asking
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kLds));
        if (e != hipSuccess) return e;
    }
    hipLaunchKernelGGL(kernel, grid, dim3(64 * WAVES), kLds, s, p);
    return hipGetLastError();
}

template <bool E4M3>
hipError_t launch_few(const AttentionParams& p, dim3 grid, hipStream_t s)
{
    auto sized = [&](auto size) {
        constexpr int D = decltype(size)::value;
        return p.teams == 2 ? launch_tiles<D, E4M3, 8>(p, grid, s) : launch_tiles<D, E4M3, 4>(p, grid, s);
    };
    switch (p.a.cache.head_size) {
        case 64: return sized(std::integral_constant<int, 64>{});
        case 80: return sized(std::integral_constant<int, 80>{});
        case 96: return sized(std::integral_constant<int, 96>{});
        case 128: return sized(std::integral_constant<int, 128>{});
        case 256: return p.teams == 2 ? hipErrorInvalidValue : launch_tiles<256, E4M3, 4>(p, grid, s);
        default: return hipErrorInvalidValue;
    }
}

}  // namespace
}  // namespace mnb

extern "C" int rocm_cache_attention_supports(int head_size) { return head_size == 64 || head_size == 80 || head_size == 96 || head_size == 128 || head_size == 256; }

extern "C" uint64_t rocm_cache_attention_workspace_bytes(const RocmCacheAttentionArgs* args) { return mnb::plan_of(*args).bytes; }

extern "C" const char* rocm_cache_attention_variant(const RocmCacheAttentionArgs* args)
{
    const mnb::Plan plan = mnb::plan_of(*args);
    return plan.many ? plan.target ? "cache_attention_rows_pieces" : "cache_attention_rows" : plan.target ? "cache_attention_pieces" : "cache_attention";
}

extern "C" int rocm_launch_cache_attention(const RocmCacheAttentionArgs* args, void* workspace, rocm_stream_t stream)
{
    using namespace mnb;
    if (args->rows <= 0 || args->cache.sequences <= 0) return 0;
    const Plan plan = plan_of(*args);
    if (!plan.ok || (plan.bytes && !workspace)) return static_cast<int>(hipErrorInvalidValue);
    hipStream_t s = static_cast<hipStream_t>(stream);
    AttentionParams p{};
    p.a = *args;
    p.group = args->heads / args->cache.kv_heads;
    p.tile_rows = plan.tile_rows;
    p.tile_bits = __builtin_ctz(plan.tile_rows);
    p.by_group = Divisor(p.group);
    p.by_heads = Divisor(args->cache.kv_heads);
    p.target = plan.target;
    p.least_bits = __builtin_ctz(plan.least);
    p.most = plan.most;
    p.whole = plan.whole;
    p.teams = plan.teams;
    p.slots = 2 * plan.target;
    p.cap_inverse = args->softcap > 0.f ? 1.0f / args->softcap : 0.f;
    p.scale = args->softcap > 0.f ? args->scale : args->scale * 1.442695041f;
    p.partial = static_cast<float*>(workspace);
    p.partial_sums = reinterpret_cast<float2*>(static_cast<uint8_t*>(workspace) + plan.sums_at);
    const dim3 grid(static_cast<unsigned>(plan.pieces * args->cache.kv_heads));
    hipError_t e = plan.many ? launch_attention_rows(p, grid, s) : args->cache.code_dtype == ROCM_DT_E4M3 ? launch_few<true>(p, grid, s) : launch_few<false>(p, grid, s);
    if (e == hipSuccess && plan.target) {
        // A row's pieces are many where there are few tiles: then all groups of threads have one row, else two groups each.
        const int d = args->cache.head_size, groups = kThreads / (d / 4), rows = plan.tiles <= 2 ? 1 : groups / 2;
        // a few workgroups for each CU, which go on to further rows: most tiles may have nothing to join
        const int64_t all = plan.tiles * args->cache.kv_heads, most = (plan.tile_rows + rows - 1) / rows, wanted = (8 * static_cast<int64_t>(rocm_ffi_compute_units()) + all - 1) / all;
        const unsigned lds = static_cast<unsigned>((rows * (plan.target + 1) + 3) / 4 * 16 + kThreads * 16);
        hipLaunchKernelGGL(attention_join_kernel, dim3(static_cast<unsigned>(all), static_cast<unsigned>(wanted < most ? wanted : most)), dim3(kThreads), lds, s, p, d, rows);
        e = hipGetLastError();
    }
    return static_cast<int>(e);
}
