// QMoE: which launches a call is.
//
//   up to 4 tokens      gate/up (every workgroup routes for itself), down with the sum over experts
//   more                top-k and sorting by expert (one launch up to 64 tokens, then two), gate/up, down, sum over each token's experts
#include "moe.hiph"

namespace mnb {
namespace {

// Pairs an expert from which tiles have 128 rows. us of a call in tiles of 32 and of 128: 16 experts of 2880, f16: 25 pairs 127 and 198, 38 pairs 223 and 197, 62 pairs 294
// and 207; 8 experts of 4096 and 14336, f16: 24 pairs 439 and 584, 48 pairs 660 and 584; 64 experts of 2048 and 1024, bf16: 48 pairs 142 and 160, 64 pairs 169 and 165.
constexpr int64_t kTallPairs = 40;

struct MoePlan {
    bool tiled;                // or few tokens
    int slots;                 // experts that can be active, or tiles
    int tile_rows;
    int64_t kp, ip, pairs, eight_bytes;
    int slices, steps_per_slice;         // of down's K
    uint64_t table, eights, expert, weight, pair_row, token, base, tiles, counts, x, h, out, total;
};

MoePlan plan_of(const RocmMoeArgs& a)
{
    MoePlan l{};
    if (a.rows <= 0) return l;               // (no rows: no tiles to divide the chip by)
    l.pairs = a.rows * a.k;
    // Few tokens in dot products, or in tiles: 64 experts of 2048 and 1024, 1 token 16 us and 40, 4 tokens 47 and 55; 8 experts of 4096 and 14336, 51 and 84, 156 and 342.
    // (the rows of x lie in the 48 KiB of LDS that a kernel gets without asking beside its tables)
    l.tiled = !(a.rows <= kFewTokens && a.experts <= 256 && l.pairs <= kFewPairs && a.rows * ((a.hidden + 2047) / 2048) <= 12);
    l.tile_rows = l.pairs >= kTallPairs * a.experts ? 128 : 32;
    l.slots = static_cast<int>((l.tiled ? l.pairs / l.tile_rows : 0) + (l.pairs < a.experts ? l.pairs : a.experts));
    l.kp = l.tiled ? (a.hidden + 63) / 64 * 64 : (a.hidden + 7) / 8 * 8;        // (tiles read whole steps of 64)
    l.ip = (a.inter + 127) / 128 * 128;      // (steps of 64 and 128)
    // Down in slices of its K, of 16 steps or more, until four workgroups for each CU are there: one after the other its steps are trips to memory.
    l.slices = 1;
    const int steps = static_cast<int>(l.ip / 64);
    if (l.tiled) {
        const int64_t grid = (a.hidden + 127) / 128 * l.slots, wanted = 4 * rocm_ffi_compute_units() / grid;
        const int64_t most = steps / 16 < 8 ? steps / 16 : 8;
        l.slices = static_cast<int>(wanted < most ? wanted : most);
        if (l.slices < 1) l.slices = 1;
    }
    l.steps_per_slice = ((steps + l.slices - 1) / l.slices + 1) / 2 * 2;
    l.slices = (steps + l.steps_per_slice - 1) / l.steps_per_slice;
    auto part = [&](uint64_t bytes) {
        const uint64_t here = l.total;
        l.total += (bytes + 255) / 256 * 256;
        return here;
    };
    const bool tiled = l.tiled;
    l.table = part(tiled ? 0 : sizeof(MoeFewTable));
    l.expert = part(tiled ? l.pairs * 4 : 0);
    l.weight = part(tiled ? l.pairs * 4 : 0);
    l.pair_row = part(tiled ? l.pairs * 4 : 0);
    l.token = part(tiled ? l.pairs * 4 : 0);
    l.base = part(tiled ? a.rows * 4 : 0);
    l.tiles = part(tiled ? static_cast<uint64_t>(l.slots) * 16 : 0);
    l.counts = part(tiled && a.rows > 64 ? kMoeGroups * static_cast<uint64_t>(a.experts) * 4 : 0);
    // rows that do not begin at multiples of 16 bytes are copied: the address may be any
    l.x = part(a.rows * l.kp * 2);
    l.eight_bytes = tiled && (!a.gate.zp || !a.down.zp) ? ((l.kp > l.ip ? l.kp : l.ip) + 63) / 64 + 1 : 0;
    l.eights = part(l.eight_bytes);
    // (few tokens: two parts of every value of h)
    l.h = part(tiled ? l.pairs * l.ip * 2 : l.slots * kFewTokens * l.ip * 4);
    l.out = part(tiled ? l.slices * l.pairs * a.hidden * 4 : 0);
    return l;
}

MoeMatrix matrix_of(const RocmMoeArgs& a, const RocmMoeWeights& w, const RocmMoeWeights* second, int64_t k, int64_t n, int64_t expert_step, int row_step)
{
    MoeMatrix m{};
    m.w[0] = w;
    if (second) m.w[1] = *second;
    m.expert_step = expert_step;
    m.row_step = row_step;
    m.n = static_cast<int>(n);
    m.kb = static_cast<int>((k + a.block_size - 1) / a.block_size);
    m.block_size = a.block_size;
    m.row_bytes = static_cast<int64_t>(m.kb) * a.block_size / 2;
    m.zp_row = (m.kb + 1) / 2;
    m.bias_dtype = a.bias_dtype;
    return m;
}

}  // namespace
}  // namespace mnb

extern "C" uint64_t rocm_moe_workspace_bytes(const RocmMoeArgs* args) { return mnb::plan_of(*args).total; }
extern "C" const char* rocm_moe_variant(const RocmMoeArgs* args)
{
    const mnb::MoePlan l = mnb::plan_of(*args);
    return !l.tiled ? "moe_few" : l.tile_rows == 128 ? "moe_tiles_128" : "moe_tiles_32";
}

extern "C" int rocm_launch_moe(const RocmMoeArgs* args, void* workspace, rocm_stream_t stream)
{
    using namespace mnb;
    const RocmMoeArgs& a = *args;
    if (a.rows <= 0) return 0;
    hipStream_t s = static_cast<hipStream_t>(stream);
    const MoePlan l = plan_of(a);
    uint8_t* const ws = static_cast<uint8_t*>(workspace);
    auto at = [&](uint64_t offset) { return reinterpret_cast<int32_t*>(ws + offset); };
    const MoeRoute route{at(l.expert), reinterpret_cast<float*>(ws + l.weight), at(l.pair_row), at(l.token), reinterpret_cast<float*>(ws + l.base), reinterpret_cast<int4*>(ws + l.tiles), at(l.counts)};
    MoeFewTable* const table = reinterpret_cast<MoeFewTable*>(ws + l.table);
    int rc = 0;
    if (l.tiled) rc = launch_moe_plan(a, l.tile_rows, l.slots, route, ws + l.eights, static_cast<int>(l.eight_bytes), s);
    const void* x = a.x;
    if (rc == 0 && (l.kp != a.hidden || reinterpret_cast<uintptr_t>(a.x) % 16 != 0)) {
        rc = launch_moe_pad_rows(a.x, a.rows, a.hidden, l.kp, ws + l.x, s);
        x = ws + l.x;
    }
    if (rc != 0) return rc;
    MoeUpCall up{};
    up.m = matrix_of(a, a.gate, &a.up, a.hidden, a.inter, a.up_expert_step, a.up_row_step);
    up.x = static_cast<const uint16_t*>(x);
    up.ldx = l.kp;
    up.h = reinterpret_cast<uint16_t*>(ws + l.h);
    up.ip = l.ip;
    up.alpha = a.alpha;
    up.beta = a.beta;
    up.limit = a.limit;
    up.table = table;
    up.logits = a.logits;
    up.logits_dtype = a.logits_dtype;
    up.rows = static_cast<int>(a.rows);
    up.experts = a.experts;
    up.k = a.k;
    up.normalize = a.normalize;
    MoeDownCall down{};
    down.m = matrix_of(a, a.down, nullptr, a.inter, a.hidden, a.hidden, 1);
    down.h = up.h;
    down.ip = l.ip;
    down.table = table;
    down.rows = up.rows;
    down.y = a.y;
    if (!l.tiled) return launch_moe_few(a, up, down, l.slots, s);
    auto tiled = [&](const MoeMatrix& m, const uint16_t* rows, int64_t ldx) {
        MoeTileCall t{};
        t.m = m;
        if (!m.w[0].zp) {
            t.m.w[0].zp = t.m.w[1].zp = ws + l.eights;
            t.m.zp_row = 0;
        }
        t.x = rows;
        t.ldx = ldx;
        t.tiles = route.tiles;
        t.count = static_cast<unsigned>(l.slots);
        t.h = up.h;
        t.ldh = l.ip;
        t.out = reinterpret_cast<float*>(ws + l.out);
        t.slices = l.slices;
        t.steps_per_slice = l.steps_per_slice;
        t.slice_elements = l.pairs * a.hidden;
        t.alpha = a.alpha;
        t.beta = a.beta;
        t.limit = a.limit;
        return t;
    };
    MoeTileCall first = tiled(up.m, up.x, up.ldx), second = tiled(down.m, up.h, l.ip);
    first.token = route.token;
    rc = launch_moe_tile(a, first, true, l.tile_rows, s);
    if (rc == 0) rc = launch_moe_tile(a, second, false, l.tile_rows, s);
    return rc != 0 ? rc : launch_moe_combine(a, route, reinterpret_cast<const float*>(ws + l.out), l.slices, s);
}
