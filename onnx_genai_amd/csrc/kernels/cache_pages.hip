// CachePages: the block table of the next step, and the pages that have to move for it.
//
// A step: slot i goes on from sequence parents[i]. Whole pages are shared. A begun page is written by the step's new tokens, so it stays with one slot, the lowest that
// continues it, unless it is a whole page of some other; every other one gets a fresh page and a copy. Fresh pages, for copies and for the tokens to come, are the
// lowest that no slot holds, dealt out slot by slot. Nothing is kept between calls: what is in use is what the table says, and a slot is freed by giving it no parent.
// Compacting: with n pages in use, the ones from n on, in rising order, go to the free ones below n, in rising order. No page is read and written by one call.
//
// Two launches. The first, one workgroup, holds a bit for each page in LDS and ranks pages and slots by sums over the workgroup; what it costs is its trips through
// the tables. The second copies: a workgroup for 8 KB of a move: a part of a page, or its pages in several layers; memory bounds it.
//
// 32 beams over 28 layers of 4 heads of 128 (42 MB read and written): 17 us, of which the copies are 7.5; 128 beams over two layers 16 us (21 with slots compared one by one).
// A half empty pool of 1500 pages in 24 layers compacted (295 MB): 76 us, the copies 66 at 4.5 TB/s, where the largest copies reach 5.2.
#include "common.hiph"

namespace mnb {
namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64, kCopyThreads = 256, kCopyBytes = 8192, kCopyGroups = 16;

struct PagesWorkspace {
    int32_t* count;       // [1]: moves
    int32_t* from;        // [pages]: sources of moves
    int32_t* to;          // [pages]: and where they go; -1: nowhere
    int32_t* list;        // [pages]: free pages by rank; compacting, where a page goes
};

// N sums over the threads below this one, and over every thread, at once. Two barriers.
template <int N>
__device__ __forceinline__ void sums_below(const int (&v)[N], int (*slots)[kWaves], int (&below)[N], int (&all)[N])
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int upto[N];
#pragma unroll
    for (int k = 0; k < N; ++k) {
        upto[k] = v[k];
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const int lower = __shfl_up(upto[k], off, 64);
            if (lane >= off) upto[k] += lower;
        }
    }
    __syncthreads();
    if (lane == 63) {
#pragma unroll
        for (int k = 0; k < N; ++k) slots[k][wave] = upto[k];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < N; ++k) {
        below[k] = upto[k] - v[k];
        all[k] = 0;
        for (int i = 0; i < kWaves; ++i) {
            below[k] += i < wave ? slots[k][i] : 0;
            all[k] += slots[k][i];
        }
    }
}

__device__ __forceinline__ bool is_set(const uint32_t* bits, int page) { return (bits[page >> 5] >> (page & 31)) & 1; }
__device__ __forceinline__ void set(uint32_t* bits, int page) { atomicOr(bits + (page >> 5), 1u << (page & 31)); }

__global__ __launch_bounds__(kThreads) void plan_kernel(RocmCachePagesArgs a, PagesWorkspace w)
{
    extern __shared__ uint32_t held[];                         // a bit for each page
    __shared__ int parent[ROCM_PAGES_MAX_SLOTS], length[ROCM_PAGES_MAX_SLOTS], begun[ROCM_PAGES_MAX_SLOTS], start[ROCM_PAGES_MAX_SLOTS], keeps[ROCM_PAGES_MAX_SLOTS];
    __shared__ int list[kThreads], slots[3][kWaves], missing, made, refused;
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const int pages = static_cast<int>(a.pages), words = (pages + 31) / 32, capacity = a.width * a.page;
    auto page_at = [&](int slot, int j) {
        const int p = a.table[static_cast<int64_t>(slot) * a.width + j];
        return p >= 0 && p < pages ? p : -1;
    };
    for (int i = t; i < words; i += kThreads) held[i] = 0;
    if (t == 0) missing = made = refused = 0;
    if (t < a.slots) {
        const int p = a.parents && !a.compact ? a.parents[t] : t;
        parent[t] = p >= 0 && p < a.slots ? p : -1;
        const int n = parent[t] < 0 ? 0 : a.lengths[parent[t]];
        length[t] = n < 0 ? 0 : n > capacity ? capacity : n;
        // a begun page counts as one like the others where nothing forks
        begun[t] = !a.compact && length[t] % a.page ? page_at(parent[t], length[t] / a.page) : -1;
    }
    __syncthreads();
    auto whole = [&](int slot) { return a.compact ? (length[slot] + a.page - 1) / a.page : length[slot] / a.page; };
    // entries of all slots side by side: a short table is one trip to memory
    const uint32_t entries = static_cast<uint32_t>(a.slots) * static_cast<uint32_t>(a.width);
    for (uint32_t e = t; e < entries; e += kThreads) {
        const int i = static_cast<int>(e / static_cast<uint32_t>(a.width)), j = static_cast<int>(e - static_cast<uint32_t>(i) * a.width), n = whole(i);
        const int p = j < n ? page_at(parent[i], j) : -1;
        if (p >= 0) set(held, p);
        else if (j < n) atomicAdd(&missing, 1);
        a.next[e] = p;
    }
    __syncthreads();
    // words of the bit map are dealt out in runs, so that ranks rise with the pages
    const int run = (words + kThreads - 1) / kThreads, first = t * run, last = first + run < words ? first + run : words;
    auto valid = [&](int word) { return 32 * word + 32 <= pages ? 0xffffffffu : (1u << (pages - 32 * word)) - 1; };

    if (a.compact) {
        int set_bits[1] = {0}, unused[1], all[1];
        for (int i = first; i < last; ++i) set_bits[0] += __popc(held[i]);
        sums_below(set_bits, slots, unused, all);
        const int live = all[0];
        auto below = [&](int word) { return 32 * word + 32 <= live ? 0xffffffffu : 32 * word >= live ? 0u : (1u << (live - 32 * word)) - 1; };
        int counts[2] = {0, 0}, at[2], both[2];                // sources and holes: as many of one as of the other
        for (int i = first; i < last; ++i) {
            counts[0] += __popc(held[i] & ~below(i));
            counts[1] += __popc(~held[i] & below(i));
        }
        sums_below(counts, slots, at, both);
        int source = at[0], hole = at[1];
        const int moves = both[0];
        for (int i = first; i < last; ++i) {
            for (uint32_t bits = held[i] & ~below(i); bits; bits &= bits - 1) w.from[source++] = 32 * i + __ffs(bits) - 1;
            for (uint32_t bits = ~held[i] & below(i); bits; bits &= bits - 1) w.to[hole++] = 32 * i + __ffs(bits) - 1;
        }
        __syncthreads();
        for (int i = t; i < moves; i += kThreads) w.list[w.from[i]] = w.to[i];
        const int room = pages / 2;
        for (int i = t; i < room; i += kThreads) {
            a.moves[2 * i] = i < moves ? w.from[i] : -1;
            a.moves[2 * i + 1] = i < moves ? w.to[i] : -1;
        }
        __syncthreads();
        for (uint32_t e = t; e < entries; e += kThreads) {
            const int i = static_cast<int>(e / static_cast<uint32_t>(a.width)), j = static_cast<int>(e - static_cast<uint32_t>(i) * a.width);
            const int p = j < whole(i) ? page_at(i, j) : -1;
            if (p >= live) a.next[e] = w.list[p];
        }
        if (t < a.slots) a.next_lengths[t] = length[t];
        if (t == 0) {
            *w.count = moves;
            a.counts[0] = live;
            a.counts[1] = missing;
        }
        return;
    }

    int need = 0, copies = 0;
    const bool rest = t < a.slots && length[t] % a.page != 0;
    bool keep = false;
    if (t < a.slots) {
        if (begun[t] >= 0) {
            // eight slots at a time, whose reads do not wait for one another (entries from t on count for nothing)
            static_assert(ROCM_PAGES_MAX_SLOTS % 8 == 0, "the last eight are there");
            const int own = begun[t];
            keep = !is_set(held, own);
            for (int i = 0; i < t && keep; i += 8) {
                bool other = false;
#pragma unroll
                for (int k = 0; k < 8; ++k) other |= (begun[i + k] == own) & (i + k < t);
                keep = !other;
            }
            copies = !keep;
        }
        const int more = a.grow && parent[t] >= 0 && a.grow[t] > 0 ? a.grow[t] : 0;
        const int end = more < capacity - length[t] ? length[t] + more : capacity;
        need = copies + (end + a.page - 1) / a.page - (length[t] + a.page - 1) / a.page;
    }
    __syncthreads();
    if (keep) set(held, begun[t]);
    __syncthreads();
    int counts[3] = {need, 0, copies}, at[3], all[3];            // fresh pages wanted, pages that are free, copies
    for (int i = first; i < last; ++i) counts[1] += __popc(~held[i] & valid(i));
    sums_below(counts, slots, at, all);
    const int mine = at[0], needed = all[0], free_pages = all[1], moves = all[2];
    if (t < a.slots) {
        start[t] = mine;
        keeps[t] = keep;
    }
    int rank = at[1];
    for (int i = first; i < last && rank < needed; ++i)
        for (uint32_t bits = ~held[i] & valid(i); bits && rank < needed; bits &= bits - 1, ++rank) {
            const int p = 32 * i + __ffs(bits) - 1;
            if (rank < kThreads) list[rank] = p;
            else w.list[rank] = p;
        }
    __syncthreads();
    // Where pages run out, the inputs' table is what the caller goes on with: no page that it has is written. A copy into one is not made, and its entry is missing.
    const bool run_out = needed > free_pages;
    if (run_out) {
        for (int i = t; i < words; i += kThreads) held[i] = 0;
        __syncthreads();
        for (uint32_t e = t; e < entries; e += kThreads) {
            const int i = static_cast<int>(e / static_cast<uint32_t>(a.width)), j = static_cast<int>(e - static_cast<uint32_t>(i) * a.width), n = a.lengths[i];
            const int p = n > 0 && j < ((n > capacity ? capacity : n) + a.page - 1) / a.page ? page_at(i, j) : -1;
            if (p >= 0) set(held, p);
        }
        __syncthreads();
    }
    auto fresh = [&](int k) { return k >= free_pages ? -1 : k < kThreads ? list[k] : w.list[k]; };
    constexpr int kOwn = 2;                                      // further pages that a slot's thread enters itself
    if (t < a.slots) {
        const int dealt = copies ? fresh(mine) : -1, copy = run_out && dealt >= 0 && is_set(held, dealt) ? -1 : dealt, have = (length[t] + a.page - 1) / a.page;
        int32_t* const next = a.next + static_cast<int64_t>(t) * a.width;
        if (rest) {
            const int p = keep ? begun[t] : copy;
            next[length[t] / a.page] = p;
            if (p < 0) atomicAdd(&missing, 1);
        }
        for (int k = copies; k < need && k < copies + kOwn; ++k) {
            const int p = fresh(mine + k);
            next[have + k - copies] = p;
            if (p < 0) atomicAdd(&missing, 1);
        }
        a.moves[2 * t] = copy >= 0 ? begun[t] : -1;
        a.moves[2 * t + 1] = copy;
        // Copies that got a page alone: fresh pages are dealt out in the order of the slots, so those are the first copies, and there are no more of them than pages.
        if (dealt >= 0) {
            w.from[at[2]] = begun[t];
            w.to[at[2]] = copy;
            if (run_out) atomicAdd(&made, 1);
            if (copy < 0) atomicAdd(&refused, 1);
        }
        a.next_lengths[t] = length[t];
    }
    for (int i = wave; i < a.slots; i += kWaves) {
        const int have = (length[i] + a.page - 1) / a.page, begins = start[i] + (begun[i] >= 0 && !keeps[i]);
        const int ends = i + 1 < a.slots ? start[i + 1] : needed;
        for (int k = begins + kOwn + lane; k < ends; k += 64) {
            const int p = fresh(k);
            if (p < 0) atomicAdd(&missing, 1);
            a.next[static_cast<int64_t>(i) * a.width + have + k - begins] = p;
        }
    }
    __syncthreads();
    if (t == 0) {
        *w.count = run_out ? made : moves;
        a.counts[0] = pages - free_pages + (run_out ? free_pages - refused : needed);
        a.counts[1] = missing;
    }
}

__global__ __launch_bounds__(kThreads) void no_slots_kernel(int32_t* counts, int32_t* moves, int room)
{
    if (counts && threadIdx.x < 2) counts[threadIdx.x] = 0;
    for (int i = threadIdx.x; moves && i < 2 * room; i += kThreads) moves[i] = -1;
}

struct CopyPlan {
    int pieces[ROCM_PAGES_MAX_POOLS];      // workgroups for one move, up to and with each pool
    int layers[ROCM_PAGES_MAX_POOLS];      // layers of a workgroup: several of pools with small pages
};

// A pool's units of W bytes: those of one move that workgroup `index` of the pool has.
template <typename W>
__device__ __forceinline__ void copy_units(const RocmCachePagesArgs& a, const PagesWorkspace& w, const RocmPool& pool, int index, int layers, int moves)
{
    constexpr int kWhole = kCopyBytes / kCopyThreads / static_cast<int>(sizeof(W)), kEach = kWhole < 8 ? kWhole : 8;
    const int parts = static_cast<int>((pool.page_bytes + kCopyBytes - 1) / kCopyBytes);          // of a page; 1 where layers > 1
    const int layer0 = index / parts * layers;
    const int64_t skip = static_cast<int64_t>(index % parts) * kCopyBytes, left = pool.page_bytes - skip;
    const int units = static_cast<int>(left < kCopyBytes ? left : kCopyBytes) / static_cast<int>(sizeof(W));
    const int these = pool.layers - layer0 < layers ? static_cast<int>(pool.layers - layer0) : layers, all = units * these;
    // where a thread's units lie in a page of the pool's first layer
    int64_t at[kEach];
    for (int base = 0; base < all; base += kEach * kCopyThreads) {
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const int u = base + threadIdx.x + i * kCopyThreads, layer = these > 1 ? u / units : 0;
            at[i] = u < all ? (layer0 + layer) * a.pages * pool.page_bytes + skip + static_cast<int64_t>(u - layer * units) * static_cast<int>(sizeof(W)) : -1;
        }
        // two moves at a time, their loads together
        const int step = gridDim.y;
        for (int m = blockIdx.y; m < moves; m += 2 * step) {
            const bool second = m + step < moves;
            const int other = second ? m + step : m;
            const int64_t from[2] = {w.from[m] * pool.page_bytes, w.from[other] * pool.page_bytes};
            const int to[2] = {w.to[m], second ? w.to[other] : -1};
            W v[2][kEach];
#pragma unroll
            for (int k = 0; k < 2; ++k)
#pragma unroll
                for (int i = 0; i < kEach; ++i) v[k][i] = at[i] >= 0 && to[k] >= 0 ? *reinterpret_cast<const W*>(static_cast<const uint8_t*>(pool.at) + from[k] + at[i]) : W{};
#pragma unroll
            for (int k = 0; k < 2; ++k)
#pragma unroll
                for (int i = 0; i < kEach; ++i)
                    if (at[i] >= 0 && to[k] >= 0) *reinterpret_cast<W*>(static_cast<uint8_t*>(pool.at) + to[k] * pool.page_bytes + at[i]) = v[k][i];
        }
    }
}

__global__ __launch_bounds__(kCopyThreads) void copy_kernel(RocmCachePagesArgs a, PagesWorkspace w, CopyPlan plan)
{
    int k = 0;
    while (static_cast<int>(blockIdx.x) >= plan.pieces[k]) ++k;
    const int index = blockIdx.x - (k ? plan.pieces[k - 1] : 0), moves = *w.count;
    const RocmPool pool = a.pool[k];
    const uint64_t aligned = reinterpret_cast<uintptr_t>(pool.at) | static_cast<uint64_t>(pool.page_bytes);
    if (aligned % 16 == 0) copy_units<uint4>(a, w, pool, index, plan.layers[k], moves);
    else if (aligned % 4 == 0) copy_units<uint32_t>(a, w, pool, index, plan.layers[k], moves);
    else copy_units<uint8_t>(a, w, pool, index, plan.layers[k], moves);
}

}  // namespace
}  // namespace mnb

extern "C" uint64_t rocm_cache_pages_workspace_bytes(const RocmCachePagesArgs* args) { return 256 + 3 * ((static_cast<uint64_t>(args->pages) * 4 + 255) / 256 * 256); }

extern "C" int rocm_launch_cache_pages(const RocmCachePagesArgs* args, void* workspace, rocm_stream_t stream)
{
    using namespace mnb;
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (args->slots <= 0) {
        hipLaunchKernelGGL(no_slots_kernel, dim3(1), dim3(kThreads), 0, s, args->counts, args->moves, static_cast<int>(args->pages / 2));
        return static_cast<int>(hipGetLastError());
    }
    if (args->slots > ROCM_PAGES_MAX_SLOTS || args->pages < 1 || args->pages > ROCM_PAGES_MAX_PAGES || args->width < 1 || args->page < 1 || static_cast<int64_t>(args->width) * args->page >= (1 << 30) || static_cast<int64_t>(args->slots) * args->width > 0x7fffffff ||
        args->pools < 0 || args->pools > ROCM_PAGES_MAX_POOLS || !workspace)
        return static_cast<int>(hipErrorInvalidValue);
    uint8_t* const at = static_cast<uint8_t*>(workspace);
    const uint64_t each = (static_cast<uint64_t>(args->pages) * 4 + 255) / 256 * 256;
    const PagesWorkspace w{reinterpret_cast<int32_t*>(at), reinterpret_cast<int32_t*>(at + 256), reinterpret_cast<int32_t*>(at + 256 + each), reinterpret_cast<int32_t*>(at + 256 + 2 * each)};
    CopyPlan plan{};
    int64_t pieces = 0;
    for (int i = 0; i < args->pools; ++i) {
        const RocmPool& pool = args->pool[i];
        const int64_t together = pool.page_bytes > 0 && pool.page_bytes < kCopyBytes ? kCopyBytes / pool.page_bytes : 1;
        plan.layers[i] = static_cast<int>(together < pool.layers ? together : pool.layers > 0 ? pool.layers : 1);
        pieces += (pool.layers + plan.layers[i] - 1) / plan.layers[i] * ((pool.page_bytes + kCopyBytes - 1) / kCopyBytes);
        if (pieces >= (1 << 20)) return static_cast<int>(hipErrorInvalidValue);
        plan.pieces[i] = static_cast<int>(pieces);
    }
    for (int i = args->pools; i < ROCM_PAGES_MAX_POOLS; ++i) plan.pieces[i] = static_cast<int>(pieces);
    hipLaunchKernelGGL(plan_kernel, dim3(1), dim3(kThreads), static_cast<unsigned>((args->pages + 31) / 32 * 4), s, *args, w);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || pieces == 0) return static_cast<int>(e);
    const int64_t most = args->compact ? args->pages / 2 : args->slots;
    if (most == 0) return 0;
    // workgroups for every CU several times over; each takes every so many of the moves, whose number only the GPU knows
    const int64_t wanted = (kCopyGroups * static_cast<int64_t>(rocm_ffi_compute_units()) + pieces - 1) / pieces, rows = most < wanted ? most : wanted;
    hipLaunchKernelGGL(copy_kernel, dim3(static_cast<unsigned>(pieces), static_cast<unsigned>(rows < 65535 ? rows : 65535)), dim3(kCopyThreads), 0, s, *args, w, plan);
    return static_cast<int>(hipGetLastError());
}
