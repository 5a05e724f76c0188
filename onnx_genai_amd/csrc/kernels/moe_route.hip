// QMoE, from router logits to the experts' rows.
//
// A token's k experts are those of its largest logits, the lowest index first among equal ones. Its weights are the softmax over all experts, or, normalized,
// over the chosen ones. An expert of weight 0 (a logit of -inf, or one so far below the largest that exp gives 0) is not chosen; a row of -inf has none, and
// its result is 0. A NaN or +inf among a token's logits makes its result NaN.
// The (token, expert) pairs are then sorted by expert, and each expert's pairs are cut into tiles of rows. The order of an expert's rows follows from atomics
// and differs from run to run; each row's result does not depend on where it lies.
// Measured (8 of 64 experts): 48 tokens 11 us, one launch; 4096 tokens 7 and 7; the sums of 4096 tokens' results of 2048 58 us (285 MB: 4.9 TB/s).
#include "moe_route.hiph"

namespace mnb {
namespace {

// What the sum over the threads before a thread is, for two values at once: rows and tiles of the experts before its own.
__device__ __forceinline__ int2 sums_before(int a, int b, int2* of_wave, int2& all)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int2 v = make_int2(a, b);
    for (int d = 1; d < 64; d *= 2) {
        const int x = __shfl_up(v.x, d), y = __shfl_up(v.y, d);
        if (lane >= d) v = make_int2(v.x + x, v.y + y);
    }
    if (lane == 63) of_wave[wave] = v;
    __syncthreads();
    int2 before = make_int2(0, 0);
    all = before;
    for (int w = 0; w < 16; ++w) {
        const int2 x = of_wave[w];
        if (w < wave) before = make_int2(before.x + x.x, before.y + x.y);
        all = make_int2(all.x + x.x, all.y + x.y);
    }
    return make_int2(before.x + v.x - a, before.y + v.y - b);
}

struct MoePlanCall {
    int tile_rows, max_tiles;
    uint8_t* eights;
    int eight_bytes;
};

// By 1024 threads, a thread an expert: `own` pairs in all, `before` of them in the workgroups before. The experts' rows and tiles; row0[e]: where this workgroup's
// pairs of e begin.
__device__ __forceinline__ void cut_tiles(int own, int before, int* row0, bool write, const MoePlanCall& c, const MoeRoute& r)
{
    __shared__ int2 of_wave[16];
    const int t = threadIdx.x, tiles = (own + c.tile_rows - 1) / c.tile_rows;
    int2 all;
    const int2 to = sums_before(own, tiles, of_wave, all);
    row0[t] = to.x + before;
    if (write) {
        for (int i = 0; i < tiles; ++i) r.tiles[to.y + i] = make_int4(t, to.x + i * c.tile_rows, min(c.tile_rows, own - i * c.tile_rows), 0);
        for (int i = all.y + t; i < c.max_tiles; i += 1024) r.tiles[i] = make_int4(0, 0, 0, 0);
        for (int i = t; i < c.eight_bytes; i += 1024) c.eights[i] = 0x88;
    }
    __syncthreads();
}

__device__ __forceinline__ void place_pairs(int first, int end, int k, const int* row0, const MoeRoute& r)
{
    for (int p = first + static_cast<int>(threadIdx.x); p < end; p += 1024) {
        const int e = r.expert[p], row = e >= 0 ? row0[e] + r.pair_row[p] : -1;
        if (row >= 0) r.token[row] = p / k;
        r.pair_row[p] = row;
    }
}

// A workgroup chooses for `share` tokens and counts their experts; a pair's place among its workgroup's of that expert goes where its row will stand. The only
// workgroup of a short call cuts the tiles at once.
template <int NL>
__global__ __launch_bounds__(1024) void moe_top_k_kernel(const void* logits, int dtype, int rows, int experts, int k, int normalize, int share, MoePlanCall c, MoeRoute r)
{
    __shared__ int count[1024];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    count[threadIdx.x] = 0;
    __syncthreads();
    const int first = blockIdx.x * share, end = min(first + share, rows);
    for (int token = first + wave; token < end; token += 16) {
        const MoeChoice choice = choose_experts<NL>(logits, dtype, token, experts, k, normalize);
        if (lane < k) {
            r.expert[token * k + lane] = choice.expert;
            r.weight[token * k + lane] = choice.weight;
            if (choice.expert >= 0) r.pair_row[token * k + lane] = atomicAdd(&count[choice.expert], 1);
        }
        if (lane == 0) r.base[token] = choice.base;
    }
    __syncthreads();
    const int own = count[threadIdx.x];
    if (gridDim.x > 1) {
        if (static_cast<int>(threadIdx.x) < experts) r.counts[blockIdx.x * experts + threadIdx.x] = own;
        return;
    }
    __syncthreads();
    cut_tiles(own, 0, count, true, c, r);
    place_pairs(0, rows * k, k, count, r);
}

// The rows of the pairs of workgroup blockIdx.x of the launch before. (One workgroup for all, counting again, took 50 us for 32768 pairs.)
__global__ __launch_bounds__(1024) void moe_plan_kernel(int rows, int experts, int k, int share, MoePlanCall c, MoeRoute r)
{
    __shared__ int row0[1024];
    const int t = threadIdx.x, groups = static_cast<int>(gridDim.x), group = static_cast<int>(blockIdx.x);
    int own = 0, before = 0;
    if (t < experts)
#pragma unroll 16
        for (int i = 0; i < groups; ++i) {
            const int n = r.counts[i * experts + t];
            own += n;
            before += i < group ? n : 0;
        }
    cut_tiles(own, before, row0, group == 0, c, r);
    place_pairs(group * share * k, min((group + 1) * share, rows) * k, k, row0, r);
}

// y = base + sum over a token's experts, in the order of their logits, of weight * (out + bias), out the sum of its slices.
template <typename T, bool BF16>
__global__ __launch_bounds__(256) void moe_combine_kernel(RocmMoeArgs a, MoeRoute r, const float* __restrict__ out, int slices)
{
    const int64_t token = static_cast<int64_t>(blockIdx.z) * gridDim.y + blockIdx.y;
    if (token >= a.rows) return;
    const int64_t h = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) * 8;
    const int left = static_cast<int>(a.hidden - h < 8 ? a.hidden - h : 8);
    if (left <= 0) return;
    float sum[8];
    const float base = r.base[token];
#pragma unroll
    for (int e = 0; e < 8; ++e) sum[e] = base;
    for (int j = 0; j < a.k; ++j) {
        const int row = r.pair_row[token * a.k + j];
        if (row < 0) continue;
        const float w = r.weight[token * a.k + j];
        const float* const from = out + static_cast<int64_t>(row) * a.hidden + h;
        const int64_t bias_at = static_cast<int64_t>(r.expert[token * a.k + j]) * a.hidden + h;
        Eight<float, false> v;
        if (left == 8) v.load(from);
        else v.load_first(from, left);
        for (int i = 1; i < slices; ++i) {
            Eight<float, false> more;
            if (left == 8) more.load(from + i * (a.rows * a.k * a.hidden));
            else more.load_first(from + i * (a.rows * a.k * a.hidden), left);
#pragma unroll
            for (int e = 0; e < 8; ++e) v.raw[e] += more.raw[e];
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) sum[e] = fmaf(w, v.raw[e] + (a.down.bias && e < left ? load_as_f32(a.down.bias, a.bias_dtype, bias_at + e) : 0.f), sum[e]);
    }
    Eight<T, BF16> o;
    o.set(sum);
    T* const to = static_cast<T*>(a.y) + token * a.hidden + h;
    if (left == 8) o.store(to);
    else o.store_first(to, left);
}

// Rows of `k` elements -> rows of `kp`, zeros behind: for rows that do not begin at a multiple of 16 bytes.
__global__ __launch_bounds__(256) void moe_pad_rows_kernel(const uint16_t* __restrict__ from, int64_t rows, int64_t k, int64_t kp, uint16_t* __restrict__ to)
{
    const int64_t row = static_cast<int64_t>(blockIdx.z) * gridDim.y + blockIdx.y, i = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) * 8;
    if (i >= kp || row >= rows) return;
    Eight<uint16_t, false> e;
    const int64_t left = k - i;
    if (left >= 8) e.load(from + row * k + i);
    else e.load_first(from + row * k + i, left > 0 ? static_cast<int>(left) : 0);
    e.store(to + row * kp + i);
}

}  // namespace

int launch_moe_plan(const RocmMoeArgs& a, int tile_rows, int max_tiles, const MoeRoute& r, uint8_t* eights, int eight_bytes, hipStream_t s)
{
    // up to kMoeGroups workgroups of 32 tokens or more (a wave's tokens follow one another, 1.5 us each), but one for up to 64, which saves a launch
    const int rows = static_cast<int>(a.rows), share = rows <= 64 ? 64 : rows <= 32 * kMoeGroups ? 32 : (rows + kMoeGroups - 1) / kMoeGroups, groups = (rows + share - 1) / share;
    const MoePlanCall c{tile_rows, max_tiles, eights, eight_bytes};
    auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3(groups), dim3(1024), 0, s, a.logits, a.logits_dtype, rows, a.experts, a.k, a.normalize, share, c, r);
        return static_cast<int>(hipGetLastError());
    };
    const int rc = a.experts <= 64 ? go(moe_top_k_kernel<1>) : a.experts <= 128 ? go(moe_top_k_kernel<2>) : a.experts <= 256 ? go(moe_top_k_kernel<4>) : go(moe_top_k_kernel<16>);
    if (rc != 0 || groups == 1) return rc;
    hipLaunchKernelGGL(moe_plan_kernel, dim3(groups), dim3(1024), 0, s, rows, a.experts, a.k, share, c, r);
    return static_cast<int>(hipGetLastError());
}

int launch_moe_combine(const RocmMoeArgs& a, const MoeRoute& r, const float* out, int slices, hipStream_t s)
{
    const dim3 grid = moe_grid(static_cast<unsigned>((a.hidden + 2047) / 2048), static_cast<int>(a.rows));
    if (a.dtype == ROCM_DT_BF16) hipLaunchKernelGGL((moe_combine_kernel<uint16_t, true>), grid, dim3(256), 0, s, a, r, out, slices);
    else hipLaunchKernelGGL((moe_combine_kernel<uint16_t, false>), grid, dim3(256), 0, s, a, r, out, slices);
    return static_cast<int>(hipGetLastError());
}

int launch_moe_pad_rows(const void* from, int64_t rows, int64_t k, int64_t kp, void* to, hipStream_t s)
{
    hipLaunchKernelGGL(moe_pad_rows_kernel, moe_grid(static_cast<unsigned>((kp + 2047) / 2048), static_cast<int>(rows)), dim3(256), 0, s, static_cast<const uint16_t*>(from), rows, k, kp,
                       static_cast<uint16_t*>(to));
    return static_cast<int>(hipGetLastError());
}

}  // namespace mnb
