// QMoE, from router logits to the experts' rows.
//
// A token's k experts are those of its largest logits, the lowest index first among equal ones. Its weights are the softmax over all experts, or, normalized,
// over the chosen ones. An expert of weight 0 (a logit of -inf, or one so far below the largest that exp gives 0) is not chosen; a row of -inf has none, and
// its result is 0. A NaN or +inf among a token's logits makes its result NaN.
// The (token, expert) pairs are then sorted by expert, and each expert's pairs are cut into tiles of rows. The order of an expert's rows follows from atomics
// and differs from run to run; each row's result does not depend on where it lies.
#include "moe_route.hiph"

namespace mnb {
namespace {

template <int NL>
__global__ __launch_bounds__(256) void moe_top_k_kernel(const void* logits, int dtype, int64_t rows, int experts, int k, int normalize, MoeRoute r)
{
    const int lane = threadIdx.x & 63;
    const int64_t token = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
    if (token >= rows) return;
    const MoeChoice c = choose_experts<NL>(logits, dtype, token, experts, k, normalize);
    if (lane < k) {
        r.expert[token * k + lane] = c.expert;
        r.weight[token * k + lane] = c.weight;
    }
    if (lane == 0) r.base[token] = c.base;
}

__global__ __launch_bounds__(1024) void moe_route_few_kernel(const void* logits, int dtype, int rows, int experts, int k, int normalize, MoeFewTable* table)
{
    __shared__ MoeFewRouting routing;
    route_few<16>(routing, logits, dtype, rows, experts, k, normalize);
    write_table(routing, rows, k, table);
}

// One workgroup sorts the pairs and cuts the tiles.
__global__ __launch_bounds__(1024) void moe_plan_kernel(int pairs, int k, int tile_rows, int max_tiles, MoeRoute r, uint8_t* eights, int eight_bytes)
{
    __shared__ int count[1024], rows_to[1024], tiles_to[1024];
    const int t = threadIdx.x;
    for (int i = t; i < eight_bytes; i += 1024) eights[i] = 0x88;
    count[t] = 0;
    __syncthreads();
    // (kBatch pairs a thread at once: one at a time the trips to memory alone are 1.5 us for each 1024 pairs)
    constexpr int kBatch = 8;
    for (int p = t; p < pairs; p += kBatch * 1024) {
        int e[kBatch], place[kBatch];
#pragma unroll
        for (int i = 0; i < kBatch; ++i) e[i] = r.expert[min(p + i * 1024, pairs - 1)];
#pragma unroll
        for (int i = 0; i < kBatch; ++i) place[i] = p + i * 1024 < pairs && e[i] >= 0 ? atomicAdd(&count[e[i]], 1) : 0;
#pragma unroll
        for (int i = 0; i < kBatch; ++i)
            if (p + i * 1024 < pairs) r.pair_row[p + i * 1024] = place[i];
    }
    __syncthreads();
    const int own = count[t], own_tiles = (own + tile_rows - 1) / tile_rows;
    rows_to[t] = own;
    tiles_to[t] = own_tiles;
    __syncthreads();
    for (int d = 1; d < 1024; d *= 2) {
        const int a = t >= d ? rows_to[t - d] : 0, b = t >= d ? tiles_to[t - d] : 0;
        __syncthreads();
        rows_to[t] += a;
        tiles_to[t] += b;
        __syncthreads();
    }
    const int row0 = rows_to[t] - own, tile0 = tiles_to[t] - own_tiles;
    for (int i = 0; i < own_tiles; ++i) r.tiles[tile0 + i] = make_int4(t, row0 + i * tile_rows, min(tile_rows, own - i * tile_rows), 0);
    for (int i = tiles_to[1023] + t; i < max_tiles; i += 1024) r.tiles[i] = make_int4(0, 0, 0, 0);
    for (int p = t; p < pairs; p += kBatch * 1024) {
        int e[kBatch], place[kBatch];
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const int at = min(p + i * 1024, pairs - 1);
            e[i] = r.expert[at];
            place[i] = r.pair_row[at];
        }
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const int at = p + i * 1024;
            if (at >= pairs) break;
            const int row = e[i] >= 0 ? rows_to[e[i]] - count[e[i]] + place[i] : -1;
            if (row >= 0) r.token[row] = at / k;
            r.pair_row[at] = row;
        }
    }
}

// y = base + sum over a token's experts, in the order of their logits, of weight * (out + bias).
template <typename T, bool BF16>
__global__ __launch_bounds__(256) void moe_combine_kernel(RocmMoeArgs a, MoeRoute r, const float* __restrict__ out)
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

int launch_moe_top_k(const RocmMoeArgs& a, const MoeRoute& r, hipStream_t s)
{
    const dim3 grid(static_cast<unsigned>((a.rows + 3) / 4));
    auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, grid, dim3(256), 0, s, a.logits, a.logits_dtype, a.rows, a.experts, a.k, a.normalize, r);
        return static_cast<int>(hipGetLastError());
    };
    return a.experts <= 64 ? go(moe_top_k_kernel<1>) : a.experts <= 128 ? go(moe_top_k_kernel<2>) : a.experts <= 256 ? go(moe_top_k_kernel<4>) : go(moe_top_k_kernel<16>);
}

int launch_moe_route_few(const RocmMoeArgs& a, MoeFewTable* table, hipStream_t s)
{
    hipLaunchKernelGGL(moe_route_few_kernel, dim3(1), dim3(1024), 0, s, a.logits, a.logits_dtype, static_cast<int>(a.rows), a.experts, a.k, a.normalize, table);
    return static_cast<int>(hipGetLastError());
}

int launch_moe_plan(const RocmMoeArgs& a, int tile_rows, int max_tiles, const MoeRoute& r, uint8_t* eights, int eight_bytes, hipStream_t s)
{
    hipLaunchKernelGGL(moe_plan_kernel, dim3(1), dim3(1024), 0, s, static_cast<int>(a.rows * a.k), a.k, tile_rows, max_tiles, r, eights, eight_bytes);
    return static_cast<int>(hipGetLastError());
}

int launch_moe_combine(const RocmMoeArgs& a, const MoeRoute& r, const float* out, hipStream_t s)
{
    const dim3 grid = moe_grid(static_cast<unsigned>((a.hidden + 2047) / 2048), static_cast<int>(a.rows));
    if (a.dtype == ROCM_DT_BF16) hipLaunchKernelGGL((moe_combine_kernel<uint16_t, true>), grid, dim3(256), 0, s, a, r, out);
    else hipLaunchKernelGGL((moe_combine_kernel<uint16_t, false>), grid, dim3(256), 0, s, a, r, out);
    return static_cast<int>(hipGetLastError());
}

int launch_moe_pad_rows(const void* from, int64_t rows, int64_t k, int64_t kp, void* to, hipStream_t s)
{
    hipLaunchKernelGGL(moe_pad_rows_kernel, moe_grid(static_cast<unsigned>((kp + 2047) / 2048), static_cast<int>(rows)), dim3(256), 0, s, static_cast<const uint16_t*>(from), rows, k, kp,
                       static_cast<uint16_t*>(to));
    return static_cast<int>(hipGetLastError());
}

}  // namespace mnb
