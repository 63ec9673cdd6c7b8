// Eviction from a KV cache by accumulated attention weight, in place (no counterpart in the reference, which drops no
// rows).
//
// Per (sequence, kv head) with n > budget rows: the `budget` largest 32-bit keys are kept (protected rows 2^32-1, NaN 0,
// otherwise the weight's bits in an order-preserving form; ties to the lowest row), and the j-th evicted row below the
// budget receives the j-th kept row from beyond it.  Order among rows does not matter to attention once the keys are
// rotated, so this moves as few rows as any arrangement can: one per evicted row below the budget (a cache a few rows
// over its budget moves a few rows, where an order-preserving compaction would move half the cache).  Sources lie at or
// beyond the budget and destinations below it, so the moves need no order among themselves.
//
// HBM-bound for large caches: 8 bytes per row for the selection, 4 KiB (bf16: 2 KiB) per moved row; a small one is bound
// by the latency of the selection's steps.  A cluster of CTAs owns a unit; each holds the keys of a contiguous run of
// rows in shared memory, so weights and positions are read once.  The border key is found by a radix selection
// (11 + 11 + 10 bits) whose histograms are summed through distributed shared memory.  A warp walks its rows 32 at a time:
// ballots give the ranks of ties, and the holes and movers it finds go to a list of its own, in shared memory; the moves
// are dealt over all warps of the cluster, which find move j by a search over the lists' lengths.
#include <cooperative_groups.h>

#include "common.cuh"
#include "kernels.h"

namespace cg = cooperative_groups;

namespace mfc {

namespace {

constexpr int EV_THREADS = 512;
constexpr int EV_WARPS = EV_THREADS / 32;
constexpr int EV_BINS = 2048;
constexpr int EV_MAX_CLUSTER = 16;
constexpr int EV_MOVES = 8;
constexpr int EV_MIN_ROWS = 2048;
constexpr int EV_MAX_ROWS_PER_CTA = 16384;  // 8 bytes of shared memory each: 128 KiB

__device__ __forceinline__ uint32_t weight_key(float w, bool safe) {
    if (safe) return 0xffffffffu;
    if (w != w) return 0u;
    const uint32_t u = __float_as_uint(w == 0.0f ? 0.0f : w);  // -0 and +0 are one weight
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// Exclusive prefix sum of v over the block's threads; *total: the sum.  Contains two __syncthreads.
__device__ __forceinline__ int block_scan(int v, int *s_warp, int *total) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int inc = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += up;
    }
    if (lane == 31) s_warp[warp] = inc;
    __syncthreads();
    int base = 0, sum = 0;
#pragma unroll
    for (int w = 0; w < EV_WARPS; w++) {
        const int t = s_warp[w];
        if (w < warp) base += t;
        sum += t;
    }
    __syncthreads();
    *total = sum;
    return base + inc - v;
}

constexpr int EV_LISTS = EV_MAX_CLUSTER * EV_WARPS;  // lists of a unit, one per warp
static_assert(EV_LISTS <= EV_THREADS, "one thread per list");

struct EvShared {
    uint4 hist[3][EV_BINS / 4];
    int warp_sum[EV_WARPS];
    int holes[EV_WARPS], movers[EV_WARPS];          // of this CTA's warps, for its peers
    int hole0[EV_LISTS + 1], mover0[EV_LISTS + 1];  // first hole / mover of every list of the unit
    int digit, above;                               // result of a selection pass
};

// the list that holds element j: the largest l with first[l] <= j
__device__ __forceinline__ int find_list(const int *first, int lists, int j) {
    int lo = 0, hi = lists - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (first[mid] <= j) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

__global__ void __launch_bounds__(EV_THREADS) kv_evict_kernel(const EvictParams p, int rows_cap) {
    extern __shared__ uint32_t dyn[];  // [rows_cap] keys; [rows_cap] lists: a warp's range holds its holes from the front,
                                       // its movers from the back
    __shared__ EvShared sh;
    cg::cluster_group cluster = cg::this_cluster();
    const int cs = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int unit = (int)blockIdx.x / cs;
    const int b = unit / p.Hkv, h = unit % p.Hkv;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    uint32_t *keys = dyn, *list = dyn + rows_cap;

    int n = p.lens[b];
    if (n < 0 || n > p.cap) {
        if (rank == 0 && h == 0 && tid == 0) atomicOr(p.status, STATUS_BAD_ITEM);
        n = 0;
    }
    const int kept_n = min(n, p.budget);
    if (rank == 0 && h == 0 && tid == 0) p.lens_out[b] = kept_n;
    const size_t m0 = (size_t)b * p.map_seq + (size_t)h * p.map_head;
    const float *w = p.w + m0;
    const int32_t *pos = p.pos + m0;
    float *w_out = p.w_out + m0;
    int32_t *pos_out = p.pos_out + m0;

    // this CTA's run of rows
    const int chunk = (n + cs - 1) / cs;
    const int r0 = min(rank * chunk, n), r1 = min(r0 + chunk, n), rows = r1 - r0;

    if (n <= p.budget) {  // nothing to evict (the same decision in every CTA of the cluster)
        for (int i = r0 + tid; i < r1; i += EV_THREADS) {
            w_out[i] = w[i];
            pos_out[i] = pos[i];
        }
        return;
    }

    for (int i = tid; i < 3 * EV_BINS / 4; i += EV_THREADS) (&sh.hist[0][0])[i] = make_uint4(0u, 0u, 0u, 0u);
    const long long recent = (long long)p.next_pos[b] - p.n_recent;
    __syncthreads();
    for (int i = tid; i < rows; i += EV_THREADS) {
        const int ps = pos[r0 + i];
        const uint32_t k = weight_key(w[r0 + i], ps < p.n_sink || ps >= recent);
        keys[i] = k;
        atomicAdd(reinterpret_cast<unsigned *>(sh.hist[0]) + (k >> 21), 1u);
    }

    // radix selection: after pass k the leading digits of the border key are known, and how many kept rows share them
    uint32_t border = 0;
    int need = kept_n;  // kept rows among those that share the known digits
#pragma unroll
    for (int ps = 0; ps < 3; ps++) {
        const int shift = ps == 0 ? 21 : (ps == 1 ? 10 : 0);
        const int bins = ps == 2 ? 1024 : 2048;
        if (ps > 0) {
            const int known = ps == 1 ? 21 : 10;
            for (int i = tid; i < rows; i += EV_THREADS) {
                const uint32_t k = keys[i];
                if ((k >> known) == (border >> known)) atomicAdd(reinterpret_cast<unsigned *>(sh.hist[ps]) + ((k >> shift) & (bins - 1)), 1u);
            }
        }
        cluster.sync();
        // every CTA sums the histograms of all; thread t owns the four bins below bins - 4t, from the largest down
        const int quad = bins / 4 - 1 - tid;
        uint4 c = make_uint4(0u, 0u, 0u, 0u);
        if (quad >= 0)
            for (int r = 0; r < cs; r++) {
                const uint4 h4 = *cluster.map_shared_rank(&sh.hist[ps][quad], r);
                c.x += h4.x;
                c.y += h4.y;
                c.z += h4.z;
                c.w += h4.w;
            }
        int total;
        int above = block_scan((int)(c.x + c.y + c.z + c.w), sh.warp_sum, &total);
        const int cnt[4] = {(int)c.w, (int)c.z, (int)c.y, (int)c.x};
#pragma unroll
        for (int e = 0; e < 4; e++) {
            if (above < need && above + cnt[e] >= need) {
                sh.digit = quad * 4 + 3 - e;
                sh.above = above;
            }
            above += cnt[e];
        }
        __syncthreads();
        border |= (uint32_t)sh.digit << shift;
        need -= sh.above;
        __syncthreads();
    }
    // rows whose key equals the border: the `need` lowest ones are kept; those of the CTAs before this one come first
    int tie = 0;
    for (int r = 0; r < rank; r++) tie += (int)*(cluster.map_shared_rank(reinterpret_cast<unsigned *>(sh.hist[2]), r) + (border & 1023u));

    // warp w owns the rows [w0, w1) of the run
    const int per = ((rows + EV_WARPS - 1) / EV_WARPS + 31) & ~31;
    const int w0 = min(warp * per, rows), w1 = min(w0 + per, rows);
    const unsigned below = (1u << lane) - 1u;
    int ties = 0;
    for (int i = w0 + lane; i < w1; i += 32) ties += keys[i] == border;
    ties = __reduce_add_sync(0xffffffffu, ties);
    if (lane == 0) sh.warp_sum[warp] = ties;
    __syncthreads();
    for (int k = 0; k < warp; k++) tie += sh.warp_sum[k];
    int holes = 0, movers = 0;
    for (int i0 = w0; i0 < w1; i0 += 32) {
        const int i = i0 + lane, r = r0 + i;
        const bool in = i < w1;
        const uint32_t k = in ? keys[i] : 0u;
        const bool eq = in && k == border;
        const unsigned eqs = __ballot_sync(0xffffffffu, eq);
        const bool kept = in && (k > border || (eq && tie + __popc(eqs & below) < need));
        const bool hole = in && !kept && r < p.budget, mover = kept && r >= p.budget;
        const unsigned hs = __ballot_sync(0xffffffffu, hole), ms = __ballot_sync(0xffffffffu, mover);
        if (hole) list[w0 + holes + __popc(hs & below)] = (uint32_t)r;
        if (mover) list[w1 - 1 - movers - __popc(ms & below)] = (uint32_t)r;
        if (kept && !mover) {  // stays where it is
            if (w_out != w) w_out[r] = w[r];
            if (pos_out != pos) pos_out[r] = pos[r];
        }
        tie += __popc(eqs);
        holes += __popc(hs);
        movers += __popc(ms);
    }
    if (lane == 0) {
        sh.holes[warp] = holes;
        sh.movers[warp] = movers;
    }
    cluster.sync();

    // every CTA learns where each list of the unit starts
    const int lists = cs * EV_WARPS;
    int moves, all_movers;
    {
        const int r = tid / EV_WARPS, k = tid % EV_WARPS;
        const int nh = tid < lists ? *cluster.map_shared_rank(&sh.holes[k], r) : 0, nm = tid < lists ? *cluster.map_shared_rank(&sh.movers[k], r) : 0;
        const int h0 = block_scan(nh, sh.warp_sum, &moves), q0 = block_scan(nm, sh.warp_sum, &all_movers);
        if (tid < lists) {
            sh.hole0[tid] = h0;
            sh.mover0[tid] = q0;
        }
        __syncthreads();
    }
    // row of the j-th hole / mover
    auto pick = [&](int j, bool want_hole) -> int {
        const int l = find_list(want_hole ? sh.hole0 : sh.mover0, lists, j);
        const int r = l / EV_WARPS, k = l % EV_WARPS;
        const int rr = max(0, min((r + 1) * chunk, n) - min(r * chunk, n));  // rows of that CTA, its warp's range
        const int pw = ((rr + EV_WARPS - 1) / EV_WARPS + 31) & ~31;
        const int a = min(k * pw, rr), z = min(a + pw, rr);
        return (int)*cluster.map_shared_rank(&list[want_hole ? a + (j - sh.hole0[l]) : z - 1 - (j - sh.mover0[l])], r);
    };
    const size_t base = (size_t)b * p.seq_stride + (size_t)h * p.head_stride;
    const int vecs = p.row_bytes >> 4;  // 16-byte pieces of a row: 32 or 64
    const int warps = cs * EV_WARPS;
    // EV_MOVES moves a turn, both tensors: EV_MOVES * 32 bytes of each lane's loads in flight together
    for (int j0 = (rank * EV_WARPS + warp) * EV_MOVES; j0 < moves; j0 += warps * EV_MOVES) {
        const int cnt = min(EV_MOVES, moves - j0);
        int row = 0;  // lane u: destination of move u; lane EV_MOVES + u: its source
        if ((lane & (EV_MOVES - 1)) < cnt && lane < 2 * EV_MOVES) row = pick(j0 + (lane & (EV_MOVES - 1)), lane < EV_MOVES);
        const int src_row = __shfl_down_sync(0xffffffffu, row, EV_MOVES);
        if (lane < cnt) {
            w_out[row] = w[src_row];
            pos_out[row] = pos[src_row];
        }
        for (int v = lane; v < vecs; v += 32) {
            uint4 kx[EV_MOVES], vx[EV_MOVES];
#pragma unroll
            for (int u = 0; u < EV_MOVES; u++) {
                const size_t so = base + (size_t)__shfl_sync(0xffffffffu, row, EV_MOVES + u) * p.row_stride + (size_t)v * 16;
                if (u < cnt) {
                    kx[u] = *reinterpret_cast<const uint4 *>(p.k + so);
                    vx[u] = *reinterpret_cast<const uint4 *>(p.v + so);
                }
            }
#pragma unroll
            for (int u = 0; u < EV_MOVES; u++) {
                const size_t dof = base + (size_t)__shfl_sync(0xffffffffu, row, u) * p.row_stride + (size_t)v * 16;
                if (u < cnt) {
                    *reinterpret_cast<uint4 *>(p.k + dof) = kx[u];
                    *reinterpret_cast<uint4 *>(p.v + dof) = vx[u];
                }
            }
        }
    }
    cluster.sync();  // a CTA's lists stay until its peers have read them
}

}  // namespace

cudaError_t kv_evict_configure() {
    cudaError_t e = cudaFuncSetAttribute(kv_evict_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return e;
    return cudaFuncSetAttribute(kv_evict_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, EV_MAX_ROWS_PER_CTA * 8);
}

cudaError_t launch_kv_evict(const EvictParams &p, int n_sms, cudaStream_t stream) {
    const int units = p.B * p.Hkv;
    if (units <= 0) return cudaSuccess;
    // As many CTAs per unit as keep every SM busy twice, but at least EV_MIN_ROWS rows each: a small unit is over sooner
    // without the exchanges through distributed shared memory.
    int cs = 1;
    while (cs < EV_MAX_CLUSTER && ((int64_t)units * cs < 2 * n_sms || p.cap > cs * EV_MAX_ROWS_PER_CTA) && p.cap > cs * EV_MIN_ROWS) cs *= 2;
    const int rows_cap = (p.cap + cs - 1) / cs;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(units * cs));
    cfg.blockDim = dim3(EV_THREADS);
    cfg.dynamicSmemBytes = (size_t)rows_cap * 8;
    cfg.stream = stream;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned)cs;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kv_evict_kernel, p, rows_cap);
}

}  // namespace mfc
