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
// HBM-bound: 8 bytes per row for the selection, 4 KiB (bf16: 2 KiB) per moved row.  A cluster of CTAs owns a
// unit; each holds the keys of a contiguous run of rows in shared memory, so weights and positions are read once.  The
// border key is found by a radix selection (11 + 11 + 10 bits) whose histograms are summed through distributed shared
// memory; the ranks of ties, holes and movers are prefix sums over threads, then over the cluster's CTAs.
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

struct EvShared {
    unsigned hist[3][EV_BINS];
    int warp_sum[EV_WARPS];
    int n_holes, n_movers;  // of this CTA's rows, for its peers
    int digit, above;       // result of a selection pass
};

__global__ void __launch_bounds__(EV_THREADS) kv_evict_kernel(const EvictParams p, int rows_cap) {
    extern __shared__ uint32_t dyn[];  // [rows_cap] keys, [rows_cap] list: holes from the front, movers from the back
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

    for (int i = tid; i < 3 * EV_BINS; i += EV_THREADS) (&sh.hist[0][0])[i] = 0u;
    const long long recent = (long long)p.next_pos[b] - p.n_recent;
    __syncthreads();
    for (int i = tid; i < rows; i += EV_THREADS) {
        const int ps = pos[r0 + i];
        const uint32_t k = weight_key(w[r0 + i], ps < p.n_sink || ps >= recent);
        keys[i] = k;
        atomicAdd(&sh.hist[0][k >> 21], 1u);
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
                if ((k >> known) == (border >> known)) atomicAdd(&sh.hist[ps][(k >> shift) & (bins - 1)], 1u);
            }
        }
        cluster.sync();
        // every CTA sums the histograms of all; thread t owns the bins [hi - 4t - 3, hi - 4t], from the largest down
        int c[EV_BINS / EV_THREADS];
        int sum = 0;
#pragma unroll
        for (int e = 0; e < EV_BINS / EV_THREADS; e++) {
            const int bin = bins - 1 - (tid * (EV_BINS / EV_THREADS) + e);
            c[e] = 0;
            if (bin >= 0)
                for (int r = 0; r < cs; r++) c[e] += (int)*cluster.map_shared_rank(&sh.hist[ps][bin], r);
            sum += c[e];
        }
        int total;
        int above = block_scan(sum, sh.warp_sum, &total);
#pragma unroll
        for (int e = 0; e < EV_BINS / EV_THREADS; e++) {
            if (above < need && above + c[e] >= need) {
                sh.digit = bins - 1 - (tid * (EV_BINS / EV_THREADS) + e);
                sh.above = above;
            }
            above += c[e];
        }
        __syncthreads();
        border |= (uint32_t)sh.digit << shift;
        need -= sh.above;
        __syncthreads();
    }
    // rows whose key equals the border: the `need` lowest ones are kept; those of the CTAs before this one come first
    int ties_before = 0;
    for (int r = 0; r < rank; r++) ties_before += (int)*cluster.map_shared_rank(&sh.hist[2][border & 1023u], r);

    // thread t owns the rows [t * per, (t + 1) * per) of the run
    const int per = (rows + EV_THREADS - 1) / EV_THREADS;
    const int t0 = min(tid * per, rows), t1 = min(t0 + per, rows);
    int ties = 0;
    for (int i = t0; i < t1; i++) ties += keys[i] == border;
    int total;
    const int tie0 = ties_before + block_scan(ties, sh.warp_sum, &total);
    int holes = 0, movers = 0, tie = tie0;
    for (int i = t0; i < t1; i++) {
        const uint32_t k = keys[i];
        const bool kept = k > border || (k == border && tie < need);
        tie += k == border;
        holes += !kept && r0 + i < p.budget;
        movers += kept && r0 + i >= p.budget;
    }
    int n_holes, n_movers;
    int hole = block_scan(holes, sh.warp_sum, &n_holes);
    int mover = block_scan(movers, sh.warp_sum, &n_movers);
    tie = tie0;
    for (int i = t0; i < t1; i++) {
        const uint32_t k = keys[i];
        const bool kept = k > border || (k == border && tie < need);
        tie += k == border;
        const int r = r0 + i;
        if (!kept && r < p.budget) list[hole++] = (uint32_t)r;
        if (kept && r >= p.budget) list[rows - 1 - mover++] = (uint32_t)r;
        if (kept && r < p.budget) {
            w_out[r] = w[r];
            pos_out[r] = pos[r];
        }
    }
    if (tid == 0) {
        sh.n_holes = n_holes;
        sh.n_movers = n_movers;
    }
    cluster.sync();

    // the moves, dealt to the cluster's warps: move j takes the j-th mover to the j-th hole
    int moves = 0;
    for (int r = 0; r < cs; r++) moves += *cluster.map_shared_rank(&sh.n_holes, r);
    auto pick = [&](int j, bool want_hole) -> int {
        for (int r = 0; r < cs; r++) {
            const int cnt = *cluster.map_shared_rank(want_hole ? &sh.n_holes : &sh.n_movers, r);
            if (j < cnt) {
                const int rr = max(0, min((r + 1) * chunk, n) - min(r * chunk, n));
                return (int)*cluster.map_shared_rank(&list[want_hole ? j : rr - 1 - j], r);
            }
            j -= cnt;
        }
        return 0;  // not reached: holes and movers are equally many
    };
    const size_t base = (size_t)b * p.seq_stride + (size_t)h * p.head_stride;
    const int vecs = p.row_bytes >> 4;  // 16-byte pieces of a row: 32 or 64
    const int warps = cs * EV_WARPS;
    for (int j0 = (rank * EV_WARPS + warp) * 4; j0 < moves; j0 += warps * 4) {
        const int cnt = min(4, moves - j0);
        int dst = 0, src = 0;
        if (lane < cnt) {
            dst = pick(j0 + lane, true);
            src = pick(j0 + lane, false);
            w_out[dst] = w[src];
            pos_out[dst] = pos[src];
        }
        for (int v = lane; v < vecs; v += 32) {
            uint4 kx[4], vx[4];
#pragma unroll
            for (int u = 0; u < 4; u++) {
                const size_t so = base + (size_t)__shfl_sync(0xffffffffu, src, u) * p.row_stride + (size_t)v * 16;
                if (u < cnt) {
                    kx[u] = *reinterpret_cast<const uint4 *>(p.k + so);
                    vx[u] = *reinterpret_cast<const uint4 *>(p.v + so);
                }
            }
#pragma unroll
            for (int u = 0; u < 4; u++) {
                const size_t dof = base + (size_t)__shfl_sync(0xffffffffu, dst, u) * p.row_stride + (size_t)v * 16;
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
    int cs = 1;  // as many CTAs per unit as keep every SM busy twice, but at least 512 rows each
    while (cs < EV_MAX_CLUSTER && ((int64_t)units * cs < 2 * n_sms || p.cap > cs * EV_MAX_ROWS_PER_CTA) && p.cap > cs * EV_THREADS) cs *= 2;
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
