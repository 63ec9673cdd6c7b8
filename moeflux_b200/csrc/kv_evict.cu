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
// Two kernels.  The selection is bound by latency (8 bytes per row, then some ten dependent steps): a cluster of CTAs owns
// a unit, each holds the keys of a contiguous run of rows in shared memory; the border (key, row) is found by a radix
// selection (11 + 11 bits, histograms summed through distributed shared memory, then the few rows that share those 22 bits
// are ranked one by one; many of them: 10 bits more, and the ties in the order of rows).  A warp walks its rows 32 at a
// time, ballots give the ranks of holes and movers, and the pairs (destination, source) go to a list in device memory.
// The copy is bound by HBM (4 KiB per moved row, bf16: 2 KiB): all moves of all units are dealt evenly over all SMs,
// whatever the units' sizes (with the copies in the selecting CTAs, 8 sequences of 7 to 20 thousand rows took twice as
// long).  A small call -- EV_FUSED_ROWS rows per unit at most -- copies in the selecting CTA and saves the second launch.
#include <cooperative_groups.h>

#include "common.cuh"
#include "kernels.h"

namespace cg = cooperative_groups;

namespace mfc {

namespace {

constexpr int EV_THREADS = 1024;
constexpr int EV_WARPS = EV_THREADS / 32;
constexpr int EV_BINS = 2048;
constexpr int EV_MAX_CLUSTER = 16;
constexpr int EV_MAX_ROWS_PER_CTA = 16384;  // 4 bytes of shared memory each: 64 KiB
constexpr int EV_MIN_ROWS = 2048;           // rows per CTA below which a cluster does not grow
constexpr int EV_FUSED_ROWS = 2048;
constexpr int EV_CAND = 32;                 // rows that are ranked one by one, a lane each
static_assert(EV_BINS / 4 <= EV_THREADS, "four bins per thread");
static_assert(EV_MAX_ROWS_PER_CTA / EV_THREADS <= 32, "a warp's masks, one per 32 rows, are held by its lanes");
static_assert(EV_FUSED_ROWS / 2 * sizeof(int2) <= EV_BINS * 4, "the moves of a small unit take the place of a histogram");

__device__ __forceinline__ uint32_t weight_key(float w, bool safe) {
    if (safe) return 0xffffffffu;
    if (w != w) return 0u;
    const uint32_t u = __float_as_uint(w == 0.0f ? 0.0f : w);  // -0 and +0 are one weight
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// Exclusive prefix sum of v over the block's threads; *total: the sum.  Contains two __syncthreads.
__device__ __forceinline__ int block_scan(int v, int *s_warp, int *total) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    int inc = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += up;
    }
    if (lane == 31) s_warp[warp] = inc;
    __syncthreads();
    const int mine = lane < warps ? s_warp[lane] : 0;  // at most 32 warps
    const int base = __reduce_add_sync(0xffffffffu, lane < warp ? mine : 0);
    *total = __reduce_add_sync(0xffffffffu, mine);
    __syncthreads();
    return base + inc - v;
}

// Copies the rows of `cnt` <= MOVES moves, both tensors; lane u < MOVES holds move u as (destination, source) rows.
template <int MOVES>
__device__ __forceinline__ void copy_rows(const EvictParams &p, size_t base, int2 move, int cnt) {
    const int lane = threadIdx.x & 31;
    const int vecs = p.row_bytes >> 4;  // 16-byte pieces of a row: 32 or 64
    for (int v = lane; v < vecs; v += 32) {
        uint4 kx[MOVES], vx[MOVES];
#pragma unroll
        for (int u = 0; u < MOVES; u++) {
            const size_t so = base + (size_t)__shfl_sync(0xffffffffu, move.y, u) * p.row_stride + (size_t)v * 16;
            if (u < cnt) {
                kx[u] = *reinterpret_cast<const uint4 *>(p.k + so);
                vx[u] = *reinterpret_cast<const uint4 *>(p.v + so);
            }
        }
#pragma unroll
        for (int u = 0; u < MOVES; u++) {
            const size_t dof = base + (size_t)__shfl_sync(0xffffffffu, move.x, u) * p.row_stride + (size_t)v * 16;
            if (u < cnt) {
                *reinterpret_cast<uint4 *>(p.k + dof) = kx[u];
                *reinterpret_cast<uint4 *>(p.v + dof) = vx[u];
            }
        }
    }
}

struct EvShared {
    uint4 hist[3][EV_BINS / 4];
    uint4 sums[EV_BINS / 4];                // of a pass, over the cluster's CTAs
    int warp_sum[3][EV_WARPS];
    int ties[EV_WARPS];
    int holes[EV_WARPS], movers[EV_WARPS];
    int2 cta_moves[EV_MAX_CLUSTER];         // the sums of both, of every CTA of the cluster
    int digit[3], above[3], count[3];       // of a pass: the border's digit, the rows above it, those that share it
    int last;                               // the last tie that is kept
    unsigned n_cand;                        // of the first CTA: rows that share the border's first 22 bits
    unsigned long long cand[EV_CAND];       // key, row (inverted: of equal keys the lower row ranks higher)
};

__global__ void __launch_bounds__(EV_THREADS, 1) kv_evict_select_kernel(const EvictParams p) {
    extern __shared__ uint32_t keys[];
    __shared__ EvShared sh;
    cg::cluster_group cluster = cg::this_cluster();
    const int cs = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int unit = (int)blockIdx.x / cs;
    const int b = unit / p.Hkv, h = unit % p.Hkv;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    for (int i = tid; i < 3 * EV_BINS / 4; i += EV_THREADS) (&sh.hist[0][0])[i] = make_uint4(0u, 0u, 0u, 0u);
    if (tid == 0) sh.n_cand = 0u;
    dependency_wait();
    dependency_allow();
    int n = p.lens[b];
    const long long recent = (long long)p.next_pos[b] - p.n_recent;
    if (n < 0 || n > p.cap) {
        if (rank == 0 && h == 0 && tid == 0) atomicOr(p.status, STATUS_BAD_ITEM);
        n = 0;
    }
    const int kept_n = min(n, p.budget);
    if (rank == 0 && tid == 0) {
        if (h == 0) p.lens_out[b] = kept_n;
        if (n <= p.budget) p.counts[unit] = 0;
    }
    const size_t m0 = (size_t)b * p.map_seq + (size_t)h * p.map_head;
    const float *w = p.w + m0;
    const int32_t *pos = p.pos + m0;
    float *w_out = p.w_out + m0;
    int32_t *pos_out = p.pos_out + m0;

    // this CTA's run of rows
    const int chunk = (n + cs - 1) / cs;
    const int r0 = min(rank * chunk, n), r1 = min(r0 + chunk, n), rows = r1 - r0;
    const bool all = n <= p.budget;  // nothing to evict (the same decision in every CTA of the cluster)
    __syncthreads();
    // keys, and the rows below the budget as if none were evicted (the moves overwrite the holes)
    for (int i0 = tid; i0 < rows; i0 += 4 * EV_THREADS) {
        float wv[4];
        int ps[4];
#pragma unroll
        for (int u = 0; u < 4; u++) {
            const int i = i0 + u * EV_THREADS;
            wv[u] = i < rows ? w[r0 + i] : 0.0f;
            ps[u] = i < rows ? pos[r0 + i] : 0;
        }
#pragma unroll
        for (int u = 0; u < 4; u++) {
            const int i = i0 + u * EV_THREADS;
            if (i >= rows) break;
            if (r0 + i < kept_n) {
                if (w_out != w) w_out[r0 + i] = wv[u];
                if (pos_out != pos) pos_out[r0 + i] = ps[u];
            }
            if (!all) {
                const uint32_t k = weight_key(wv[u], ps[u] < p.n_sink || ps[u] >= recent);
                keys[i] = k;
                atomicAdd(reinterpret_cast<unsigned *>(sh.hist[0]) + (k >> 21), 1u);
            }
        }
    }
    if (all) return;
    auto sync_unit = [&]() {
        if (cs > 1) cluster.sync();
        else __syncthreads();
    };

    // radix selection: after pass k the leading digits of the border key are known, how many of the rows that share them
    // are kept, and how many there are
    uint32_t border = 0;
    int need = kept_n, sharing = 0;
    auto select_digit = [&](int ps, int shift, int bins) {  // histogram ps is complete in every CTA's shared memory
        sync_unit();
        if (cs > 1) {
            // every CTA sums its share of the bins over all CTAs and hands the sums to all (every CTA summing every bin
            // moves cs times as much through distributed shared memory: 6.5 thousand cycles a pass against 3.5 with eight)
            const int share = bins / 4 / cs;
            if (tid < share) {
                uint4 c = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll 4
                for (int r = 0; r < cs; r++) {
                    const uint4 h4 = *cluster.map_shared_rank(&sh.hist[ps][rank * share + tid], r);
                    c.x += h4.x;
                    c.y += h4.y;
                    c.z += h4.z;
                    c.w += h4.w;
                }
#pragma unroll 4
                for (int r = 0; r < cs; r++) *cluster.map_shared_rank(&sh.sums[rank * share + tid], r) = c;
            }
            cluster.sync();
        }
        // thread t owns the four bins below bins - 4t, from the largest down
        const int quad = bins / 4 - 1 - tid;
        uint4 c = make_uint4(0u, 0u, 0u, 0u);
        if (quad >= 0) c = cs > 1 ? sh.sums[quad] : sh.hist[ps][quad];
        const int mine = (int)(c.x + c.y + c.z + c.w), sum = __reduce_add_sync(0xffffffffu, mine);
        if (lane == 0) sh.warp_sum[ps][warp] = sum;
        __syncthreads();
        const int before = __reduce_add_sync(0xffffffffu, lane < warp ? sh.warp_sum[ps][lane] : 0);
        if (before < need && before + sum >= need) {  // the border lies among this warp's bins
            int inc = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int up = __shfl_up_sync(0xffffffffu, inc, o);
                if (lane >= o) inc += up;
            }
            int above = before + inc - mine;
            const int cnt[4] = {(int)c.w, (int)c.z, (int)c.y, (int)c.x};
#pragma unroll
            for (int e = 0; e < 4; e++) {
                if (above < need && above + cnt[e] >= need) {
                    sh.digit[ps] = quad * 4 + 3 - e;
                    sh.above[ps] = above;
                    sh.count[ps] = cnt[e];
                }
                above += cnt[e];
            }
        }
        __syncthreads();
        border |= (uint32_t)sh.digit[ps] << shift;
        need -= sh.above[ps];
        sharing = sh.count[ps];
    };
    select_digit(0, 21, 2048);
    for (int i = tid; i < rows; i += EV_THREADS) {
        const uint32_t k = keys[i];
        if (k >> 21 == border >> 21) atomicAdd(reinterpret_cast<unsigned *>(sh.hist[1]) + ((k >> 10) & 2047u), 1u);
    }
    select_digit(1, 10, 2048);
    // kept: the rows whose key is above the border's, and of those that have it the rows up to `last`
    const int per = ((rows + EV_WARPS - 1) / EV_WARPS + 31) & ~31;  // warp w owns the rows [w0, w1) of the run
    const int w0 = min(warp * per, rows), w1 = min(w0 + per, rows);
    int last;
    if (sharing <= EV_CAND) {
        EvShared *first = cs > 1 ? cluster.map_shared_rank(&sh, 0) : &sh;
        for (int i = tid; i < rows; i += EV_THREADS) {
            const uint32_t k = keys[i];
            if (k >> 10 == border >> 10) first->cand[atomicAdd(&first->n_cand, 1u)] = (unsigned long long)k << 32 | (uint32_t)~(r0 + i);
        }
        sync_unit();
        const unsigned long long mine = lane < sharing ? first->cand[lane] : 0ull;
        int ahead = 0;
        for (int j = 0; j < sharing; j++) ahead += __shfl_sync(0xffffffffu, mine, j) > mine;
        const unsigned at = __ballot_sync(0xffffffffu, lane < sharing && ahead == need - 1);
        const unsigned long long edge = __shfl_sync(0xffffffffu, mine, __ffs(at) - 1);
        border = (uint32_t)(edge >> 32);
        last = (int)~(uint32_t)edge;
    } else {
        for (int i = tid; i < rows; i += EV_THREADS) {
            const uint32_t k = keys[i];
            if (k >> 10 == border >> 10) atomicAdd(reinterpret_cast<unsigned *>(sh.hist[2]) + (k & 1023u), 1u);
        }
        select_digit(2, 0, 1024);
        // the `need` lowest of the rows that have the border's key are kept; those of the CTAs before this one come first
        int here = 0;
        for (int r = 0; r <= rank; r++) {
            const int t = (int)*(cluster.map_shared_rank(reinterpret_cast<unsigned *>(sh.hist[2]), r) + (border & 1023u));
            if (r < rank) need -= t;
            else here = t;
        }
        last = need <= 0 ? -1 : n;
        if (need > 0 && need < here) {  // (the same in all threads of the CTA)
            int ties = 0;
            for (int i = w0 + lane; i < w1; i += 32) ties += keys[i] == border;
            ties = __reduce_add_sync(0xffffffffu, ties);
            if (lane == 0) sh.ties[warp] = ties;
            __syncthreads();
            int left = need - __reduce_add_sync(0xffffffffu, lane < warp ? sh.ties[lane] : 0);
            if (left > 0 && left <= ties)  // the last one that is kept is this warp's
                for (int i0 = w0; i0 < w1; i0 += 32) {
                    const unsigned eq = __ballot_sync(0xffffffffu, i0 + lane < w1 && keys[i0 + lane] == border);
                    if (left > 0 && left <= __popc(eq)) {
                        if (eq >> lane & 1u && __popc(eq & ((1u << lane) - 1u)) == left - 1) sh.last = r0 + i0 + lane;
                    }
                    left -= __popc(eq);
                }
            __syncthreads();
            last = sh.last;
        }
    }
    // Lane g holds the rows of the warp's g-th 32 that move (holes below the budget, movers beyond it).
    const int w_rows = max(w1 - w0, 0);
    unsigned hits = 0;
#pragma unroll 4
    for (int g = 0; g < (w_rows + 31) / 32; g++) {
        const int i = w0 + 32 * g + lane;
        const uint32_t k = i < w1 ? keys[i] : 0u;
        const bool kept = k > border || (k == border && r0 + i <= last);
        const unsigned m = __ballot_sync(0xffffffffu, i < w1 && kept != (r0 + i < p.budget));
        if (lane == g) hits = m;
    }
    const int low = p.budget - (r0 + w0 + 32 * lane);  // rows of lane g's 32 that lie below the budget
    const unsigned side = low >= 32 ? 0xffffffffu : (low <= 0 ? 0u : (1u << low) - 1u);
    int hole = __popc(hits & side), mover = __popc(hits & ~side);
    const int n_holes = __reduce_add_sync(0xffffffffu, hole), n_movers = __reduce_add_sync(0xffffffffu, mover);
    if (lane == 0) {
        sh.holes[warp] = n_holes;
        sh.movers[warp] = n_movers;
    }
    if (cs > 1) {  // one warp hands the CTA's sums to all (all warps fetching them took 2.5 thousand cycles longer)
        __syncthreads();
        if (warp == 0) {
            const int2 sum = make_int2(__reduce_add_sync(0xffffffffu, sh.holes[lane]), __reduce_add_sync(0xffffffffu, sh.movers[lane]));
            if (lane < cs) *cluster.map_shared_rank(&sh.cta_moves[rank], lane) = sum;
        }
    }
    // lane g: ranks of the first hole and mover of its 32 rows, within the warp and then within the unit
    {
        int ih = hole, im = mover;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int uh = __shfl_up_sync(0xffffffffu, ih, o), um = __shfl_up_sync(0xffffffffu, im, o);
            if (lane >= o) {
                ih += uh;
                im += um;
            }
        }
        hole = ih - hole;
        mover = im - mover;
    }
    sync_unit();
    const int wh = sh.holes[lane], wm = sh.movers[lane];
    int moves = __reduce_add_sync(0xffffffffu, wh);  // holes and movers of a unit are equally many
    hole += __reduce_add_sync(0xffffffffu, lane < warp ? wh : 0);
    mover += __reduce_add_sync(0xffffffffu, lane < warp ? wm : 0);
    if (cs > 1) {
        const int2 of = lane < cs ? sh.cta_moves[lane] : make_int2(0, 0);
        moves = __reduce_add_sync(0xffffffffu, of.x);
        hole += __reduce_add_sync(0xffffffffu, lane < rank ? of.x : 0);
        mover += __reduce_add_sync(0xffffffffu, lane < rank ? of.y : 0);
    }
    int2 *list = p.fused ? reinterpret_cast<int2 *>(sh.hist[0]) : p.moves + (size_t)unit * p.max_moves;
    for (int g = 0; g < (w_rows + 31) / 32; g++) {
        const unsigned m = __shfl_sync(0xffffffffu, hits, g), s = __shfl_sync(0xffffffffu, side, g);
        const int h0 = __shfl_sync(0xffffffffu, hole, g), q0 = __shfl_sync(0xffffffffu, mover, g);
        const unsigned below = (1u << lane) - 1u;
        const int row = r0 + w0 + 32 * g + lane;
        if (m & s & (1u << lane)) list[h0 + __popc(m & s & below)].x = row;
        if (m & ~s & (1u << lane)) list[q0 + __popc(m & ~s & below)].y = row;
    }
    if (rank == 0 && tid == 0) p.counts[unit] = moves;
    if (cs > 1) {
        cluster.sync();  // the histograms stay until the peers have read them
    } else if (p.fused) {
        __syncthreads();
        const size_t base = (size_t)b * p.seq_stride + (size_t)h * p.head_stride;
        for (int j0 = warp * 2; j0 < moves; j0 += EV_WARPS * 2) {
            const int cnt = min(2, moves - j0);
            int2 mv = make_int2(0, 0);
            if (lane < cnt) {
                mv = list[j0 + lane];
                w_out[mv.x] = w[mv.y];
                pos_out[mv.x] = pos[mv.y];
            }
            copy_rows<2>(p, base, mv, cnt);
        }
    }
}

// The moves of all units, dealt evenly: CTA c takes the c-th of equal runs of the units' lists laid end to end.
constexpr int EC_THREADS = 256;
constexpr int EC_MOVES = 4;  // a warp's moves a turn: 8 rows in flight, 64 bytes of each lane's loads per tensor
__global__ void __launch_bounds__(EC_THREADS) kv_evict_copy_kernel(const EvictParams p) {
    extern __shared__ int first[];  // [units + 1] first move of every unit
    __shared__ int s_warp[EC_THREADS / 32];
    const int units = p.B * p.Hkv, tid = threadIdx.x, lane = tid & 31;
    dependency_wait();  // the lists are written by the kernel before
    const int per = (units + EC_THREADS - 1) / EC_THREADS;
    const int u0 = min(tid * per, units), u1 = min(u0 + per, units);
    int sum = 0, total;
    for (int u = u0; u < u1; u++) sum += p.counts[u];
    int at = block_scan(sum, s_warp, &total);
    for (int u = u0; u < u1; u++) {
        first[u] = at;
        at += p.counts[u];
    }
    if (tid == 0) first[units] = total;
    __syncthreads();
    const int run = (total + (int)gridDim.x - 1) / (int)gridDim.x;
    const int j1 = min(((int)blockIdx.x + 1) * run, total);
    for (int j = (int)blockIdx.x * run + (tid >> 5) * EC_MOVES; j < j1; j += EC_THREADS / 32 * EC_MOVES) {
        int lo = 0, hi = units - 1;  // the unit that holds move j
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (first[mid] <= j) lo = mid;
            else hi = mid - 1;
        }
        // a turn's moves may reach into the next units: one unit at a time
        for (int a = j, z = min(j + EC_MOVES, j1); a < z;) {
            while (first[lo + 1] <= a) lo++;
            const int cnt = min(z, first[lo + 1]) - a;
            const int b = lo / p.Hkv, h = lo % p.Hkv;
            int2 mv = make_int2(0, 0);
            if (lane < cnt) {
                mv = p.moves[(size_t)lo * p.max_moves + (a - first[lo]) + lane];
                const size_t m0 = (size_t)b * p.map_seq + (size_t)h * p.map_head;
                p.w_out[m0 + mv.x] = p.w[m0 + mv.y];
                p.pos_out[m0 + mv.x] = p.pos[m0 + mv.y];
            }
            copy_rows<EC_MOVES>(p, (size_t)b * p.seq_stride + (size_t)h * p.head_stride, mv, cnt);
            a += cnt;
        }
    }
}

}  // namespace

cudaError_t kv_evict_configure() {
    cudaError_t e = cudaFuncSetAttribute(kv_evict_select_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return e;
    e = cudaFuncSetAttribute(kv_evict_select_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, EV_MAX_ROWS_PER_CTA * 4);
    if (e != cudaSuccess) return e;
    return cudaFuncSetAttribute(kv_evict_copy_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (EVICT_MAX_UNITS + 1) * 4);
}

cudaError_t launch_kv_evict(EvictParams p, int n_sms, cudaStream_t stream, int *launches) {
    const int units = p.B * p.Hkv;
    *launches = 0;
    if (units <= 0) return cudaSuccess;
    // As many CTAs per unit as there are SMs for, but at least EV_MIN_ROWS rows each: a small unit is over sooner without
    // the exchanges through distributed shared memory (4 x 1088 rows: 6.9 us in one CTA, 14.0 in eight).
    int cs = 1;
    while (cs < EV_MAX_CLUSTER && ((int64_t)units * cs * 2 <= n_sms || p.cap > cs * EV_MAX_ROWS_PER_CTA) && p.cap > cs * EV_MIN_ROWS) cs *= 2;
    p.fused = cs == 1 && p.cap <= EV_FUSED_ROWS;
    const int rows_cap = (p.cap + cs - 1) / cs;
    cudaError_t e = launch_dependent(kv_evict_select_kernel, dim3((unsigned)(units * cs)), EV_THREADS, (size_t)rows_cap * 4, stream, (unsigned)cs, p);
    if (e != cudaSuccess) return e;
    *launches = 1;
    if (p.fused) return cudaSuccess;
    e = launch_dependent(kv_evict_copy_kernel, dim3((unsigned)(n_sms * 4)), EC_THREADS, (size_t)(units + 1) * 4, stream, 1u, p);
    if (e == cudaSuccess) *launches = 2;
    return e;
}

}  // namespace mfc
