// Verification of drafted tokens from given uniforms (no counterpart in the reference, which decodes one token at a
// time).
//
// Draft i of a sequence is accepted while u_i q_i(x_i) < p_i(x_i): products of two fp32 values are exact in fp64, so the
// decision is exact.  At the first refusal n the token is drawn from w = max(p_n - q_n, 0), behind the last accepted
// draft from w = p_n: the lowest v with cumsum(w)[v] > u * sum(w), sums in fp64 (a step of the cumulative sum of 10^5
// entries is about 10^-5 of the total; fp32 prefix sums would move the border by a hundredth of a step).
//
// HBM-bound: of the K+1 rows of a sequence only the refused one of p and q is read, once.  A cluster of CTAs owns a
// sequence, each a run of segments of 128 to 1024 entries; a warp sums a segment and keeps the sum in shared memory; the CTAs
// exchange their totals through distributed shared memory, every CTA finds out whether the border lies in its run, and
// the one that owns it re-reads the 1024 entries of that segment (from L2).  Order of all sums fixed by the sizes.
// 128 sequences, 131072 entries, eight drafts: 26.5 us, 24.6 without draft probabilities; 64 x 262144, four drafts: 25.4 and
// 23.8.  (A sequence without a refusal, or without draft probabilities, reads p alone and its cluster is done sooner; nothing
// takes its place, the launch is one wave.)
#include <cooperative_groups.h>

#include <utility>

#include "common.cuh"
#include "kernels.h"

namespace cg = cooperative_groups;

namespace mfc {

namespace {

constexpr int VD_MAX_THREADS = 512;
constexpr int VD_MIN_SEG = 128, VD_SEG = 1024;  // entries of a segment: at least, and at most unless the row is very long
constexpr int VD_MAX_SEGS = 512;  // segments of a CTA's run kept in shared memory; longer runs use longer segments
constexpr int VD_MAX_CLUSTER = 8;

// A negative or NaN probability counts as nothing, on either side of the difference (fmaxf takes the number beside a NaN).
__device__ __forceinline__ double weight(float p, float q) {
    const double w = (double)p - (double)fmaxf(q, 0.0f);
    return w > 0.0 ? w : 0.0;  // false for a NaN p; a p that is not positive leaves nothing above any q
}

__device__ __forceinline__ double warp_sum_f64(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// inclusive prefix sum over the lanes
__device__ __noinline__ double warp_scan_f64(double v) {
    const int lane = threadIdx.x & 31;
#pragma unroll 1
    for (int o = 1; o < 32; o <<= 1) {
        const double up = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += up;
    }
    return v;
}

// Where the cumulative sum of the lanes' values, from c on, first exceeds the target: the lane (else the last lane with a
// positive value, else -1), whether it exceeds there, the sum ahead of that lane and the sum behind all of them.  One copy
// of this code serves the three levels of the search: it runs once per sequence, so what it takes is the fetching of its
// instructions (unrolled, with 128 entries a step, the search took 8.5 thousand cycles).
struct Found {
    int lane;
    bool over;
    double ahead, behind;
};
__device__ __noinline__ Found locate(double v, double c, double target) {
    const double run = warp_scan_f64(v);
    const unsigned over = __ballot_sync(0xffffffffu, v > 0.0 && c + run > target), any = __ballot_sync(0xffffffffu, v > 0.0);
    Found f;
    f.lane = over ? __ffs(over) - 1 : (any ? 31 - __clz(any) : -1);
    f.over = over != 0;
    f.ahead = c + __shfl_sync(0xffffffffu, run - v, f.lane < 0 ? 0 : f.lane);
    f.behind = c + __shfl_sync(0xffffffffu, run, 31);
    return f;
}

// entries [v, v + 4) of the row's weights; x: the drafted token whose q is 1 when there are no draft probabilities
template <bool VEC>
__device__ __forceinline__ void load_w4(const float *p, const float *q, int x, int v, int V, double (&w)[4]) {
    float pv[4], qv[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (VEC && v + 4 <= V) {
        const float4 a = *reinterpret_cast<const float4 *>(p + v);
        pv[0] = a.x; pv[1] = a.y; pv[2] = a.z; pv[3] = a.w;
        if (q) {
            const float4 b = *reinterpret_cast<const float4 *>(q + v);
            qv[0] = b.x; qv[1] = b.y; qv[2] = b.z; qv[3] = b.w;
        }
    } else {
#pragma unroll
        for (int e = 0; e < 4; e++) {
            pv[e] = v + e < V ? p[v + e] : 0.0f;
            if (q) qv[e] = v + e < V ? q[v + e] : 0.0f;
        }
    }
#pragma unroll
    for (int e = 0; e < 4; e++) w[e] = (x == v + e) ? 0.0 : weight(pv[e], qv[e]);
}

// Sums of the segments [s0, s1) of `seg` entries into s_sum, one warp per segment.
template <bool VEC>
__device__ __forceinline__ void sum_segments(const float *p, const float *q, int x, int V, int seg, int s0, int s1, double *s_sum) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int s = s0 + warp; s < s1; s += (int)blockDim.x / 32) {
        const int v1 = min((s + 1) * seg, V);
        double acc = 0.0;
        int v0 = s * seg;
        // whole steps of 512 entries that do not hold the drafted token: a lane's loads of a step are in flight together
        for (; v0 + 512 <= v1 && (x < v0 || x >= v0 + 512); v0 += 512) {
            double t[4];
            if (VEC) {
                float4 a[4], b[4];
#pragma unroll
                for (int u = 0; u < 4; u++) a[u] = *reinterpret_cast<const float4 *>(p + v0 + 4 * lane + 128 * u);
#pragma unroll
                for (int u = 0; u < 4; u++) b[u] = q ? *reinterpret_cast<const float4 *>(q + v0 + 4 * lane + 128 * u) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                for (int u = 0; u < 4; u++)
                    t[u] = (weight(a[u].x, b[u].x) + weight(a[u].y, b[u].y)) + (weight(a[u].z, b[u].z) + weight(a[u].w, b[u].w));
            } else {  // rows that start anywhere: 32 consecutive entries a load
                float a[16], b[16];
#pragma unroll
                for (int u = 0; u < 16; u++) a[u] = p[v0 + 32 * u + lane];
#pragma unroll
                for (int u = 0; u < 16; u++) b[u] = q ? q[v0 + 32 * u + lane] : 0.0f;
#pragma unroll
                for (int u = 0; u < 4; u++)
                    t[u] = (weight(a[4 * u], b[4 * u]) + weight(a[4 * u + 1], b[4 * u + 1])) +
                           (weight(a[4 * u + 2], b[4 * u + 2]) + weight(a[4 * u + 3], b[4 * u + 3]));
            }
            acc += (t[0] + t[1]) + (t[2] + t[3]);
        }
#pragma unroll 4
        for (int v = v0 + 4 * lane; v < v1; v += 128) {
            double w[4];
            load_w4<VEC>(p, q, x, v, V, w);
            acc += (w[0] + w[1]) + (w[2] + w[3]);
        }
        acc = warp_sum_f64(acc);
        if (lane == 0) s_sum[s - s0] = acc;
    }
}

__global__ void __launch_bounds__(VD_MAX_THREADS) verify_drafts_kernel(const VerifyParams p, int seg) {
    cg::cluster_group cluster = cg::this_cluster();
    const int cs = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int b = (int)blockIdx.x / cs;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    __shared__ double s_sum[VD_MAX_SEGS];
    __shared__ double s_tot[2];  // this CTA's total, for the first pass and for the pass over p alone
    __shared__ double s_part[VD_MAX_THREADS / 32];
    __shared__ int s_n;

    dependency_wait();
    dependency_allow();
    const float u = p.u_sample[b];  // needed at the end: asked for now
    const int len = p.draft_lens ? min(p.draft_lens[b], p.K) : p.K;
    if (warp == 0) {
        bool refused = false;
        // (the drafted tokens are asked for beside the length, not behind it)
        const int x = lane < p.K ? p.drafts[(size_t)b * p.K + lane] : -1;
        if (lane < len) {
            refused = true;
            if (x >= 0 && x < p.V) {
                const float px = p.p[(size_t)b * p.p_seq + (size_t)lane * p.p_row + x];
                const float qx = p.q ? p.q[(size_t)b * p.q_seq + (size_t)lane * p.q_row + x] : 1.0f;
                refused = !((double)p.u_accept[(size_t)b * p.K + lane] * (double)fmaxf(qx, 0.0f) < (double)fmaxf(px, 0.0f));
            }
        }
        const unsigned m = __ballot_sync(0xffffffffu, refused);
        if (lane == 0) {
            s_n = m ? __ffs(m) - 1 : max(len, 0);
        }
    }
    __syncthreads();
    const int n = s_n;
    if (rank == 0 && tid <= p.K) {  // the accepted drafts, then -1; the drawn token is written behind a cluster barrier
        p.tokens[(size_t)b * (p.K + 1) + tid] = tid < n ? p.drafts[(size_t)b * p.K + tid] : -1;
        if (tid == 0) p.n_accepted[b] = n;
    }
    if (len < 0) return;  // an idle place: every CTA of the cluster leaves here

    const float *prow = p.p + (size_t)b * p.p_seq + (size_t)n * p.p_row;
    const bool cut = n < len;
    const float *qrow = (cut && p.q) ? p.q + (size_t)b * p.q_seq + (size_t)n * p.q_row : nullptr;
    int x = (cut && !p.q) ? p.drafts[(size_t)b * p.K + n] : -1;
    const bool vec = !((reinterpret_cast<uintptr_t>(prow) | reinterpret_cast<uintptr_t>(qrow)) & 15);
    const int n_segs = (p.V + seg - 1) / seg, per = (n_segs + cs - 1) / cs;
    const int s0 = min(rank * per, n_segs), s1 = min(s0 + per, n_segs);

    double total = 0.0, before = 0.0, behind = 0.0;
    for (int pass = 0; pass < 2; pass++) {
        if (vec) sum_segments<true>(prow, qrow, x, p.V, seg, s0, s1, s_sum);
        else sum_segments<false>(prow, qrow, x, p.V, seg, s0, s1, s_sum);
        __syncthreads();
        if (warp == 0) {
            double t = 0.0;
            for (int s = lane; s < s1 - s0; s += 32) t += s_sum[s];
            t = warp_sum_f64(t);
            if (lane == 0) s_tot[pass] = t;
        }
        cluster.sync();
        // every warp by itself: the sum before this CTA's run, behind it, and behind all runs, added in the order of the
        // runs, so that it never falls from one run to the next (a scan by doubling adds in another order for every lane:
        // behind a run without weight its sum can be the smaller one in the last bit)
        const double t = lane < cs ? *cluster.map_shared_rank(&s_tot[pass], lane) : 0.0;
        double run = 0.0;
#pragma unroll
        for (int r = 0; r < VD_MAX_CLUSTER; r++) {
            const double of = __shfl_sync(0xffffffffu, t, r);
            if (r <= lane) run += of;
        }
        behind = __shfl_sync(0xffffffffu, run, rank);
        before = rank > 0 ? __shfl_sync(0xffffffffu, run, rank - 1) : 0.0;
        total = __shfl_sync(0xffffffffu, run, 31);
        if (total > 0.0 || (!qrow && x < 0)) break;
        qrow = nullptr;  // the residual is zero everywhere: draw from p
        x = -1;
    }
    auto read = cluster.barrier_arrive();  // this CTA has read what it needs of its peers' memory
    // a uniform outside [0, 1) counts as the nearest end, so that the border lies in exactly one run
    const double target = fmin(fmax((double)u, 0.0), 1.0 - 1.0 / (1ll << 50)) * total;
    int *tok = p.tokens + (size_t)b * (p.K + 1) + n;
    if (s1 > s0 && total > 0.0) {
        // the border lies in this CTA's run when the sum before the run does not exceed the target and the sum behind it
        // does; all CTAs compare the same sums, which do not fall and end above the target, so exactly one run qualifies
        if (before <= target && behind > target) {
            // Four levels: the segment, a warp's part of it, a lane's, the entry.  Sums of the same entries in two orders may
            // differ in the last bit; where a level then finds no place, its last entry of any weight counts.  The first
            // two levels run in every warp alike.
            double c = before, c_last = before;
            int s = -1, s_last = s0;
#pragma unroll 1
            for (int k0 = s0; k0 < s1 && s < 0; k0 += 32) {
                const Found f = locate(k0 + lane < s1 ? s_sum[k0 + lane - s0] : 0.0, c, target);
                if (f.lane >= 0) {
                    s_last = k0 + f.lane;
                    c_last = f.ahead;
                    if (f.over) s = s_last;
                }
                c = f.behind;
            }
            // warps that share the segment (a short one is left to the first), a lane's entries
            const int parts = seg <= 512 ? 1 : min((int)blockDim.x / 32, seg / 128), per = seg / (32 * parts);
            const int v0 = s_last * seg + (warp * 32 + lane) * per;
            double mine = 0.0;
            if (warp < parts)
#pragma unroll 2
                for (int k = 0; k < per; k += 4) {
                    double w[4];
                    if (vec) load_w4<true>(prow, qrow, x, v0 + k, p.V, w);
                    else load_w4<false>(prow, qrow, x, v0 + k, p.V, w);
                    mine += (w[0] + w[1]) + (w[2] + w[3]);
                }
            int owner = 0;
            if (parts > 1) {
                const double sum = warp_sum_f64(mine);
                if (lane == 0) s_part[warp] = sum;
                __syncthreads();
                const Found wf = locate(lane < parts ? s_part[lane] : 0.0, c_last, target);
                owner = max(wf.lane, 0);
                c_last = wf.ahead;
            }
            if (warp == owner) {
                const Found lf = locate(mine, c_last, target);
                const int from = __shfl_sync(0xffffffffu, v0, max(lf.lane, 0));
                int found = -1;
                c = lf.ahead;
#pragma unroll 1
                for (int k = 0; k < per; k += 32) {
                    const int v = from + k + lane;
                    const Found f = locate(k + lane < per && v < p.V && v != x ? weight(prow[v], qrow ? qrow[v] : 0.0f) : 0.0, c, target);
                    if (f.lane >= 0) found = from + k + f.lane;
                    if (f.over) break;
                    c = f.behind;
                }
                if (lane == 0) *tok = found;
            }
        }
    }
    cluster.barrier_wait(std::move(read));  // a CTA's shared memory stays until its peers have read it
}

}  // namespace

cudaError_t verify_drafts_configure() {
    return cudaFuncSetAttribute(verify_drafts_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
}

cudaError_t launch_verify_drafts(const VerifyParams &p, int n_sms, cudaStream_t stream) {
    if (p.B <= 0) return cudaSuccess;
    // Up to eight CTAs per sequence, of 512, 256 or 128 threads: about a thousand threads per SM in one wave (128 sequences
    // of 131072 entries, 128 threads: 134, 74, 46, 32, 38 us with 1, 2, 4, 8, 16 CTAs).  A segment per warp where that
    // makes segments of at most VD_SEG entries.
    int cs = 1;
    while (cs < VD_MAX_CLUSTER && (int64_t)p.B * cs * 2 <= 7 * n_sms && (int64_t)p.V > (int64_t)cs * 8 * VD_MIN_SEG) cs *= 2;
    int threads = VD_MAX_THREADS;
    while (threads > 128 && ((int64_t)p.B * cs * threads > (int64_t)n_sms * 1024 || (int64_t)cs * threads * 4 > p.V)) threads /= 2;
    int64_t seg = VD_MIN_SEG;
    while (seg < VD_SEG && (int64_t)cs * (threads / 32) * seg < p.V) seg *= 2;
    while ((p.V + seg - 1) / seg > (int64_t)cs * VD_MAX_SEGS) seg *= 2;
    return launch_dependent(verify_drafts_kernel, dim3((unsigned)(p.B * cs)), (unsigned)threads, 0, stream, (unsigned)cs, p, (int)seg);
}

}  // namespace mfc
