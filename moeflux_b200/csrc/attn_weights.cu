// Attention weight that every cached row received in a step, added to its running sum (no counterpart in the reference).
//
//   weights[b][hk][j] = decay * weights[b][hk][j] + sum_{t, heads of hk that see j} exp(scale q.k_j - lse)
//
// With the lse of the attention call at hand this is one pass over K: 512 bytes read per row beside 8 for the sum.  The
// cached rows are the M index (128, one lane of tensor memory each) and the unit's n_tokens * group queries the N index of
// tcgen05.mma, so a thread owns a cached row, reads its scores for all queries from tensor memory and sums their
// exponentials without exchanging anything; N is a multiple of 16, so no query slot of a group of 12 heads times three
// tokens is wasted on a tile of 128.  With 16 queries a tile of 64 KiB takes 128 tensor cycles, with 256 it takes 2048;
// HBM needs about 2800 to deliver it.  Up to 64 queries a unit the call is HBM-bound, beyond it is not, because the queries
// take the place of the ring: one query buffer in place of two, and with 256 a ring of two granules, one tile, so that no
// rows are on their way while the products of the tile at hand run.  Caches of up to 32768 rows, 32 sequences x 2 kv heads,
// 16, 64, 80, 128, 192, 256 queries a unit: 6.3, 6.1, 5.4, 4.6, 3.5, 2.5 TB/s (87, 90, 101, 119, 165, 216 us); 512 sequences of
// up to 256 rows, where the queries weigh more than the rows: 2.3, 1.6, 1.1, 1.0 and, with 256, 0.8 TB/s.  (The first form ran the
// same products on mma.sync m16n8k16 with the rows loaded straight into fragments: as fast for 16 queries, twice as long
// for 64.)
//
// Work split: the 128-row tiles of all (sequence, kv head) units form one sequence, cut into equal runs, one persistent
// CTA per run and SM; lengths are read on the device.  Every row belongs to exactly one thread: no atomics, the same bits
// every time.  CTA (384 threads): warps 0-3 and 4-7 sum alternate tiles (scores double-buffered in tensor memory), warp 8
// issues the tensor instructions, warp 9 the TMA loads (ring of 32 KiB granules, 128 dims x 128 rows), warps 10-11 bring
// the queries and lse of the next unit (a second buffer in shared memory where two fit).
// Every mbarrier wait is bounded; when one runs out a flag ends all others, a status bit is set and the CTA leaves.
#include <math.h>

#include "common.cuh"
#include "kernels.h"
#include "tcgen05.cuh"

namespace mfc {

namespace {

constexpr int AW_THREADS = 384;
constexpr int AW_TILE = 128;
constexpr uint32_t AW_GRAN_BYTES = 32768;
constexpr int AW_MAX_GRAN = 6;
constexpr uint32_t AW_CTRL = 1024;         // barriers and flags
constexpr uint32_t AW_SMEM_MAX = 232448;
constexpr float LOG2E_AW = 1.4426950408889634f;

// Shared memory: ring of granules | query buffers | their lse and limits | control
struct AwLayout {
    int np;      // queries padded to a multiple of 16
    int bufs;    // query buffers
    int gran;    // granules of the ring
    uint32_t q_bytes, off_q, off_lse, off_ctrl, total;
};
__host__ __device__ inline AwLayout aw_layout(int nq) {
    AwLayout l;
    l.np = (nq + 15) & ~15;
    l.bufs = l.np <= 64 ? 2 : 1;
    l.q_bytes = (uint32_t)l.np * HEAD_DIM * 2;
    const uint32_t rest = (uint32_t)l.bufs * (l.q_bytes + (uint32_t)l.np * 8) + AW_CTRL + 1024;  // + alignment slack
    const uint32_t fit = (AW_SMEM_MAX - rest) / AW_GRAN_BYTES;
    l.gran = fit < AW_MAX_GRAN ? (int)fit : AW_MAX_GRAN;
    l.off_q = (uint32_t)l.gran * AW_GRAN_BYTES;
    l.off_lse = l.off_q + (uint32_t)l.bufs * l.q_bytes;
    l.off_ctrl = l.off_lse + (uint32_t)l.bufs * (uint32_t)l.np * 8;
    l.total = l.off_ctrl + AW_CTRL + 1024;
    return l;
}

__device__ __forceinline__ int aw_len(const AttnWeightsParams &p, int b) {
    const int n = p.lens[b];
    return (n < 0 || n > p.cap) ? 0 : n;
}
__device__ __forceinline__ int aw_tiles(const AttnWeightsParams &p, int b) { return (aw_len(p, b) + AW_TILE - 1) / AW_TILE; }

// A segment: the tiles [t0, t0 + nt) of one unit.  Every role of a CTA walks the same segments by itself.
struct AwWalk {
    int at, end;
    int b, begin;  // sequence at hand and its first tile
    int hk, t0, nt, len;
    __device__ __forceinline__ bool next(const AttnWeightsParams &p) {
        if (at >= end) return false;
        int nb = aw_tiles(p, b);
        while (at >= begin + p.Hkv * nb) {
            begin += p.Hkv * nb;
            b++;
            nb = aw_tiles(p, b);
        }
        hk = (at - begin) / nb;
        t0 = at - begin - hk * nb;
        nt = min(nb - t0, end - at);
        len = aw_len(p, b);
        at += nt;
        return true;
    }
};

__device__ __forceinline__ void tmem_ld16(uint32_t taddr, float (&v)[16]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
                 : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]), "=f"(v[9]),
                   "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15])
                 : "r"(taddr)
                 : "memory");
}

__global__ void __launch_bounds__(AW_THREADS, 1)
attn_weights_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ AttnWeightsParams p) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    const int nq = p.T * p.group;
    const AwLayout lay = aw_layout(nq);
    const uint32_t np = (uint32_t)lay.np;
    uint64_t *bars = reinterpret_cast<uint64_t *>(smem + lay.off_ctrl);
    // arrivals a phase: bars[0 .. 13] one, s_free 4, q_full 2, q_empty 9
    uint64_t *full = bars;            // [6] TMA: granule landed
    uint64_t *empty = bars + 6;       // [6] tcgen05.commit: the products that read the granule are done
    uint64_t *s_ready = bars + 12;    // [2] tcgen05.commit: scores of a tile are in tensor memory
    uint64_t *s_free = bars + 14;     // [2] a group's warps: scores are in registers
    uint64_t *q_full = bars + 16;     // [2] two warps: a unit's queries, lse and limits are in shared memory
    uint64_t *q_empty = bars + 18;    // [2] tcgen05.commit and the summing warps: the unit is done with them
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + 20);
    volatile int *s_fail = reinterpret_cast<volatile int *>(bars + 21);
    uint64_t *drained = bars + 22;    // tcgen05.commit, after a failure: the products in flight are done

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    // tensor memory: two buffers of np columns
    const uint32_t cols = np <= 16 ? 32 : (np <= 32 ? 64 : (np <= 64 ? 128 : (np <= 128 ? 256 : 512)));
    if (warp == 8) {
        tmem_alloc(tmem_slot, cols);
        tmem_relinquish();
    }
    if (warp == 1) {
        if (lane < 20) mbar_init(&bars[lane], lane < 14 ? 1 : (lane < 16 ? 4 : (lane < 18 ? 2 : 9)));
        if (lane == 20) *s_fail = 0;
        if (lane == 22) mbar_init(drained, 1);
        mbar_fence_init();
    }
    if (tid == 64) prefetch_tmap(&k_map);
    __syncwarp();
    dependency_wait();
    // ---- every warp by itself: scan over the lengths, this CTA's run, its first sequence ----
    AwWalk walk;
    {
        const int chunk = (p.B + 31) / 32;
        const int b_lo = min(lane * chunk, p.B), b_hi = min(b_lo + chunk, p.B);
        int mine = 0;
        bool bad = false;
        for (int b = b_lo; b < b_hi; b++) {
            mine += p.Hkv * aw_tiles(p, b);
            bad |= p.lens[b] < 0 || p.lens[b] > p.cap;
        }
        if (bad && blockIdx.x == 0 && warp == 0) atomicOr(p.status, STATUS_BAD_ITEM);
        int inc = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int up = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += up;
        }
        const int total = __shfl_sync(0xffffffffu, inc, 31);
        const int run = (total + (int)gridDim.x - 1) / (int)gridDim.x;
        walk.at = min((int)blockIdx.x * run, total);
        walk.end = min(walk.at + run, total);
        const unsigned has = __ballot_sync(0xffffffffu, inc > walk.at);
        const int src = has ? __ffs(has) - 1 : 31;
        walk.b = __shfl_sync(0xffffffffu, b_lo, src);
        walk.begin = __shfl_sync(0xffffffffu, inc - mine, src);  // next() walks on from there
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    // (only now: a CTA of the next kernel may take tensor memory and then wait for this one, which so has its own already)
    dependency_allow();
    const uint32_t tmem = *tmem_slot;
    auto warp_wait = [&](uint64_t *bar, unsigned parity) -> bool {
        for (unsigned i = 0; i < p.wait_spins; i++) {
            if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
            if (*s_fail) return false;
        }
        return false;
    };
    auto elect_one = [&]() -> bool {  // one lane of a converged warp, always the same
        uint32_t r;
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "elect.sync _|p, 0xffffffff;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(r)::"memory");
        return r != 0;
    };
    auto warp_arrive = [&](uint64_t *bar) {
        __syncwarp();
        if (lane == 0) mbar_arrive(bar);
    };
    bool ok = true;
    unsigned gi = 0, gst = 0, gph = 0;  // granules so far, ring place and phase of the next one
    auto advance = [&]() {
        gi++;
        if (++gst == (unsigned)lay.gran) {
            gst = 0;
            gph ^= 1u;
        }
    };

    if (warp == 9) {
        // ================= producer =================
        while (ok && walk.next(p)) {
            for (int j = 0; j < walk.nt && ok; j++)
                for (int d = 0; d < 2; d++) {
                    if (gi >= (unsigned)lay.gran && !(ok = warp_wait(&empty[gst], gph ^ 1u))) break;
                    if (elect_one()) {
                        mbar_expect_tx(&full[gst], AW_GRAN_BYTES);
                        if (!(p.inject_lost_load && blockIdx.x == 0 && gi == 0))
                            tma_load_5d(smem + gst * AW_GRAN_BYTES, &k_map, 0, (walk.t0 + j) * AW_TILE, 2 * d, walk.hk, walk.b, &full[gst]);
                    }
                    advance();
                }
        }
        if (!ok) *s_fail = 1;
    } else if (warp == 8) {
        // ================= issuer =================
        const uint32_t idesc = (1u << 4) | (1u << 7) | (1u << 10) | ((np >> 3) << 17) | ((128u >> 4) << 24);  // as idesc_bf16
        const uint64_t k_desc = smem_desc_sw128(smem_u32(smem), 16, 1024);
        unsigned n = 0, seg = 0;
        while (ok && walk.next(p)) {
            const unsigned qb = lay.bufs == 2 ? seg & 1u : 0u, qph = lay.bufs == 2 ? (seg >> 1) & 1u : seg & 1u;
            const uint64_t q_desc = smem_desc_sw128(smem_u32(smem + lay.off_q + qb * lay.q_bytes), 16, 1024);
            ok = warp_wait(&q_full[qb], qph);
            for (int j = 0; j < walk.nt && ok; j++) {
                const unsigned tile = n + j, par = tile & 1u;
                if (tile >= 2 && !(ok = warp_wait(&s_free[par], ((tile >> 1) - 1) & 1u))) break;
                for (int d = 0; d < 2; d++) {
                    if (!(ok = warp_wait(&full[gst], gph))) break;
                    tc_fence_after();
                    if (elect_one()) {
                        const uint64_t kd = k_desc + (uint64_t)((gst * AW_GRAN_BYTES) >> 4), qd = q_desc + (uint64_t)((2 * d * np * 128) >> 4);
#pragma unroll
                        for (int ks = 0; ks < 8; ks++)
                            tc_mma_bf16(tmem + par * np, kd + (uint64_t)(((ks >> 2) * 16384 + (ks & 3) * 32) >> 4),
                                        qd + (uint64_t)(((ks >> 2) * np * 128 + (ks & 3) * 32) >> 4), idesc, d > 0 || ks > 0);
                        tc_commit(&empty[gst]);
                        if (d == 1) {
                            tc_commit(&s_ready[par]);
                            if (j + 1 == walk.nt) tc_commit(&q_empty[qb]);
                        }
                    }
                    advance();
                }
            }
            n += walk.nt;
            seg++;
        }
        if (!ok) *s_fail = 1;
    } else if (warp >= 10) {
        // ================= queries of the units, with their lse and limits =================
        const int ltid = tid - 320;
        unsigned seg = 0;
        while (ok && walk.next(p)) {
            const unsigned qb = lay.bufs == 2 ? seg & 1u : 0u, round = lay.bufs == 2 ? seg >> 1 : seg;
            if (round > 0 && !(ok = warp_wait(&q_empty[qb], (round - 1) & 1u))) break;
            const uint32_t dst = smem_u32(smem + lay.off_q + qb * lay.q_bytes);
            const __nv_bfloat16 *qbase = p.q + (int64_t)walk.b * p.q_seq + (int64_t)walk.hk * p.group * p.q_head;
            for (int i = ltid; i < (int)np * 32; i += 64) {  // 32 pieces of 16 bytes per query
                const int r = i >> 5, c = i & 31, t = r / p.group, g = r - t * p.group;
                const uint32_t bytes = r < nq ? 16u : 0u;  // 0: filled with zeros
                const __nv_bfloat16 *src = r < nq ? qbase + (int64_t)t * p.q_token + (int64_t)g * p.q_head + 8 * c : p.q;
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst + (c >> 3) * np * 128 + r * 128 + (((c & 7) ^ (r & 7)) << 4)),
                             "l"(src), "r"(bytes)
                             : "memory");
            }
            float *lse = reinterpret_cast<float *>(smem + lay.off_lse + qb * np * 8);
            int *lim = reinterpret_cast<int *>(lse + np);
            for (int r = ltid; r < (int)np; r += 64) {
                const int t = r / p.group;
                lse[r] = r < nq ? p.lse[((size_t)walk.b * p.T + t) * p.H + walk.hk * p.group + (r - t * p.group)] * LOG2E_AW : 0.0f;
                lim[r] = r < nq ? walk.len - (p.T - 1 - t) : 0;  // rows the query sees
            }
            asm volatile("cp.async.wait_all;" ::: "memory");
            fence_proxy_async_smem();
            warp_arrive(&q_full[qb]);
            seg++;
        }
        if (!ok) *s_fail = 1;
    } else {
        // ================= sums: thread = cached row; group g takes the tiles of parity g =================
        const unsigned grp = (unsigned)warp >> 2;
        const int row = 32 * (warp & 3) + lane;
        const uint32_t src = tmem + ((uint32_t)(32 * (warp & 3)) << 16) + grp * np;
        const float sl2 = p.scale * LOG2E_AW;
        unsigned n = 0, seg = 0;
        while (ok && walk.next(p)) {
            const unsigned qb = lay.bufs == 2 ? seg & 1u : 0u, qph = lay.bufs == 2 ? (seg >> 1) & 1u : seg & 1u;
            const float *lse = reinterpret_cast<const float *>(smem + lay.off_lse + qb * np * 8);
            const int *lim = reinterpret_cast<const int *>(lse + np);
            float *wbase = p.w + (int64_t)walk.b * p.w_seq + (int64_t)walk.hk * p.w_head;
            ok = warp_wait(&q_full[qb], qph);
            for (int j = (int)((grp ^ n) & 1u); j < walk.nt && ok; j += 2) {
                const unsigned tile = n + j;
                const int r0 = (walk.t0 + j) * AW_TILE, r = r0 + row;
                const bool in = r < walk.len;
                const float old = in && p.decay != 0.0f ? wbase[r] : 0.0f;  // decay 0 starts afresh, whatever is there
                ok = warp_wait(&s_ready[grp], (tile >> 1) & 1u);
                if (!ok) break;
                tc_fence_after();
                const bool masked = r0 + AW_TILE > walk.len - (p.T - 1);  // some query does not see some row of the tile
                float s0 = 0.0f, s1 = 0.0f;
                auto add16 = [&](const float (&v)[16], uint32_t c) {  // queries c .. c + 15
                    if (masked || c + 16 > (uint32_t)nq) {  // (padded queries see nothing)
#pragma unroll
                        for (int e = 0; e < 16; e += 2) {
                            s0 += r < lim[c + e] ? ex2_approx(fmaf(v[e], sl2, -lse[c + e])) : 0.0f;
                            s1 += r < lim[c + e + 1] ? ex2_approx(fmaf(v[e + 1], sl2, -lse[c + e + 1])) : 0.0f;
                        }
                    } else {
#pragma unroll
                        for (int e = 0; e < 16; e += 4) {
                            const float4 z = *reinterpret_cast<const float4 *>(lse + c + e);
                            s0 += ex2_approx(fmaf(v[e], sl2, -z.x));
                            s1 += ex2_approx(fmaf(v[e + 1], sl2, -z.y));
                            s0 += ex2_approx(fmaf(v[e + 2], sl2, -z.z));
                            s1 += ex2_approx(fmaf(v[e + 3], sl2, -z.w));
                        }
                    }
                };
                float va[16], vb[16];  // the next 16 scores are on their way while these are summed
                tmem_ld16(src, va);
                for (uint32_t c = 0; c < np; c += 32) {
                    tc_wait_ld();
                    if (c + 16 < np) tmem_ld16(src + c + 16, vb);
                    add16(va, c);
                    if (c + 16 < np) {
                        tc_wait_ld();
                        if (c + 32 < np) tmem_ld16(src + c + 32, va);
                        add16(vb, c + 16);
                    }
                }
                tc_fence_before();
                warp_arrive(&s_free[grp]);
                if (in) wbase[r] = fmaf(p.decay, old, s0 + s1);
            }
            n += walk.nt;
            seg++;
            warp_arrive(&q_empty[qb]);
        }
        if (!ok && lane == 0) *s_fail = 1;
    }
    tc_fence_before();
    __syncthreads();
    if (tid == 0 && *s_fail) atomicOr(p.status, STATUS_TMA_TIMEOUT);
    // on the ordinary path every granule has been used; after a failure the copies in flight land before the CTA leaves
    if (warp == 9 && lane == 0 && *s_fail) {
        unsigned st = gst, ph = gph;
        for (unsigned k = 0; k < gi && k < (unsigned)lay.gran; k++) {
            if (st == 0) {
                st = (unsigned)lay.gran;
                ph ^= 1u;
            }
            st--;
            mbar_wait_bounded(&full[st], ph, p.wait_spins);
        }
    }
    if (warp == 8) {
        if (*s_fail) {  // and so do the products in flight
            if (elect_one()) tc_commit(drained);
            mbar_wait_bounded(drained, 0, p.wait_spins);
            __syncwarp();
        }
        tmem_dealloc(tmem, cols);
    }
}

}  // namespace

cudaError_t attn_weights_configure() {
    return cudaFuncSetAttribute(attn_weights_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)AW_SMEM_MAX);
}

cudaError_t launch_attn_weights(const CUtensorMap &k_map, const AttnWeightsParams &p, int n_sms, cudaStream_t stream) {
    if (p.B <= 0 || p.cap <= 0) return cudaSuccess;
    const int64_t most = (int64_t)p.B * p.Hkv * ((p.cap + AW_TILE - 1) / AW_TILE);
    const int grid = most < n_sms ? (int)most : n_sms;
    return launch_dependent(attn_weights_kernel, dim3((unsigned)grid), AW_THREADS, aw_layout(p.T * p.group).total, stream, 1u, k_map, p);
}

}  // namespace mfc
