// Attention of a batch whose sequences share a long prefix, on the 5th-generation tensor cores (no counterpart in the
// reference, which serves one sequence).
//
// out[b,t,h] = softmax(scale q K^T) V over the prefix rows and the sequence's own rows, an optional sigmoid gate, and
// lse[b,t,h].  The prefix rows are multiplied with the queries of all sequences at once: the query rows (b, t, head of
// the group) of a kv head are the M index of one product, 128 at a time, so a prefix row is read once per 128 query rows
// instead of once per sequence.  The own rows of a sequence meet only its own t * group query rows; they run through the
// same 128 x 128 tiles with the unused query rows idle: such a tile takes 2048 tensor cycles for 128 KiB of rows, a
// third of what HBM needs to deliver them, so the idle rows cost nothing.
//
// Work split: the 128-row tiles of all units -- (kv head, 128 query rows) over the prefix, (sequence, kv head) over its
// own rows -- form one sequence, cut into equal runs, one persistent CTA per run and SM.  A CTA writes one un-normalised
// partial (o, m, l) per unit it touches; merge_kernel joins the partials of a query row by log-sum-exp, in a fixed order,
// and applies the gate.  Lengths are read on the device: every CTA finds its place by a scan over them.
//
// CTA (320 threads): warps 0-7 softmax (thread = query row x half of the 128 columns), warp 8 issues every tcgen05.mma,
// warp 9 every TMA load.  Shared memory: Q 64 KiB and a ring of ten 16 KiB granules that K and V share in the order in
// which the tensor core takes them (K: 64 dims x 128 rows, V: 256 dims x 32 rows).  Tensor memory (512 columns): O 256,
// S 128, P twice 64 (bf16, the A operand of P V straight from tensor memory).  S is free again as soon as the softmax
// has read it, so Q K^T of tile j+1 runs under the softmax of tile j, and P V of tile j under that of tile j+1.  O is
// rescaled only when a row maximum grows by more than 2^8.  P is rounded to bf16 (the type of V: both operands of one
// instruction have the same type); the row sums l are taken before that rounding.
// Every mbarrier wait is bounded; a wait that runs out sets a status bit, and the CTA waits for its copies in flight,
// frees its tensor memory and leaves.
#include <math.h>

#include "common.cuh"
#include "kernels.h"
#include "tcgen05.cuh"

namespace mfc {

namespace {

constexpr int SP_M = SHARED_ATTN_M;
constexpr int SP_N = SHARED_ATTN_N;
constexpr int SP_THREADS = 320;
constexpr int SP_GRAN = 10;                                // granules of the K/V ring
constexpr uint32_t GRAN_BYTES = 16384;
constexpr uint32_t SP_Q_BOX = SP_M * 128;                  // 64 dims of 128 query rows
constexpr uint32_t SP_OFF_RING = 4 * SP_Q_BOX;
constexpr uint32_t SP_OFF_XM = SP_OFF_RING + SP_GRAN * GRAN_BYTES;  // row-maximum / row-sum exchange
constexpr uint32_t SP_OFF_BAR = SP_OFF_XM + 1024;
constexpr uint32_t SP_SMEM = SP_OFF_BAR + 512 + 1024;      // + alignment slack
static_assert(SP_SMEM <= 232448, "shared memory of an SM");
constexpr float LOG2E_SP = 1.4426950408889634f;

constexpr uint32_t SP_TMEM_COLS = 512;
constexpr uint32_t TM_O = 0, TM_S = 256, TM_P = 384;       // P: two buffers of 64 columns

__device__ __forceinline__ void tma_load_4d(void *smem_dst, const void *tmap, int c0, int c1, int c2, int c3, uint64_t *bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes "
        "[%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(smem_u32(smem_dst)),
        "l"(tmap), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(smem_u32(bar))
        : "memory");
}
// D[tmem] (+)= A[tmem] * B[smem desc], bf16 inputs, fp32 accumulate; A: lane = row, one 32-bit column = two k
__device__ __forceinline__ void tc_mma_bf16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc,
                                               uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, {%5, %6, %7, %8}, p;\n\t}"
        ::"r"(d_tmem), "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(0), "r"(0), "r"(0), "r"(0)
        : "memory");
}

__device__ __forceinline__ int own_len(const SharedAttnParams &p, int b) {
    const int n = p.lens[b];
    return (n < 0 || n > p.own_cap) ? 0 : n;
}
__device__ __forceinline__ int own_tiles(const SharedAttnParams &p, int b) { return (own_len(p, b) + SP_N - 1) / SP_N; }

// A segment: the tiles [t0, t0 + nt) of one unit.  Every role of a CTA walks the same segments by itself.
struct Walk {
    int at, end;        // tiles of the launch-wide sequence left to this CTA
    int b, begin;       // own region: sequence at hand and its first tile
    // the segment at hand
    bool own;
    int unit;           // index among the units of its kind
    int hk, mt;         // kv head, tile of 128 query rows
    int t0, nt, len;    // len: rows of the unit

    __device__ __forceinline__ bool next(const SharedAttnParams &p) {
        if (at >= end) return false;
        const int total_p = p.Hkv * p.prefix_mtiles * p.prefix_tiles;
        if (at < total_p) {
            own = false;
            unit = at / p.prefix_tiles;
            hk = unit / p.prefix_mtiles;
            mt = unit - hk * p.prefix_mtiles;
            t0 = at - unit * p.prefix_tiles;
            nt = min(p.prefix_tiles - t0, end - at);
            len = p.prefix_len;
        } else {
            const int per = p.Hkv * p.own_mtiles;
            int nb = own_tiles(p, b);
            while (at >= begin + per * nb) {
                begin += per * nb;
                b++;
                nb = own_tiles(p, b);
            }
            own = true;
            const int u = (at - begin) / nb;
            hk = u / p.own_mtiles;
            mt = u - hk * p.own_mtiles;
            unit = b * per + u;
            t0 = at - begin - u * nb;
            nt = min(nb - t0, end - at);
            len = own_len(p, b);
        }
        at += nt;
        return true;
    }
};

__global__ void __launch_bounds__(SP_THREADS, 1)
shared_prefix_attn_kernel(const __grid_constant__ CUtensorMap pk_map, const __grid_constant__ CUtensorMap pv_map,
                          const __grid_constant__ CUtensorMap ok_map, const __grid_constant__ CUtensorMap ov_map,
                          const __grid_constant__ SharedAttnParams p) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint64_t *bars = reinterpret_cast<uint64_t *>(smem + SP_OFF_BAR);
    uint64_t *full = bars;                  // [10] TMA: granule landed
    uint64_t *empty = bars + SP_GRAN;       // [10] tcgen05.commit: the products that read the granule are done
    uint64_t *s_ready = bars + 20;          // tcgen05.commit: scores of a tile are in tensor memory
    uint64_t *s_read = bars + 21;           // 8 warps: scores are in registers
    uint64_t *p_ready = bars + 22;          // [2] 8 warps: P of a tile is in tensor memory, O may be added to
    uint64_t *pv_done = bars + 24;          // [2] tcgen05.commit: P V of a tile has been accumulated
    uint64_t *q_ready = bars + 26;          // 8 warps: the segment's Q is in shared memory, O has been read out
    uint64_t *x_ready = bars + 27;          // [4] 2 warps: both column halves of a lane quadrant have published
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + 31);
    volatile int *s_fail = reinterpret_cast<volatile int *>(bars + 32);
    int *s_scan = reinterpret_cast<int *>(bars + 33);  // [10] + location [2]

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    // ---- scan over the lengths: tiles in all, this CTA's run, its first sequence ----
    const int per_seq = p.Hkv * p.own_mtiles;
    const int chunk = (p.B + SP_THREADS - 1) / SP_THREADS;
    const int b_lo = min(tid * chunk, p.B), b_hi = min(b_lo + chunk, p.B);
    int mine = 0;
    for (int b = b_lo; b < b_hi; b++) {
        mine += per_seq * own_tiles(p, b);
        if (blockIdx.x == 0 && (p.lens[b] < 0 || p.lens[b] > p.own_cap)) atomicOr(p.status, STATUS_BAD_ITEM);
    }
    int inc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += up;
    }
    if (lane == 31) s_scan[warp] = inc;
    if (tid == 0) {
        for (int i = 0; i < SP_GRAN; i++) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], 1);
        }
        mbar_init(s_ready, 1);
        mbar_init(s_read, 8);
        for (int i = 0; i < 2; i++) {
            mbar_init(&p_ready[i], 8);
            mbar_init(&pv_done[i], 1);
        }
        mbar_init(q_ready, 8);
        for (int i = 0; i < 4; i++) mbar_init(&x_ready[i], 2);
        *s_fail = 0;
        mbar_fence_init();
    }
    __syncthreads();
    const int total_p = p.Hkv * p.prefix_mtiles * p.prefix_tiles;
    int base = 0, total = total_p;
    for (int w = 0; w < SP_THREADS / 32; w++) {
        if (w < warp) base += s_scan[w];
        total += s_scan[w];
    }
    const int run = max(1, (total + (int)gridDim.x - 1) / (int)gridDim.x);
    Walk walk;
    walk.at = min((int)blockIdx.x * run, total);
    walk.end = min(walk.at + run, total);
    {
        int first = total_p + base + inc - mine;
        const int want = max(walk.at, total_p);
        for (int b = b_lo; b < b_hi; b++) {
            const int n = per_seq * own_tiles(p, b);
            if (blockIdx.x == 0) p.plan[8 + b] = first;
            if (want >= first && want < first + n) {
                s_scan[10] = b;
                s_scan[11] = first;
            }
            first += n;
        }
        if (blockIdx.x == 0 && tid == 0) {
            p.plan[0] = run;
            p.plan[1] = total;
        }
    }
    if (walk.at >= walk.end) return;  // more CTAs than tiles

    if (warp == 0) {
        tmem_alloc(tmem_slot, SP_TMEM_COLS);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    walk.b = s_scan[10];  // used only when the run reaches the own region (then some thread has set them)
    walk.begin = s_scan[11];
    const uint32_t tmem = *tmem_slot;
    bool ok = true;
    unsigned gi = 0;  // granules requested (producer) or consumed (issuer)

    if (warp == 9) {
        // ================= producer: one lane issues every TMA load =================
        if (lane == 0) {
            auto granule = [&]() -> uint8_t * {  // waits until the next granule is free, arms its barrier
                const unsigned st = gi % SP_GRAN, round = gi / SP_GRAN;
                if (round > 0 && !mbar_wait_bounded(&empty[st], (round - 1) & 1u)) return nullptr;
                if (*s_fail) return nullptr;
                mbar_expect_tx(&full[st], GRAN_BYTES);
                return smem + SP_OFF_RING + st * GRAN_BYTES;
            };
            auto load_k = [&](const Walk &s, int tile) {
                for (int d = 0; d < 4 && ok; d++) {
                    uint8_t *dst = granule();
                    if (!(ok = dst != nullptr)) break;
                    uint64_t *bar = &full[gi % SP_GRAN];
                    if (s.own) tma_load_4d(dst, &ok_map, d * 64, tile * SP_N, s.hk, s.b, bar);
                    else tma_load_3d(dst, &pk_map, d * 64, tile * SP_N, s.hk, bar);
                    gi++;
                }
            };
            auto load_v = [&](const Walk &s, int tile) {
                for (int r = 0; r < 4 && ok; r++) {
                    uint8_t *dst = granule();
                    if (!(ok = dst != nullptr)) break;
                    uint64_t *bar = &full[gi % SP_GRAN];
#pragma unroll
                    for (int d = 0; d < 4; d++) {
                        if (s.own) tma_load_4d(dst + d * 4096, &ov_map, d * 64, tile * SP_N + r * 32, s.hk, s.b, bar);
                        else tma_load_3d(dst + d * 4096, &pv_map, d * 64, tile * SP_N + r * 32, s.hk, bar);
                    }
                    gi++;
                }
            };
            while (ok && walk.next(p)) {
                load_k(walk, walk.t0);
                for (int j = 0; j < walk.nt && ok; j++) {
                    if (j + 1 < walk.nt) load_k(walk, walk.t0 + j + 1);
                    load_v(walk, walk.t0 + j);
                }
            }
            if (!ok) *s_fail = 1;
        }
    } else if (warp == 8) {
        // ================= issuer: one lane drives the tensor core =================
        if (lane == 0) {
            constexpr uint32_t IDESC_QK = idesc_bf16(SP_N, 0);
            constexpr uint32_t IDESC_PV = idesc_bf16(HEAD_DIM, 1);
            const uint64_t q_desc = smem_desc_sw128(smem_u32(smem), 16, 1024);
            const uint64_t k_desc = smem_desc_sw128(smem_u32(smem + SP_OFF_RING), 16, 1024);
            // V: MN-major; 64-dim boxes 4096 B apart (LBO), 8-row groups 1024 B apart (SBO)
            const uint64_t v_desc = smem_desc_sw128(smem_u32(smem + SP_OFF_RING), 4096, 1024);
            unsigned n = 0;   // tiles so far, over all segments
            unsigned seg = 0;
            auto issue_qk = [&](unsigned tile) -> bool {
                if (tile > 0 && !mbar_wait_bounded(s_read, (tile - 1) & 1u)) return false;
                for (int d = 0; d < 4; d++) {
                    const unsigned st = gi % SP_GRAN;
                    if (!mbar_wait_bounded(&full[st], (gi / SP_GRAN) & 1u)) return false;
                    tc_fence_after();
#pragma unroll
                    for (int ks = 0; ks < 4; ks++)
                        tc_mma_bf16(tmem + TM_S, q_desc + (uint64_t)((d * SP_Q_BOX + ks * 32) >> 4),
                                    k_desc + (uint64_t)((st * GRAN_BYTES + ks * 32) >> 4), IDESC_QK, d > 0 || ks > 0);
                    tc_commit(&empty[st]);
                    gi++;
                }
                tc_commit(s_ready);
                return true;
            };
            while (ok && walk.next(p)) {
                ok = mbar_wait_bounded(q_ready, seg & 1u);
                if (!ok) break;
                tc_fence_after();
                ok = issue_qk(n);
                for (int j = 0; j < walk.nt && ok; j++) {
                    if (j + 1 < walk.nt) ok = issue_qk(n + j + 1);
                    const unsigned tile = n + j, pb = tile & 1u;
                    ok = ok && mbar_wait_bounded(&p_ready[pb], (tile >> 1) & 1u);
                    if (!ok) break;
                    tc_fence_after();
                    for (int r = 0; r < 4; r++) {
                        const unsigned st = gi % SP_GRAN;
                        ok = mbar_wait_bounded(&full[st], (gi / SP_GRAN) & 1u);
                        if (!ok) break;
                        tc_fence_after();
#pragma unroll
                        for (int ks = 0; ks < 2; ks++)
                            tc_mma_bf16_ts(tmem + TM_O, tmem + TM_P + pb * 64 + (r * 2 + ks) * 8,
                                           v_desc + (uint64_t)((st * GRAN_BYTES + ks * 2048) >> 4), IDESC_PV,
                                           j > 0 || r > 0 || ks > 0);
                        tc_commit(&empty[st]);
                        gi++;
                    }
                    if (ok) tc_commit(&pv_done[pb]);
                }
                n += walk.nt;
                seg++;
            }
            if (!ok) *s_fail = 1;
        }
    } else {
        // ================= softmax warps: thread = (query row, half of the columns) =================
        const int quad = warp & 3, hf = warp >> 2;
        const int row = 32 * quad + lane;  // query row of the tile = lane of tensor memory
        const uint32_t lane_base = tmem + ((uint32_t)(32 * quad) << 16);
        __nv_bfloat16 *xm = reinterpret_cast<__nv_bfloat16 *>(smem + SP_OFF_XM);  // [2 tiles][2 halves][128 rows]
        float *xl = reinterpret_cast<float *>(smem + SP_OFF_XM);                  // [2 halves][128 rows]
        const float sl2 = p.scale * LOG2E_SP;
        const int tg = p.T * p.group;
        auto warp_arrive = [&](uint64_t *bar) {
            __syncwarp();
            if (lane == 0) mbar_arrive(bar);
        };
        auto warp_wait = [&](uint64_t *bar, unsigned parity) -> bool {
            return __all_sync(0xffffffffu, mbar_wait_bounded(bar, parity) && *s_fail == 0);
        };
        unsigned x_phase = 0;
        auto pair_sync = [&]() -> bool {  // the two warps of a quadrant
            warp_arrive(&x_ready[quad]);
            const bool done = warp_wait(&x_ready[quad], x_phase & 1u);
            x_phase++;
            return done;
        };
        unsigned n = 0;
        while (ok && walk.next(p)) {
            // ---- Q: this warp brings 16 rows, one 512-byte row per load; rows without a query are zero ----
            const int rows = walk.own ? min(SP_M, tg - walk.mt * SP_M) : min(SP_M, p.B * tg - walk.mt * SP_M);
            {
                uint4 v[16];
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    const int r = 16 * warp + i;
                    v[i] = make_uint4(0u, 0u, 0u, 0u);
                    if (r < rows) {
                        const int idx = walk.mt * SP_M + r;
                        const int bt = idx / p.group, hg = idx - bt * p.group;
                        const int b = walk.own ? walk.b : bt / p.T, t = walk.own ? bt : bt % p.T;
                        v[i] = *reinterpret_cast<const uint4 *>(p.q + (int64_t)b * p.q_seq + (int64_t)t * p.q_token +
                                                                (int64_t)(walk.hk * p.group + hg) * p.q_head + 8 * lane);
                    }
                }
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    const int r = 16 * warp + i;
                    *reinterpret_cast<uint4 *>(smem + (lane >> 3) * SP_Q_BOX + r * 128 + (((lane & 7) ^ (r & 7)) << 4)) = v[i];
                }
            }
            fence_proxy_async_smem();
            tc_fence_before();  // O of the previous segment has been read
            warp_arrive(q_ready);

            // columns of the unit this row sees
            int lim = walk.len;
            if (walk.own) lim = walk.len - (p.T - 1 - (walk.mt * SP_M + row) / p.group);
            const int safe = walk.own ? walk.len - (p.T - 1) : walk.len;  // columns that every row sees
            const bool live = 32 * quad < rows;                           // some row of this warp carries a query
            float m_run = -INFINITY, l_run = 0.0f;  // l_run: this thread's half of the columns
            for (int j = 0; j < walk.nt && ok; j++) {
                const unsigned tile = n + j, pb = tile & 1u;
                const int col0 = (walk.t0 + j) * SP_N;
                ok = warp_wait(s_ready, tile & 1u);
                if (!ok) break;
                tc_fence_after();
                float s[64];
                if (live) {
                    tmem_ld32(lane_base + TM_S + 64 * hf, s);
                    tmem_ld32(lane_base + TM_S + 64 * hf + 32, s + 32);
                    tc_wait_ld();
                }
                tc_fence_before();
                warp_arrive(s_read);
                float corr = 1.0f;
                bool warp_rescale = false;
                uint32_t pk[32];
                if (live) {
                    const int c0 = col0 + 64 * hf;
                    if (col0 + SP_N > safe) {
#pragma unroll
                        for (int c = 0; c < 64; c++)
                            if (c0 + c >= lim) s[c] = -INFINITY;
                    }
                    float mx = s[0];
#pragma unroll
                    for (int c = 1; c < 64; c++) mx = fmaxf(mx, s[c]);
                    // both halves of a row use one maximum: each rounds its own up to bf16 (the running maximum only
                    // has to bound the scores, roughly) and takes the larger
                    const __nv_bfloat16 mx_b = __float2bfloat16_ru(mx);
                    xm[(pb * 2 + hf) * SP_M + row] = mx_b;
                    ok = pair_sync();
                    if (!ok) break;
                    const float m_tile = fmaxf(__bfloat162float(mx_b), __bfloat162float(xm[(pb * 2 + (hf ^ 1)) * SP_M + row]));
                    const float m_new = fmaxf(m_run, m_tile);
                    const bool need = (m_new - m_run) * sl2 > 8.0f;  // also true for the first finite maximum
                    warp_rescale = __any_sync(0xffffffffu, need);
                    if (warp_rescale) {
                        corr = m_new == -INFINITY ? 1.0f : ex2_approx((m_run - m_new) * sl2);
                        m_run = m_new;
                    }
                    const float mb = m_run == -INFINITY ? 0.0f : m_run * sl2;
                    float rs = 0.0f;
#pragma unroll
                    for (int c = 0; c < 64; c += 2) {
                        const float p0 = ex2_approx(fmaf(s[c], sl2, -mb));
                        const float p1 = ex2_approx(fmaf(s[c + 1], sl2, -mb));
                        rs += p0 + p1;
                        pk[c >> 1] = pack_bf16x2(p0, p1);
                    }
                    l_run = l_run * corr + rs;
                }
                // P buffer pb was last read by P V of tile - 2
                if (tile >= 2) {
                    ok = warp_wait(&pv_done[pb], ((tile - 2) >> 1) & 1u);
                    if (!ok) break;
                }
                if (warp_rescale && j > 0) {  // O may be touched once P V of the tile before has been added
                    ok = warp_wait(&pv_done[pb ^ 1u], ((tile - 1) >> 1) & 1u);
                    if (!ok) break;
                    tc_fence_after();
#pragma unroll 1
                    for (int c0 = 128 * hf; c0 < 128 * hf + 128; c0 += 32) {
                        float o[32];
                        tmem_ld32(lane_base + TM_O + c0, o);
                        tc_wait_ld();
#pragma unroll
                        for (int i = 0; i < 32; i++) o[i] *= corr;
                        tmem_st32(lane_base + TM_O + c0, *reinterpret_cast<float(*)[32]>(&o[0]));
                    }
                }
                if (live) tmem_st32(lane_base + TM_P + pb * 64 + 32 * hf, *reinterpret_cast<float(*)[32]>(&pk[0]));
                tc_wait_st();
                if (walk.own && col0 + SP_N > walk.len) {
                    // Rows of the tile at and beyond the sequence's end carry weight zero, but 0 * NaN is NaN: whatever
                    // the cache holds there is cleared before the product.  (The last tile of the segment: its V
                    // granules are the last four; they cannot be refilled before the product that this thread allows.)
                    const unsigned g_end = 8 * (n + walk.nt);
                    for (int r = 0; r < 4; r++) {
                        const unsigned gidx = g_end - 4 + r, st = gidx % SP_GRAN;
                        const int bad = max(0, walk.len - col0 - 32 * r);  // first row of the granule to clear
                        if (bad >= 32) continue;
                        ok = warp_wait(&full[st], (gidx / SP_GRAN) & 1u);
                        if (!ok) break;
                        for (int i = bad * 8 + tid; i < 32 * 8; i += 256)
#pragma unroll
                            for (int d = 0; d < 4; d++)
                                *reinterpret_cast<uint4 *>(smem + SP_OFF_RING + st * GRAN_BYTES + d * 4096 + i * 16) =
                                    make_uint4(0u, 0u, 0u, 0u);
                    }
                    if (!ok) break;
                    fence_proxy_async_smem();
                }
                tc_fence_before();
                warp_arrive(&p_ready[pb]);
            }
            if (!ok) break;
            // ---- the segment's partial ----
            n += walk.nt;
            ok = warp_wait(&pv_done[(n - 1) & 1u], ((n - 1) >> 1) & 1u);
            if (!ok) break;
            tc_fence_after();
            if (live) {
                ok = pair_sync();  // the exchange area may still be read by the other half
                if (!ok) break;
                xl[hf * SP_M + row] = l_run;
                ok = pair_sync();
                if (!ok) break;
                l_run += xl[(hf ^ 1) * SP_M + row];
                const size_t slot = (size_t)walk.unit + blockIdx.x;
                const size_t prow = walk.own ? ((size_t)p.Hkv * p.prefix_mtiles + gridDim.x) * SP_M + slot * p.own_rows + row
                                             : slot * SP_M + row;
                const bool valid = row < rows;
                if (valid && hf == 0) {
                    p.part_m[prow] = m_run == -INFINITY ? -INFINITY : m_run * sl2;
                    p.part_l[prow] = l_run;
                }
                float *dst = p.part_o + prow * HEAD_DIM;
#pragma unroll 1
                for (int c0 = 128 * hf; c0 < 128 * hf + 128; c0 += 32) {
                    float o[32];
                    tmem_ld32(lane_base + TM_O + c0, o);
                    tc_wait_ld();
                    if (valid)
#pragma unroll
                        for (int i = 0; i < 32; i += 4)
                            *reinterpret_cast<float4 *>(dst + c0 + i) = make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
                }
                ok = pair_sync();  // the other half has read the row sums
            }
        }
        if (!ok && lane == 0) *s_fail = 1;
    }
    tc_fence_before();
    __syncthreads();
    if (tid == 0 && *s_fail) atomicOr(p.status, STATUS_TMA_TIMEOUT);
    // on the ordinary path every granule has been used; after a failure the copies in flight land before the CTA leaves
    if (warp == 9 && lane == 0 && *s_fail)
        for (unsigned k = gi > SP_GRAN ? gi - SP_GRAN : 0; k < gi; k++) mbar_wait_bounded(&full[k % SP_GRAN], (k / SP_GRAN) & 1u);
    if (warp == 0) tmem_dealloc(tmem, SP_TMEM_COLS);
}

// One CTA (128 threads, two dims each) per query row: joins the partials of the prefix unit and of the own unit in the
// order of the tile sequence, applies the gate.
__global__ void __launch_bounds__(128) shared_attn_merge_kernel(const SharedAttnParams p) {
    const int tid = threadIdx.x;
    const int h = blockIdx.x % p.H, bt = blockIdx.x / p.H;
    const int t = bt % p.T, b = bt / p.T;
    const int hk = h / p.group, hg = h - hk * p.group;
    const int run = p.plan[0];
    const size_t own_base = ((size_t)p.Hkv * p.prefix_mtiles + p.grid) * SP_M;
    // prefix: partials [0, np); own: partials [np, np + no)
    int np = 0, no = 0;
    size_t prow = 0, orow = 0;
    if (p.prefix_tiles > 0) {
        const int idx = bt * p.group + hg, mt = idx / SP_M;
        const int unit = hk * p.prefix_mtiles + mt;
        const int first = unit * p.prefix_tiles / run, last = ((unit + 1) * p.prefix_tiles - 1) / run;
        np = last - first + 1;
        prow = ((size_t)unit + first) * SP_M + (idx - mt * SP_M);
    }
    const int nt = own_tiles(p, b);
    if (nt > 0) {
        const int idx = t * p.group + hg, mt = idx / SP_M;
        const int u = hk * p.own_mtiles + mt;
        const int begin = p.plan[8 + b] + u * nt;
        const int first = begin / run, last = (begin + nt - 1) / run;
        no = last - first + 1;
        orow = own_base + ((size_t)b * p.Hkv * p.own_mtiles + u + first) * p.own_rows + (idx - mt * SP_M);
    }
    auto part_row = [&](int c) -> size_t { return c < np ? prow + (size_t)c * SP_M : orow + (size_t)(c - np) * p.own_rows; };
    const int parts = np + no;
    float M = -INFINITY;
    for (int c = 0; c < parts; c++) M = fmaxf(M, p.part_m[part_row(c)]);
    float L = 0.0f;
    float2 acc = make_float2(0.0f, 0.0f);
#pragma unroll 4
    for (int c = 0; c < parts; c++) {
        const size_t r = part_row(c);
        const float m = p.part_m[r];
        const float w = m == -INFINITY ? 0.0f : ex2_approx(m - M);
        const float2 o = *reinterpret_cast<const float2 *>(p.part_o + r * HEAD_DIM + 2 * tid);
        L += w * p.part_l[r];
        if (w != 0.0f) {  // a partial without weight contributes nothing, whatever it holds
            acc.x = fmaf(w, o.x, acc.x);
            acc.y = fmaf(w, o.y, acc.y);
        }
    }
    const bool none = M == -INFINITY;
    const float inv = none ? 0.0f : 1.0f / L;
    acc.x *= inv;
    acc.y *= inv;
    if (p.gate) {
        const uint32_t gb = *reinterpret_cast<const uint32_t *>(p.gate + (int64_t)b * p.g_seq + (int64_t)t * p.g_token +
                                                                (int64_t)h * p.g_head + 2 * tid);
        acc.x *= 1.0f / (1.0f + expf(-bf16_bits_to_f32((uint16_t)(gb & 0xffffu))));
        acc.y *= 1.0f / (1.0f + expf(-bf16_bits_to_f32((uint16_t)(gb >> 16))));
    }
    *reinterpret_cast<uint32_t *>(p.out + (size_t)blockIdx.x * HEAD_DIM + 2 * tid) = pack_bf16x2(acc.x, acc.y);
    if (p.lse && tid == 0) p.lse[blockIdx.x] = none ? -INFINITY : (M + log2f(L)) * 0.6931471805599453f;
}

}  // namespace

cudaError_t shared_prefix_attn_configure() {
    return cudaFuncSetAttribute(shared_prefix_attn_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)SP_SMEM);
}

cudaError_t launch_shared_prefix_attn(const CUtensorMap &pk, const CUtensorMap &pv, const CUtensorMap &ok,
                                      const CUtensorMap &ov, const SharedAttnParams &p, cudaStream_t stream) {
    if (p.B <= 0) return cudaSuccess;
    shared_prefix_attn_kernel<<<p.grid, SP_THREADS, SP_SMEM, stream>>>(pk, pv, ok, ov, p);
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    shared_attn_merge_kernel<<<(unsigned)(p.B * p.T * p.H), 128, 0, stream>>>(p);
    return cudaGetLastError();
}

}  // namespace mfc
