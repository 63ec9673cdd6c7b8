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
// Work split: the 128-row tiles of the prefix units (kv head, 128 query rows) form one sequence, those of the own units
// (sequence, kv head) another; both are cut into equal runs for the persistent CTAs, one per SM (see Plan).  A CTA writes one
// un-normalised partial (o, m, l) per unit it touches; the merge kernel joins the partials of a query row by log-sum-exp,
// in a fixed order, and applies the gate.  Lengths are read on the device.
//
// CTA (320 threads): warps 0-7 softmax (thread = query row x half of the 128 columns), warp 8 issues every tcgen05.mma,
// warp 9 every TMA load.  Shared memory: Q 64 KiB and a ring of five 32 KiB granules that K and V share in the order in
// which the tensor core takes them (K: 128 dims x 128 rows, V: 256 dims x 64 rows).  Tensor memory (512 columns): O 256,
// S 128, P twice 64 (bf16, the A operand of P V straight from tensor memory).  S is free again as soon as the softmax
// has read it, so Q K^T of tile j+1 runs under the softmax of tile j, and P V of tile j under that of tile j+1.  The
// reference that a row's exponents are taken against is the maximum of its first tile and moves, with a rescaling of O,
// only when some exponential would exceed 2^32 (bf16 has the exponents to spare, so has fp32 for 2^30 rows with V below 2^64,
// and no digits are lost):
// so no maximum stands before the exponentials of a tile; its rows' maxima are taken along with them, and the two halves
// of a row ask one another with one barrier reduction whether either must move, which redoes the tile.  P is rounded to
// bf16 (the type of V: both operands of one instruction have the same type); the row sums l are taken before that rounding.
// Every mbarrier wait is bounded.  When one runs out the CTA sets a flag that ends all its waits; the softmax warps still
// walk their tiles, without work, so that the block barriers among them stay paired; then a status bit is set, the CTA
// waits for its copies in flight, frees its tensor memory and leaves.
#include <math.h>

#include "common.cuh"
#include "kernels.h"
#include "tcgen05.cuh"

namespace mfc {

namespace {

constexpr int SP_M = SHARED_ATTN_M;
constexpr int SP_N = SHARED_ATTN_N;
constexpr int SP_SOFT = 8;                                 // softmax warps: two per quadrant of tensor memory
constexpr int SP_THREADS = 32 * (SP_SOFT + 2);
constexpr int SP_GRAN = 5;                                 // granules of the K/V ring
constexpr uint32_t GRAN_BYTES = 32768;
constexpr uint32_t SP_Q_BOX = SP_M * 128;                  // 64 dims of 128 query rows
constexpr uint32_t SP_OFF_RING = 4 * SP_Q_BOX;
constexpr uint32_t SP_OFF_XM = SP_OFF_RING + SP_GRAN * GRAN_BYTES;  // row-maximum / row-sum exchange
constexpr uint32_t SP_OFF_BAR = SP_OFF_XM + 1024;
constexpr uint32_t SP_SMEM = SP_OFF_BAR + 512 + 1024;      // + alignment slack
static_assert(SP_SMEM <= 232448, "shared memory of an SM");
constexpr float LOG2E_SP = 1.4426950408889634f;

constexpr uint32_t SP_TMEM_COLS = 512;
constexpr uint32_t TM_O = 0, TM_S = 256, TM_P = 384;       // P: two buffers of 64 columns

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

// the 64 threads of a quadrant's rows: barrier, and whether any of them passed a non-zero value
__device__ __forceinline__ bool quad_any(int quad, bool v) {
    uint32_t r;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.u32 p, %1, 0;\n\t"
        "barrier.cta.red.or.pred q, %2, 64, p;\n\t"
        "selp.u32 %0, 1, 0, q;\n\t}"
        : "=r"(r)
        : "r"((uint32_t)v), "r"(quad + 1)
        : "memory");
    return r != 0;
}
// One lane of a converged warp, always the same.  The warps that issue TMA and tensor-core instructions run their loops
// as whole warps and let this lane issue: addresses and descriptors are then uniform values for the compiler (with a lane-0
// branch around the whole loop the largest case took 364 us where this took 342).
__device__ __forceinline__ bool elect_one() {
    uint32_t r;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "elect.sync _|p, 0xffffffff;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(r)::"memory");
    return r != 0;
}
__device__ __forceinline__ void quad_sync(int quad) { asm volatile("barrier.cta.sync %0, 64;" ::"r"(quad + 1) : "memory"); }

__device__ __forceinline__ int own_len(const SharedAttnParams &p, int b) {
    const int n = p.lens[b];
    return (n < 0 || n > p.own_cap) ? 0 : n;
}
__device__ __forceinline__ int own_tiles(const SharedAttnParams &p, int b) { return (own_len(p, b) + SP_N - 1) / SP_N; }

// How a call's tiles are dealt to CTAs: the prefix tiles in runs of `run` to the CTAs 0, 1, ..., the own tiles in runs of
// `own_run` to the CTAs grid - 1, grid - 2, ....  Either every CTA takes a run of both, or the first CTAs take prefix tiles
// only and the others own tiles only.  Prefix runs are cut within the units where that is shorter (a unit's place in the
// sequence is then `unit_place` tiles, whole runs, and no CTA takes parts of two units: 37 x 3 tokens over 10007 rows 49 ->
// 44 us).  The choice minimises the longest CTA, counted in prefix tiles (2.3 thousand cycles): an own tile, whose rows come
// from HBM and not from L2, is a quarter more; a further prefix segment 3 (writing the partial of 128 rows takes 4.3
// thousand cycles), a further own segment 1 and its share of the same.  A split has to win by a fifteenth (64 x 4 tokens
// over 32768 rows, where the estimates meet: 239 us dealt to all, 243 us split).  Elsewhere the two lie further apart (dealt to
// all, split: 16 x 8192 rows 28.2, 22.7 us; 37 x 3 tokens x 10007 46.5, 40.9; 96 x 4 tokens x 4000 99, 82; 8 x 4 tokens x 4096
// 23.5, 18.7).  Every warp computes the plan by itself from the lengths, 31 splits, one a lane.
struct Plan {
    int run, unit_place, own_run;
    int total_own;
    int chunk, lane_begin;  // lane l covers sequences [l * chunk, ...): its first own tile
};
constexpr float SP_SEG_COST = 3.0f, SP_OWN_TILE_COST = 1.25f, SP_BOTH_BIAS = 0.93f;
__device__ __forceinline__ int ceil_div(int a, int b) { return (int)(((unsigned)a + (unsigned)b - 1u) / (unsigned)b); }

__device__ __forceinline__ Plan make_plan(const SharedAttnParams &p, bool *bad) {
    const int lane = threadIdx.x & 31;
    const int per = p.Hkv * p.own_mtiles, units_p = p.Hkv * p.prefix_mtiles;
    Plan pl;
    pl.chunk = (p.B + 31) / 32;
    const int b_lo = min(lane * pl.chunk, p.B), b_hi = min(b_lo + pl.chunk, p.B);
    int mine = 0, some = 0;
    bool off = false;
    for (int b = b_lo; b < b_hi; b++) {
        const int nt = own_tiles(p, b);
        mine += per * nt;
        some += nt > 0;
        off |= p.lens[b] < 0 || p.lens[b] > p.own_cap;
    }
    *bad = off;
    int inc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += up;
    }
    pl.lane_begin = inc - mine;
    pl.total_own = __shfl_sync(0xffffffffu, inc, 31);
    const int units_o = per * (int)__reduce_add_sync(0xffffffffu, some);
    // the prefix on at most c CTAs: cost of the longest, run length, tiles a unit occupies, CTAs used
    auto prefix_cost = [&](int c, int &run, int &place, int &used) {
        run = ceil_div(units_p * p.prefix_tiles, c);
        place = p.prefix_tiles;
        used = c;
        float t = (float)run + SP_SEG_COST * (float)min(run - 1, ceil_div(units_p, c));
        if (c >= units_p) {
            const int r = ceil_div(p.prefix_tiles, (int)((unsigned)c / (unsigned)units_p));
            if ((float)r <= t) {
                const int parts = ceil_div(p.prefix_tiles, r);
                t = (float)r;
                run = r;
                place = parts * r;
                used = parts * units_p;
            }
        }
        return t;
    };
    const float own_seg = 1.0f + SP_SEG_COST * (float)p.own_rows / (float)SP_M;
    auto own_cost = [&](int c, int &run) {
        run = max(1, ceil_div(pl.total_own, c));
        return SP_OWN_TILE_COST * (float)run + own_seg * (float)min(run - 1, ceil_div(units_o, c));
    };
    // lane 31: every CTA takes both kinds; the others: c CTAs for the prefix, the rest for the own rows.  (A call with one
    // kind only is decided by lane 31 alone.)
    const bool both = lane == 31;
    const int c = both ? p.grid : (lane + 1) * p.grid / 32;
    int run = 1, place = p.prefix_tiles, used = 0, own_run = 1;
    float t = INFINITY;
    if (both || (c >= 1 && c < p.grid && p.prefix_tiles > 0 && pl.total_own > 0)) {
        const float tp = p.prefix_tiles > 0 ? prefix_cost(c, run, place, used) : 0.0f;
        const float to = own_cost(both ? p.grid : p.grid - used, own_run);
        t = both ? SP_BOTH_BIAS * (tp + to + own_seg) : fmaxf(tp, to);
    }
    // the least cost, the smallest split among equals
    const unsigned least = __reduce_min_sync(0xffffffffu, __float_as_uint(t));
    const int src = __ffs(__ballot_sync(0xffffffffu, __float_as_uint(t) == least)) - 1;
    pl.run = __shfl_sync(0xffffffffu, run, src);
    pl.unit_place = __shfl_sync(0xffffffffu, place, src);
    pl.own_run = __shfl_sync(0xffffffffu, own_run, src);
    return pl;
}
// A segment: the tiles [t0, t0 + nt) of one unit.  Every role of a CTA walks the same segments by itself: first its run
// of the prefix tiles, then its run of the own tiles.
struct Walk {
    int at, end, place;   // prefix tiles left to this CTA, tiles that a unit occupies
    int own_at, own_end;  // own tiles left to it
    int b, begin;         // sequence at hand and its first own tile
    // the segment at hand
    bool own;
    int unit;             // index among the units of its kind
    int hk, mt;           // kv head, tile of 128 query rows
    int t0, nt, len;      // len: rows of the unit

    __device__ __forceinline__ bool next(const SharedAttnParams &p) {
        if (at < end) {
            own = false;
            unit = at / place;
            hk = unit / p.prefix_mtiles;
            mt = unit - hk * p.prefix_mtiles;
            t0 = at - unit * place;
            nt = min(p.prefix_tiles - t0, end - at);
            len = p.prefix_len;
            at = t0 + nt == p.prefix_tiles ? (unit + 1) * place : at + nt;
            return true;
        }
        if (own_at >= own_end) return false;
        const int per = p.Hkv * p.own_mtiles;
        int nb = own_tiles(p, b);
        while (own_at >= begin + per * nb) {
            begin += per * nb;
            b++;
            nb = own_tiles(p, b);
        }
        own = true;
        const int u = (own_at - begin) / nb;
        hk = u / p.own_mtiles;
        mt = u - hk * p.own_mtiles;
        unit = b * per + u;
        t0 = own_at - begin - u * nb;
        nt = min(nb - t0, own_end - own_at);
        len = own_len(p, b);
        own_at += nt;
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
    // (bars[11 .. 13] and bars[16] count the softmax warps, the others one arrival)
    uint64_t *full = bars;                  // [5] TMA: granule landed
    uint64_t *empty = bars + SP_GRAN;       // [5] tcgen05.commit: the products that read the granule are done
    uint64_t *s_ready = bars + 10;          // tcgen05.commit: scores of a tile are in tensor memory
    uint64_t *s_read = bars + 11;           // softmax warps: scores are in registers
    uint64_t *p_ready = bars + 12;          // [2] softmax warps: P of a tile is in tensor memory, O may be added to
    uint64_t *pv_done = bars + 14;          // [2] tcgen05.commit: P V of a tile has been accumulated
    uint64_t *q_ready = bars + 16;          // softmax warps: the segment's Q is in shared memory
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + 17);
    volatile int *s_fail = reinterpret_cast<volatile int *>(bars + 18);
    uint64_t *drained = bars + 19;          // tcgen05.commit, after a failure: the products in flight are done

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    if (warp == SP_SOFT) {
        tmem_alloc(tmem_slot, SP_TMEM_COLS);
        tmem_relinquish();
    }
    if (warp == SP_SOFT + 1) {
        if (lane == 20) {
            prefetch_tmap(&pk_map);
            prefetch_tmap(&pv_map);
            prefetch_tmap(&ok_map);
            prefetch_tmap(&ov_map);
        }
        if (lane < 17) mbar_init(&bars[lane], (lane >= 11 && lane <= 13) || lane == 16 ? SP_SOFT : 1);
        if (lane == 17) *s_fail = 0;
        if (lane == 19) mbar_init(drained, 1);
        mbar_fence_init();
    }
    __syncwarp();
    dependency_wait();
    // ---- every warp by itself: the plan, this CTA's runs, its first sequence ----
    const int own_cta = (int)gridDim.x - 1 - (int)blockIdx.x;
    Walk walk;
    {
        bool bad;
        const Plan pl = make_plan(p, &bad);
        if (bad && blockIdx.x == 0 && warp == 0) atomicOr(p.status, STATUS_BAD_ITEM);
        const int total_p = p.Hkv * p.prefix_mtiles * pl.unit_place;
        walk.place = pl.unit_place;
        walk.at = (int)min((long long)blockIdx.x * pl.run, (long long)total_p);
        walk.end = min(walk.at + pl.run, total_p);
        walk.own_at = (int)min((long long)own_cta * pl.own_run, (long long)pl.total_own);
        walk.own_end = min(walk.own_at + pl.own_run, pl.total_own);
        // the last lane whose sequences begin at or before the first own tile; next() walks on from there
        const unsigned starts = __ballot_sync(0xffffffffu, pl.lane_begin <= walk.own_at);
        const int src = 31 - __clz(starts);
        walk.b = src * pl.chunk;
        walk.begin = __shfl_sync(0xffffffffu, pl.lane_begin, src);
        if (blockIdx.x == 0 && warp == 2) {  // for the merge kernel
            if (lane == 0) {
                p.plan[0] = pl.run;
                p.plan[1] = pl.own_run;
                p.plan[2] = pl.unit_place;
            }
            int first = pl.lane_begin;
            for (int b = min(lane * pl.chunk, p.B); b < min((lane + 1) * pl.chunk, p.B); b++) {
                p.plan[8 + b] = first;
                first += p.Hkv * p.own_mtiles * own_tiles(p, b);
            }
        }
    }
    // Q of a segment: softmax warp w copies 16 rows, one 512-byte row per instruction, without registers in between; rows
    // without a query are zero.  The copies are complete, for this thread, after q_landed().
    const int tg = p.T * p.group;
    auto request_q = [&](const Walk &w) {
        const int rows = w.own ? min(SP_M, tg - w.mt * SP_M) : min(SP_M, p.B * tg - w.mt * SP_M);
        int64_t off = 0;  // lane i: offset of row 16 * warp + i
        const int r = 16 * warp + (lane & 15);
        if (r < rows) {
            const int idx = w.mt * SP_M + r;
            const int bt = idx / p.group, hg = idx - bt * p.group;
            const int b = w.own ? w.b : bt / p.T, t = w.own ? bt : bt - b * p.T;
            off = (int64_t)b * p.q_seq + (int64_t)t * p.q_token + (int64_t)(w.hk * p.group + hg) * p.q_head;
        }
        const uint32_t qb = smem_u32(smem + (lane >> 3) * SP_Q_BOX + 16 * warp * 128);
#pragma unroll 4
        for (int i = 0; i < 16; i++) {
            const int64_t o = __shfl_sync(0xffffffffu, off, i);
            const uint32_t bytes = 16 * warp + i < rows ? 16u : 0u;  // 0: the 16 bytes are filled with zeros
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(qb + i * 128 + (((lane & 7) ^ (i & 7)) << 4)),
                         "l"(p.q + o + 8 * lane), "r"(bytes)
                         : "memory");
        }
    };
    bool more = false;
    if (warp < SP_SOFT) {  // the first segment's queries are on their way while the CTA sets itself up
        more = walk.next(p);
        if (more) request_q(walk);
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    // (only now: a CTA of the next kernel may take tensor memory and then wait for this one, which so has its own already)
    dependency_allow();
    const uint32_t tmem = *tmem_slot;
    // Bounded waits of a whole warp, on one barrier or on three at once (a wait that succeeds at once still costs a round
    // trip to shared memory, so the issuer asks for all it needs in one go).  The failure flag is looked at only after a
    // poll that found nothing.
    auto warp_wait = [&](uint64_t *bar, unsigned parity) -> bool {
        for (unsigned i = 0; i < p.wait_spins; i++) {
            if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
            if (*s_fail) return false;
        }
        return false;
    };
    auto warp_wait3 = [&](uint64_t *b0, unsigned p0, uint64_t *b1, unsigned p1, uint64_t *b2, unsigned p2) -> bool {
        for (unsigned i = 0; i < p.wait_spins; i++) {
            const bool r0 = mbar_try_wait(b0, p0), r1 = mbar_try_wait(b1, p1), r2 = mbar_try_wait(b2, p2);
            if (__all_sync(0xffffffffu, r0 && r1 && r2)) return true;
            if (*s_fail) return false;
        }
        return false;
    };
    bool ok = true;
    unsigned gi = 0;  // granules requested (producer) or consumed (issuer)

    if (warp == SP_SOFT + 1) {
        // ================= producer: one lane issues every TMA load =================
        auto granule = [&]() -> bool {  // waits until the next granule is free
            const unsigned st = gi % SP_GRAN, round = gi / SP_GRAN;
            return round == 0 || warp_wait(&empty[st], (round - 1) & 1u);
        };
        // one request per granule: a request costs its thread about 180 cycles, whatever its size
        auto load_k = [&](const Walk &s, int tile) {  // granule: 128 dims (two 64-dim boxes) of 128 rows
            for (int d = 0; d < 2 && ok; d++) {
                ok = granule();
                if (!ok) break;
                const unsigned st = gi % SP_GRAN;
                if (elect_one()) {
                    mbar_expect_tx(&full[st], GRAN_BYTES);
                    if (!(p.inject_lost_load && blockIdx.x == 0 && gi == 0))
                        tma_load_5d(smem + SP_OFF_RING + st * GRAN_BYTES, s.own ? &ok_map : &pk_map, 0, tile * SP_N, 2 * d, s.hk, s.own ? s.b : 0,
                                &full[st]);
                }
                gi++;
            }
        };
        auto load_v = [&](const Walk &s, int tile) {  // granule: 256 dims (four 64-dim boxes) of 64 rows
            for (int r = 0; r < 2 && ok; r++) {
                ok = granule();
                if (!ok) break;
                const unsigned st = gi % SP_GRAN;
                if (elect_one()) {
                    mbar_expect_tx(&full[st], GRAN_BYTES);
                    tma_load_5d(smem + SP_OFF_RING + st * GRAN_BYTES, s.own ? &ov_map : &pv_map, 0, tile * SP_N + r * 64, 0, s.hk,
                                s.own ? s.b : 0, &full[st]);
                }
                gi++;
            }
        };
        // The first K rows are asked for beside the query rows, all others behind them: query rows asked for behind every
        // CTA's first 160 KiB came 6 us later.
        bool first = true;
        while (ok && walk.next(p)) {
            load_k(walk, walk.t0);
            if (first && ok) ok = warp_wait(q_ready, 0);
            first = false;
            for (int j = 0; j < walk.nt && ok; j++) {
                if (j + 1 < walk.nt) load_k(walk, walk.t0 + j + 1);
                load_v(walk, walk.t0 + j);
            }
        }
        if (!ok) *s_fail = 1;
    } else if (warp == SP_SOFT) {
        // ================= issuer: one lane drives the tensor core =================
        constexpr uint32_t IDESC_QK = idesc_bf16(SP_N, 0);
        constexpr uint32_t IDESC_PV = idesc_bf16(HEAD_DIM, 1);
        const uint64_t q_desc = smem_desc_sw128(smem_u32(smem), 16, 1024);
        const uint64_t k_desc = smem_desc_sw128(smem_u32(smem + SP_OFF_RING), 16, 1024);
        // V: MN-major; 64-dim boxes 8192 B apart (LBO), 8-row groups 1024 B apart (SBO)
        const uint64_t v_desc = smem_desc_sw128(smem_u32(smem + SP_OFF_RING), 8192, 1024);
        unsigned n = 0;   // tiles so far, over all segments
        unsigned seg = 0;
        auto issue_qk = [&](unsigned tile) -> bool {
            const unsigned sa = gi % SP_GRAN, sb = (gi + 1) % SP_GRAN;
            // s_read: the softmax has taken the scores of the tile before (a phase ahead of the first tile passes at once)
            if (!warp_wait3(s_read, (tile - 1) & 1u, &full[sa], (gi / SP_GRAN) & 1u, &full[sb], ((gi + 1) / SP_GRAN) & 1u)) return false;
            tc_fence_after();
            if (elect_one()) {
#pragma unroll
                for (int d = 0; d < 2; d++) {
                    const uint64_t qd = q_desc + (uint64_t)((2 * d * SP_Q_BOX) >> 4);
                    const uint64_t kd = k_desc + (uint64_t)(((d ? sb : sa) * GRAN_BYTES) >> 4);
#pragma unroll
                    for (int ks = 0; ks < 8; ks++)
                        tc_mma_bf16(tmem + TM_S, qd + (uint64_t)(((ks >> 2) * SP_Q_BOX + (ks & 3) * 32) >> 4),
                                    kd + (uint64_t)(((ks >> 2) * 16384 + (ks & 3) * 32) >> 4), IDESC_QK, d > 0 || ks > 0);
                    tc_commit(&empty[d ? sb : sa]);
                }
                tc_commit(s_ready);
            }
            gi += 2;
            return true;
        };
        while (ok && walk.next(p)) {
            ok = warp_wait(q_ready, seg & 1u);
            if (!ok) break;
            tc_fence_after();
            ok = issue_qk(n);
            for (int j = 0; j < walk.nt && ok; j++) {
                if (j + 1 < walk.nt) ok = issue_qk(n + j + 1);
                const unsigned tile = n + j, pb = tile & 1u;
                const unsigned sa = gi % SP_GRAN, sb = (gi + 1) % SP_GRAN;
                ok = ok && warp_wait3(&p_ready[pb], (tile >> 1) & 1u, &full[sa], (gi / SP_GRAN) & 1u, &full[sb], ((gi + 1) / SP_GRAN) & 1u);
                if (!ok) break;
                tc_fence_after();
                if (elect_one()) {
#pragma unroll
                    for (int r = 0; r < 2; r++) {
                        const uint64_t vd = v_desc + (uint64_t)(((r ? sb : sa) * GRAN_BYTES) >> 4);
                        const uint32_t pa = tmem + TM_P + pb * 64 + r * 32;
#pragma unroll
                        for (int ks = 0; ks < 4; ks++)
                            tc_mma_bf16_ts(tmem + TM_O, pa + ks * 8, vd + (uint64_t)((ks * 2048) >> 4), IDESC_PV, j > 0 || r > 0 || ks > 0);
                        tc_commit(&empty[r ? sb : sa]);
                    }
                    tc_commit(&pv_done[pb]);
                }
                gi += 2;
            }
            n += walk.nt;
            seg++;
        }
        if (!ok) *s_fail = 1;
    } else {
        // ================= softmax warps: thread = (query row, half of the columns) =================
        const int quad = warp & 3, hf = warp >> 2;
        const int row = 32 * quad + lane;  // query row of the tile = lane of tensor memory
        const uint32_t lane_base = tmem + ((uint32_t)(32 * quad) << 16);
        float *xm = reinterpret_cast<float *>(smem + SP_OFF_XM);  // [2 halves][128 rows] row maxima, row sums
        const float sl2 = p.scale * LOG2E_SP;
        auto warp_arrive = [&](uint64_t *bar) {
            __syncwarp();
            if (lane == 0) mbar_arrive(bar);
        };
        auto give_up = [&]() {
            if (lane == 0) *s_fail = 1;
        };
        auto q_landed = [&]() {
            asm volatile("cp.async.wait_all;" ::: "memory");
            fence_proxy_async_smem();
            warp_arrive(q_ready);
        };
        unsigned n = 0;
        if (more) q_landed();
        while (more) {
            const int rows = walk.own ? min(SP_M, tg - walk.mt * SP_M) : min(SP_M, p.B * tg - walk.mt * SP_M);
            // columns of the unit this row sees
            int lim = walk.len;
            if (walk.own) lim = row < rows ? walk.len - (p.T - 1 - (walk.mt * SP_M + row) / p.group) : 0;
            const int safe = walk.own ? walk.len - (p.T - 1) : walk.len;  // columns that every row sees
            const bool live = 32 * quad < rows;                           // some row of this quadrant carries a query
            float m_run = -INFINITY, l_run = 0.0f;  // m_run: reference of the row's exponents; l_run: this thread's half
            for (int j = 0; j < walk.nt; j++) {
                const unsigned tile = n + j, pb = tile & 1u;
                const int col0 = (walk.t0 + j) * SP_N;
                ok = ok && warp_wait(s_ready, tile & 1u);
                if (!ok) give_up();
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
                bool rescale = false;
                uint32_t pk[32];
                if (live) {
                    const int c0 = col0 + 64 * hf;
                    if (col0 + SP_N > safe) {
#pragma unroll
                        for (int c = 0; c < 64; c++)
                            if (c0 + c >= lim) s[c] = -INFINITY;
                    }
                    auto row_max = [&]() {
                        float a = fmaxf(s[0], s[1]), b = fmaxf(s[2], s[3]);
#pragma unroll
                        for (int c = 4; c < 64; c += 4) {
                            a = fmaxf(a, fmaxf(s[c], s[c + 1]));
                            b = fmaxf(b, fmaxf(s[c + 2], s[c + 3]));
                        }
                        return fmaxf(a, b);
                    };
                    auto move_reference = [&](float mx) {  // to the maximum of the row so far
                        xm[hf * SP_M + row] = mx;
                        quad_sync(quad);
                        const float m_new = fmaxf(m_run, fmaxf(mx, xm[(hf ^ 1) * SP_M + row]));
                        corr = m_new == -INFINITY ? 1.0f : ex2_approx((m_run - m_new) * sl2);
                        m_run = m_new;
                        quad_sync(quad);  // the exchange area is free again
                    };
                    if (j == 0) move_reference(row_max());
                    float rs, mx;
                    auto to_p = [&]() {
                        const float mb = m_run == -INFINITY ? 0.0f : m_run * sl2;
                        float r0 = 0.0f, r1 = 0.0f, a = s[0], b = s[1];
#pragma unroll
                        for (int c = 0; c < 64; c += 2) {
                            const float p0 = ex2_approx(fmaf(s[c], sl2, -mb));
                            const float p1 = ex2_approx(fmaf(s[c + 1], sl2, -mb));
                            a = fmaxf(a, s[c]);
                            b = fmaxf(b, s[c + 1]);
                            r0 += p0;
                            r1 += p1;
                            pk[c >> 1] = pack_bf16x2(p0, p1);
                        }
                        rs = r0 + r1;
                        mx = fmaxf(a, b);
                    };
                    to_p();
                    // true as well for the first finite score of a row (m_run = -inf)
                    rescale = quad_any(quad, (mx - m_run) * sl2 > 32.0f);
                    if (rescale) {
                        move_reference(mx);
                        to_p();
                    }
                    l_run = l_run * corr + rs;
                }
                // P buffer pb was last read by P V of tile - 2
                if (tile >= 2) ok = ok && warp_wait(&pv_done[pb], ((tile - 2) >> 1) & 1u);
                if (rescale && j > 0) {  // O may be touched once P V of the tile before has been added
                    ok = ok && warp_wait(&pv_done[pb ^ 1u], ((tile - 1) >> 1) & 1u);
                    tc_fence_after();
                    if (ok)
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
                if (live && ok) tmem_st32(lane_base + TM_P + pb * 64 + 32 * hf, *reinterpret_cast<float(*)[32]>(&pk[0]));
                tc_wait_st();
                if (walk.own && col0 + SP_N > walk.len) {
                    // Rows of the tile at and beyond the sequence's end carry weight zero, but 0 * NaN is NaN: whatever
                    // the cache holds there is cleared before the product.  (The last tile of the segment: its V
                    // granules are the last two; they cannot be refilled before the product that this thread allows.)
                    const unsigned g_end = 4 * (n + walk.nt);
                    for (int r = 0; r < 2; r++) {
                        const unsigned gidx = g_end - 2 + r, st = gidx % SP_GRAN;
                        const int bad = max(0, walk.len - col0 - 64 * r);  // first row of the granule to clear
                        if (bad >= 64) continue;
                        ok = ok && warp_wait(&full[st], (gidx / SP_GRAN) & 1u);
                        if (!ok) break;
                        for (int i = bad * 8 + tid; i < 64 * 8; i += 32 * SP_SOFT)
#pragma unroll
                            for (int d = 0; d < 4; d++)
                                *reinterpret_cast<uint4 *>(smem + SP_OFF_RING + st * GRAN_BYTES + d * 8192 + i * 16) =
                                    make_uint4(0u, 0u, 0u, 0u);
                    }
                    fence_proxy_async_smem();
                }
                if (!ok) give_up();
                tc_fence_before();
                warp_arrive(&p_ready[pb]);
            }
            // ---- the segment's partial; the next segment's Q comes in meanwhile ----
            const Walk seg = walk;
            more = walk.next(p);
            if (more) request_q(walk);  // the products that read Q of this segment are done: their scores have been read
            n += seg.nt;
            ok = ok && warp_wait(&pv_done[(n - 1) & 1u], ((n - 1) >> 1) & 1u);
            if (!ok) give_up();
            tc_fence_after();
            if (more) q_landed();  // its first scores are computed under the stores below
            if (live) {
                xm[hf * SP_M + row] = l_run;
                quad_sync(quad);
                l_run = xm[row] + xm[SP_M + row];
                // [dims / 4][rows of the slot][4]: consecutive lanes (rows) store consecutive 16 bytes
                const size_t slot = (size_t)seg.unit + (seg.own ? own_cta : (int)blockIdx.x);
                const int srows = seg.own ? p.own_rows : SP_M;
                const size_t row0 = seg.own ? ((size_t)p.Hkv * p.prefix_mtiles + gridDim.x) * SP_M + slot * p.own_rows : slot * SP_M;
                const bool valid = ok && row < rows;
                if (valid && hf == 0) {
                    // (a sum that is NaN with no reference found: every score was NaN, which the merge must not leave out)
                    p.part_m[row0 + row] = m_run != -INFINITY ? m_run * sl2 : (l_run == l_run ? -INFINITY : 0.0f);
                    p.part_l[row0 + row] = l_run;
                }
                float4 *dst = reinterpret_cast<float4 *>(p.part_o + row0 * HEAD_DIM) + row;
                if (ok)
#pragma unroll 1
                    for (int c0 = 128 * hf; c0 < 128 * hf + 128; c0 += 32) {
                        float o[32];
                        tmem_ld32(lane_base + TM_O + c0, o);
                        tc_wait_ld();
                        if (valid)
#pragma unroll
                            for (int i = 0; i < 32; i += 4) dst[(size_t)((c0 + i) >> 2) * srows] = make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
                    }
            }
            if (live) quad_sync(quad);  // the exchange area is free again
            tc_fence_before();          // O has been read: P of the next segment's first tile says so to the issuer
        }
    }
    tc_fence_before();
    __syncthreads();
    if (tid == 0 && *s_fail) atomicOr(p.status, STATUS_TMA_TIMEOUT);
    // on the ordinary path every granule has been used; after a failure the copies in flight land before the CTA leaves
    if (warp == SP_SOFT + 1 && lane == 0 && *s_fail)
        for (unsigned k = gi > SP_GRAN ? gi - SP_GRAN : 0; k < gi; k++) mbar_wait_bounded(&full[k % SP_GRAN], (k / SP_GRAN) & 1u, p.wait_spins);
    if (warp == SP_SOFT) {
        if (*s_fail) {  // and so do the products in flight
            if (elect_one()) tc_commit(drained);
            mbar_wait_bounded(drained, 0, p.wait_spins);
            __syncwarp();
        }
        tmem_dealloc(tmem, SP_TMEM_COLS);
    }
}

// Joins the partials of the query rows by log-sum-exp, in a fixed order, and applies the gate.  CTA = 32 consecutive
// query rows of a kv head (lane = row) and 256 / GROUPS of their dims, a warp 32 dims of them.  One group: a warp takes all
// partials (the prefix unit's first, then the own unit's).  Several (few rows, or a long prefix cut for a small batch): group
// g takes the partials g, g + GROUPS, ..., and the groups' results are joined through shared memory.
constexpr int MG_WARPS = 8;
constexpr int MG_DIMS = 32;
constexpr int MG_CTAS = 160;
constexpr int MG_FEW = 12, MG_FEW_BLOCKS = 128;

struct RowParts {
    int np, no;      // partials of the prefix unit and of the own unit
    int pr, orow;    // the row within their slots
    size_t p0, o0;   // first row of the first slot of each
};
// Partials of query row idx of kv head hk.
__device__ __forceinline__ RowParts row_parts(const SharedAttnParams &p, int hk, int idx) {
    RowParts r = {0, 0, 0, 0, 0, 0};
    const int bt = idx / p.group, b = bt / p.T;
    const int run = p.plan[0], own_run = p.plan[1], nt = own_tiles(p, b);
    if (p.prefix_tiles > 0) {
        const int mt = idx / SP_M, unit = hk * p.prefix_mtiles + mt;
        const int place = p.plan[2], first = unit * place / run, last = (unit * place + p.prefix_tiles - 1) / run;
        r.np = last - first + 1;
        r.p0 = ((size_t)unit + first) * SP_M;
        r.pr = idx - mt * SP_M;
    }
    if (nt > 0) {
        const int i = idx - b * p.T * p.group, mt = i / SP_M, u = hk * p.own_mtiles + mt;
        const int begin = p.plan[8 + b] + u * nt;
        const int first = begin / own_run, last = (begin + nt - 1) / own_run;
        r.no = last - first + 1;
        r.o0 = ((size_t)p.Hkv * p.prefix_mtiles + p.grid) * SP_M + ((size_t)b * p.Hkv * p.own_mtiles + u + first) * p.own_rows;
        r.orow = i - mt * SP_M;
    }
    return r;
}
struct Joined {
    float M, L;
    float4 acc[MG_DIMS / 4];
};
// Partials from, from + step, ... of a row, MG_DIMS dims from d0 on.
__device__ __forceinline__ void join_parts(const SharedAttnParams &p, const RowParts &r, int from, int step, int d0, Joined &j) {
    j.M = -INFINITY;
    j.L = 0.0f;
#pragma unroll
    for (int i = 0; i < MG_DIMS / 4; i++) j.acc[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    struct Part {
        float4 o[MG_DIMS / 4];
        float m, l;
    };
    auto load = [&](int c, Part &q) {
        const bool pre = c < r.np;
        const int srows = pre ? SP_M : p.own_rows, row = pre ? r.pr : r.orow;
        const size_t row0 = pre ? r.p0 + (size_t)c * SP_M : r.o0 + (size_t)(c - r.np) * p.own_rows;
        const float4 *src = reinterpret_cast<const float4 *>(p.part_o + row0 * HEAD_DIM) + row;
#pragma unroll
        for (int i = 0; i < MG_DIMS / 4; i++) q.o[i] = src[(size_t)(d0 / 4 + i) * srows];
        q.m = p.part_m[row0 + row];
        q.l = p.part_l[row0 + row];
    };
    auto fold = [&](const Part &q) {
        if (q.m == -INFINITY) return;  // no weight: contributes nothing, whatever it holds
        const float mn = fmaxf(j.M, q.m);
        const float wa = j.M == -INFINITY ? 0.0f : ex2_approx(j.M - mn), wb = ex2_approx(q.m - mn);
        j.M = mn;
        j.L = j.L * wa + q.l * wb;
#pragma unroll
        for (int i = 0; i < MG_DIMS / 4; i++) {
            j.acc[i].x = fmaf(wb, q.o[i].x, j.acc[i].x * wa);
            j.acc[i].y = fmaf(wb, q.o[i].y, j.acc[i].y * wa);
            j.acc[i].z = fmaf(wb, q.o[i].z, j.acc[i].z * wa);
            j.acc[i].w = fmaf(wb, q.o[i].w, j.acc[i].w * wa);
        }
    };
    const int n = r.np + r.no;
    for (int c = from; c < n; c += 2 * step) {  // two partials in flight
        Part a, b;
        load(c, a);
        if (c + step < n) load(c + step, b);
        fold(a);
        if (c + step < n) fold(b);
    }
}
__device__ __forceinline__ float2 gate2(uint32_t bits) {
    return make_float2(1.0f / (1.0f + expf(-bf16_bits_to_f32((uint16_t)(bits & 0xffffu)))),
                       1.0f / (1.0f + expf(-bf16_bits_to_f32((uint16_t)(bits >> 16)))));
}

template <int GROUPS>
__global__ void __launch_bounds__(32 * MG_WARPS, GROUPS > 1 ? 2 : 1) shared_attn_merge_kernel(const SharedAttnParams p) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rows_hk = p.B * p.T * p.group;
    const int blocks_hk = (rows_hk + 31) / 32;
    const int hk = blockIdx.x / blocks_hk, idx0 = (blockIdx.x - hk * blocks_hk) * 32;
    dependency_wait();  // the plan and the partials are written by the kernel before
    RowParts parts = {0, 0, 0, 0, 0, 0};
    if (idx0 + lane < rows_hk) parts = row_parts(p, hk, idx0 + lane);
    if (GROUPS == 1) {
        const int idx = idx0 + lane, d0 = warp * MG_DIMS;
        if (idx >= rows_hk) return;
        const int bt = idx / p.group, h = hk * p.group + (idx - bt * p.group);
        uint4 g[MG_DIMS / 8];
        if (p.gate) {
            const int b = bt / p.T, t = bt - b * p.T;
            const uint4 *gp = reinterpret_cast<const uint4 *>(p.gate + (int64_t)b * p.g_seq + (int64_t)t * p.g_token + (int64_t)h * p.g_head + d0);
#pragma unroll
            for (int i = 0; i < MG_DIMS / 8; i++) g[i] = gp[i];
        }
        Joined j;
        join_parts(p, parts, 0, 1, d0, j);
        const bool none = j.M == -INFINITY;
        const float inv = none ? 0.0f : 1.0f / j.L;
        const size_t orw = (size_t)bt * p.H + h;
        uint4 *dst = reinterpret_cast<uint4 *>(p.out + orw * HEAD_DIM + d0);
#pragma unroll
        for (int i = 0; i < MG_DIMS / 8; i++) {
            const float4 a = j.acc[2 * i], c = j.acc[2 * i + 1];
            float2 x0 = make_float2(a.x * inv, a.y * inv), x1 = make_float2(a.z * inv, a.w * inv);
            float2 x2 = make_float2(c.x * inv, c.y * inv), x3 = make_float2(c.z * inv, c.w * inv);
            if (p.gate) {
                const float2 s0 = gate2(g[i].x), s1 = gate2(g[i].y), s2 = gate2(g[i].z), s3 = gate2(g[i].w);
                x0 = make_float2(x0.x * s0.x, x0.y * s0.y);
                x1 = make_float2(x1.x * s1.x, x1.y * s1.y);
                x2 = make_float2(x2.x * s2.x, x2.y * s2.y);
                x3 = make_float2(x3.x * s3.x, x3.y * s3.y);
            }
            dst[i] = make_uint4(pack_bf16x2(x0.x, x0.y), pack_bf16x2(x1.x, x1.y), pack_bf16x2(x2.x, x2.y), pack_bf16x2(x3.x, x3.y));
        }
        if (p.lse && warp == 0) p.lse[orw] = none ? -INFINITY : (j.M + log2f(j.L)) * 0.6931471805599453f;
    } else {
        __shared__ float s_m[MG_WARPS][32], s_l[MG_WARPS][32];
        __shared__ float4 s_o[MG_WARPS][MG_DIMS / 4][33];
        constexpr int CHUNKS = MG_WARPS / GROUPS;
        Joined j;
        join_parts(p, parts, warp % GROUPS, GROUPS, (blockIdx.y * CHUNKS + warp / GROUPS) * MG_DIMS, j);
        s_m[warp][lane] = j.M;
        s_l[warp][lane] = j.L;
#pragma unroll
        for (int i = 0; i < MG_DIMS / 4; i++) s_o[warp][i][lane] = j.acc[i];
        __syncthreads();
        // thread = (row of the 32, four dims): eight threads write 64 consecutive bytes of a row
        const int row = threadIdx.x >> 3, q4 = threadIdx.x & 7;
        const int idx = idx0 + row;
        if (idx >= rows_hk) return;
        const int bt = idx / p.group, h = hk * p.group + (idx - bt * p.group);
        const size_t orw = (size_t)bt * p.H + h;
#pragma unroll
        for (int chunk = 0; chunk < CHUNKS; chunk++) {
            const int w0 = chunk * GROUPS, d = (blockIdx.y * CHUNKS + chunk) * MG_DIMS + 4 * q4;
            float M = -INFINITY, L = 0.0f;
#pragma unroll
            for (int w = w0; w < w0 + GROUPS; w++) M = fmaxf(M, s_m[w][row]);
            float4 a = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int w = w0; w < w0 + GROUPS; w++) {
                const float m = s_m[w][row];
                if (m == -INFINITY) continue;
                const float wt = ex2_approx(m - M);
                const float4 o = s_o[w][q4][row];
                L += wt * s_l[w][row];
                a.x = fmaf(wt, o.x, a.x);
                a.y = fmaf(wt, o.y, a.y);
                a.z = fmaf(wt, o.z, a.z);
                a.w = fmaf(wt, o.w, a.w);
            }
            const bool none = M == -INFINITY;
            const float inv = none ? 0.0f : 1.0f / L;
            float2 x0 = make_float2(a.x * inv, a.y * inv), x1 = make_float2(a.z * inv, a.w * inv);
            if (p.gate) {
                const int b = bt / p.T, t = bt - b * p.T;
                const uint2 g = *reinterpret_cast<const uint2 *>(p.gate + (int64_t)b * p.g_seq + (int64_t)t * p.g_token + (int64_t)h * p.g_head + d);
                const float2 s0 = gate2(g.x), s1 = gate2(g.y);
                x0 = make_float2(x0.x * s0.x, x0.y * s0.y);
                x1 = make_float2(x1.x * s1.x, x1.y * s1.y);
            }
            *reinterpret_cast<uint2 *>(p.out + orw * HEAD_DIM + d) = make_uint2(pack_bf16x2(x0.x, x0.y), pack_bf16x2(x1.x, x1.y));
            if (p.lse && d == 0) p.lse[orw] = none ? -INFINITY : (M + log2f(L)) * 0.6931471805599453f;
        }
    }
}

}  // namespace

cudaError_t shared_prefix_attn_configure() {
    return cudaFuncSetAttribute(shared_prefix_attn_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)SP_SMEM);
}

cudaError_t launch_shared_prefix_attn(const CUtensorMap &pk, const CUtensorMap &pv, const CUtensorMap &ok,
                                      const CUtensorMap &ov, const SharedAttnParams &p, cudaStream_t stream) {
    if (p.B <= 0) return cudaSuccess;
    cudaError_t e = launch_dependent(shared_prefix_attn_kernel, dim3((unsigned)p.grid), SP_THREADS, SP_SMEM, stream, 1u, pk, pv, ok, ov, p);
    if (e != cudaSuccess) return e;
    // partials a row has at most, about: the CTAs a unit is spread over, of the prefix and of the own rows
    const int64_t units_p = (int64_t)p.Hkv * p.prefix_mtiles, units_o = (int64_t)p.B * p.Hkv * p.own_mtiles;
    const int64_t own_t = (p.own_cap + SP_N - 1) / SP_N, np = p.grid / units_p + 2, no = p.grid / units_o + 2;
    // One group a row where the partials are few and the rows fill the GPU (32 x 4 tokens, 300 + 2048 rows: 33.5 us against 35.0
    // in groups; 96 x 4 tokens, 4000 + 1000: 82.5 against 85.0).  With few rows the groups spread them over more SMs, with many
    // partials they shorten the chain of each (8 x 4 tokens x 4096 rows: 18.7 us in groups, 25.6 with one; 4 x 20000: 21.0, 44.9;
    // 48 x 2 tokens of 16 heads x 16000: 37.2, 40.8).
    const int64_t blocks = (int64_t)p.Hkv * ((p.B * p.T * p.group + 31) / 32);
    const bool few = (np < p.prefix_tiles ? np : p.prefix_tiles) + (no < own_t ? no : own_t) <= MG_FEW && blocks >= MG_FEW_BLOCKS;
    // otherwise as few groups as give a CTA to every SM: fewer waves of CTAs, each with a chain of latencies of its own (1332
    // rows of a head, eight partials: 42.5, 43.2, 43.9 us for the call with 2, 4, 8 groups).  MG_CTAS: somewhat more than the 148
    // SMs of a B200.
    int groups = few ? 1 : 8;
    while (groups > 2 && blocks * (groups / 2) >= MG_CTAS) groups /= 2;
    const dim3 grid((unsigned)blocks, (unsigned)groups);
    if (groups == 1) return launch_dependent(shared_attn_merge_kernel<1>, grid, 32 * MG_WARPS, 0, stream, 1u, p);
    if (groups == 2) return launch_dependent(shared_attn_merge_kernel<2>, grid, 32 * MG_WARPS, 0, stream, 1u, p);
    if (groups == 4) return launch_dependent(shared_attn_merge_kernel<4>, grid, 32 * MG_WARPS, 0, stream, 1u, p);
    return launch_dependent(shared_attn_merge_kernel<8>, grid, 32 * MG_WARPS, 0, stream, 1u, p);
}

}  // namespace mfc
