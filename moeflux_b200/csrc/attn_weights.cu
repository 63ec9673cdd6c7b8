// Attention weight that every cached row received in a step, added to its running sum (no counterpart in the reference).
//
//   weights[b][hk][j] = decay * weights[b][hk][j] + sum_{t, heads of hk that see j} exp(scale q.k_j - lse)
//
// With the lse of the attention call at hand this is one pass over K: 512 bytes read per row beside 8 for the sum, and
// 512 flop per row and query, so HBM-bound up to about 64 queries per kv head.  The cached rows are the M index of
// mma.sync m16n8k16 and the queries its N index: a warp loads 16 rows straight from global memory into A fragments (a
// lane's 16 bytes of a row are the k slots it owns in two instructions; the contraction does not care about the order of
// k as long as both operands agree) and runs all queries past them out of shared memory, eight columns at a time, so no
// query slot of a group of 12 or 5 heads is wasted on a multiple of 16, the sum over queries stays in a lane's registers
// and is finished by two shuffles.  The next 16 rows are in flight meanwhile.
//
// Work split: the 64-row blocks of all (sequence, kv head) units form one sequence, cut into equal runs, one CTA each,
// across unit boundaries; lengths are read on the device, every CTA finds its place by a scan over them.  Every row
// belongs to exactly one warp: no atomics, the same bits every time.
#include <math.h>

#include "common.cuh"
#include "kernels.h"

namespace mfc {

namespace {

constexpr int AW_THREADS = 128;
constexpr int AW_WARPS = AW_THREADS / 32;
constexpr int AW_BLOCK = 16 * AW_WARPS;  // rows of a block: 16 per warp
constexpr int AW_Q_STRIDE = HEAD_DIM + 32;  // bf16; 576 bytes: the eight lanes of a 128-bit phase touch all banks
constexpr int AW_CTAS_PER_SM = 3;
constexpr float LOG2E_AW = 1.4426950408889634f;

__global__ void __launch_bounds__(AW_THREADS, AW_CTAS_PER_SM) attn_weights_kernel(const AttnWeightsParams p) {
    extern __shared__ __align__(16) uint8_t smem[];
    const int nq = p.T * p.group, nqp = (nq + 7) & ~7;  // queries of a unit, padded to the N of the instruction
    __nv_bfloat16 *s_q = reinterpret_cast<__nv_bfloat16 *>(smem);
    float *s_lse = reinterpret_cast<float *>(smem + (size_t)nqp * AW_Q_STRIDE * 2);
    int *s_lim = reinterpret_cast<int *>(s_lse + nqp);
    __shared__ long long s_scan[AW_WARPS];
    __shared__ int s_b0;
    __shared__ long long s_begin0;

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int g = lane >> 2, t = lane & 3;
    auto len_of = [&](int b) {
        const int n = p.lens[b];
        return (n < 0 || n > p.cap) ? 0 : n;
    };
    auto blocks_of = [&](int b) -> long long { return (long long)p.Hkv * ((len_of(b) + AW_BLOCK - 1) / AW_BLOCK); };

    // ---- this CTA's run of the launch-wide block sequence ----
    const int per = (p.B + AW_THREADS - 1) / AW_THREADS;
    const int b_lo = min(tid * per, p.B), b_hi = min(b_lo + per, p.B);
    long long mine = 0;
    bool bad = false;
    for (int b = b_lo; b < b_hi; b++) {
        mine += blocks_of(b);
        bad |= p.lens[b] < 0 || p.lens[b] > p.cap;
    }
    if (bad && blockIdx.x == 0) atomicOr(p.status, STATUS_BAD_ITEM);
    long long inc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long up = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += up;
    }
    if (lane == 31) s_scan[warp] = inc;
    __syncthreads();
    long long base = 0, total = 0;
#pragma unroll
    for (int w = 0; w < AW_WARPS; w++) {
        if (w < warp) base += s_scan[w];
        total += s_scan[w];
    }
    const long long run = (total + gridDim.x - 1) / gridDim.x;
    long long at = (long long)blockIdx.x * run;
    const long long end = min(at + run, total);
    if (at >= end) return;
    long long first = base + inc - mine;
    for (int b = b_lo; b < b_hi; b++) {
        const long long n = blocks_of(b);
        if (at >= first && at < first + n) {
            s_b0 = b;
            s_begin0 = first;
        }
        first += n;
    }
    __syncthreads();
    int b = s_b0;
    long long begin = s_begin0;
    const float sl2 = p.scale * LOG2E_AW;

    while (at < end) {
        while (at >= begin + blocks_of(b)) {
            begin += blocks_of(b);
            b++;
        }
        const int len = len_of(b);
        const int nb = (len + AW_BLOCK - 1) / AW_BLOCK;
        const int hk = (int)((at - begin) / nb);
        const int blk0 = (int)((at - begin) - (long long)hk * nb);
        const int blk1 = (int)min((long long)nb, blk0 + (end - at));

        const __nv_bfloat16 *kbase = p.k + (int64_t)b * p.k_seq + (int64_t)hk * p.k_head;
        uint4 kf[2][16];  // [buffer][32-dim block * 2 + row half]
        auto load_rows = [&](uint4 (&f)[16], int blk) {
            const int row = blk * AW_BLOCK + warp * 16 + g;
            // rows past the end are read as the last row and masked
            const __nv_bfloat16 *ra = kbase + (int64_t)min(row, len - 1) * p.k_row + 8 * t;
            const __nv_bfloat16 *rb = kbase + (int64_t)min(row + 8, len - 1) * p.k_row + 8 * t;
#pragma unroll
            for (int kb = 0; kb < 8; kb++) {
                f[2 * kb] = __ldg(reinterpret_cast<const uint4 *>(ra + 32 * kb));
                f[2 * kb + 1] = __ldg(reinterpret_cast<const uint4 *>(rb + 32 * kb));
            }
        };
        load_rows(kf[0], blk0);

        // ---- the unit's queries: rows t * group + head of the group ----
        for (int i = tid; i < nqp * 32; i += AW_THREADS) {
            const int r = i >> 5, c = i & 31;
            uint4 v = make_uint4(0u, 0u, 0u, 0u);
            if (r < nq)
                v = *reinterpret_cast<const uint4 *>(p.q + (int64_t)b * p.q_seq + (int64_t)(r / p.group) * p.q_token +
                                                     (int64_t)(hk * p.group + r % p.group) * p.q_head + 8 * c);
            *reinterpret_cast<uint4 *>(s_q + r * AW_Q_STRIDE + 8 * c) = v;
        }
        for (int r = tid; r < nqp; r += AW_THREADS) {
            const int tok = r / p.group;
            s_lse[r] = r < nq ? p.lse[((size_t)b * p.T + tok) * p.H + hk * p.group + r % p.group] * LOG2E_AW : 0.0f;
            s_lim[r] = r < nq ? len - (p.T - 1 - tok) : 0;
        }
        __syncthreads();

        float *wbase = p.w + (int64_t)b * p.w_seq + (int64_t)hk * p.w_head;
        auto do_rows = [&](const uint4 (&f)[16], int blk) {
            const int ra = blk * AW_BLOCK + warp * 16 + g, rb = ra + 8;
            float old = 0.0f;  // lanes t = 0 and t = 1 own rows g and g + 8
            const int my_row = t == 0 ? ra : rb;
            if (t < 2 && my_row < len) old = wbase[my_row];
            float sum_a = 0.0f, sum_b = 0.0f;
            for (int n0 = 0; n0 < nqp; n0 += 8) {
                float c0[4] = {0.0f, 0.0f, 0.0f, 0.0f}, c1[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                const __nv_bfloat16 *qr = s_q + (n0 + g) * AW_Q_STRIDE + 8 * t;
#pragma unroll
                for (int kb = 0; kb < 8; kb++) {
                    const uint4 bq = *reinterpret_cast<const uint4 *>(qr + 32 * kb);
                    const uint32_t a0[4] = {f[2 * kb].x, f[2 * kb + 1].x, f[2 * kb].y, f[2 * kb + 1].y};
                    const uint32_t a1[4] = {f[2 * kb].z, f[2 * kb + 1].z, f[2 * kb].w, f[2 * kb + 1].w};
                    mma_bf16_16816(c0, a0, bq.x, bq.y);
                    mma_bf16_16816(c1, a1, bq.z, bq.w);
                }
                const float2 lz = *reinterpret_cast<const float2 *>(s_lse + n0 + 2 * t);
                const int2 lim = *reinterpret_cast<const int2 *>(s_lim + n0 + 2 * t);
                sum_a += ra < lim.x ? ex2_approx(fmaf(c0[0] + c1[0], sl2, -lz.x)) : 0.0f;
                sum_a += ra < lim.y ? ex2_approx(fmaf(c0[1] + c1[1], sl2, -lz.y)) : 0.0f;
                sum_b += rb < lim.x ? ex2_approx(fmaf(c0[2] + c1[2], sl2, -lz.x)) : 0.0f;
                sum_b += rb < lim.y ? ex2_approx(fmaf(c0[3] + c1[3], sl2, -lz.y)) : 0.0f;
            }
            sum_a += __shfl_xor_sync(0xffffffffu, sum_a, 1);
            sum_b += __shfl_xor_sync(0xffffffffu, sum_b, 1);
            sum_a += __shfl_xor_sync(0xffffffffu, sum_a, 2);
            sum_b += __shfl_xor_sync(0xffffffffu, sum_b, 2);
            if (t < 2 && my_row < len) wbase[my_row] = fmaf(p.decay, old, t == 0 ? sum_a : sum_b);
        };
        for (int blk = blk0; blk < blk1; blk += 2) {
            if (blk + 1 < blk1) load_rows(kf[1], blk + 1);
            do_rows(kf[0], blk);
            if (blk + 1 < blk1) {
                if (blk + 2 < blk1) load_rows(kf[0], blk + 2);
                do_rows(kf[1], blk + 1);
            }
        }
        at += blk1 - blk0;
        __syncthreads();  // the queries in shared memory are replaced by the next unit's
    }
}

size_t attn_weights_smem(int nq) {
    const int nqp = (nq + 7) & ~7;
    return (size_t)nqp * (AW_Q_STRIDE * 2 + 8);
}

}  // namespace

cudaError_t attn_weights_configure() {
    return cudaFuncSetAttribute(attn_weights_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)attn_weights_smem(16 * 16));
}

cudaError_t launch_attn_weights(const AttnWeightsParams &p, int n_sms, cudaStream_t stream) {
    if (p.B <= 0 || p.cap <= 0) return cudaSuccess;
    const size_t smem = attn_weights_smem(p.T * p.group);
    // one wave of resident CTAs, no more than there can be blocks
    int per_sm = (int)((220 * 1024) / (smem + 1024));
    if (per_sm > AW_CTAS_PER_SM) per_sm = AW_CTAS_PER_SM;
    const int64_t most = (int64_t)p.B * p.Hkv * ((p.cap + AW_BLOCK - 1) / AW_BLOCK);
    const int64_t grid = most < (int64_t)n_sms * per_sm ? most : (int64_t)n_sms * per_sm;
    attn_weights_kernel<<<(unsigned)grid, AW_THREADS, smem, stream>>>(p);
    return cudaGetLastError();
}

}  // namespace mfc
