// The gated delta rule.  For each value head, with a state S [dk, dv] and a row's k, v, q, decay e^g and beta:
//
//   S <- e^g S;   u = beta (v - k^T S);   S <- S + k u^T;   o = scale q^T S
//
// (q and k divided by sqrt(sum of squares + 1e-6) first when `normalize` is set).
#pragma once

#include "common.cuh"

namespace reax {

constexpr float kGdnNormEps = 1e-6f;

struct GdnParams {
    const __nv_bfloat16* q;      // [rows, k_heads, DK], row stride ldq
    const __nv_bfloat16* k;      // [rows, k_heads, DK], row stride ldk
    const __nv_bfloat16* v;      // [rows, v_heads, DV], row stride ldv
    const float* g;              // [rows, v_heads], log of the decay
    const float* beta;           // [rows, v_heads]
    float* state;                // [slots, v_heads, DK, DV]
    const int32_t* cu_seqlens;   // [batch + 1] (NULL: one sequence of `rows` rows)
    const int32_t* slots;        // [batch] (NULL: sequence b keeps its state in slot b)
    __nv_bfloat16* out;          // [rows, v_heads, DV]
    long long ldq, ldk, ldv;
    int rows, batch, k_heads, v_heads, n_slots;
    float scale;
    int normalize, carry;
};

REAX_DEVI float warp_sum(float v) {
#pragma unroll
    for (int m = 16; m > 0; m >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, m);
    return v;
}

// What a row with that sum of squares is multiplied by to be normalized: NaN, not 0, where the sum passes float32.
REAX_DEVI float gdn_rsqrt(float sum) { return rsqrtf(__fmaf_rn(0.0f, sum, sum + kGdnNormEps)); }

// State slot of sequence b, or -1 for one that keeps none (its outputs are zeros).
REAX_DEVI int gdn_slot(const GdnParams& p, int b) {
    const int s = p.slots ? p.slots[b] : b;
    return s < 0 || s >= p.n_slots ? -1 : s;
}
// Rows [begin, end) of sequence b, kept inside the packed rows.
REAX_DEVI void gdn_rows(const GdnParams& p, int b, int* begin, int* end) {
    int lo = p.cu_seqlens ? p.cu_seqlens[b] : 0;
    int hi = p.cu_seqlens ? p.cu_seqlens[b + 1] : p.rows;
    lo = min(max(lo, 0), p.rows);
    hi = min(max(hi, lo), p.rows);
    *begin = lo;
    *end = hi;
}

// ------------------------------------------------------------------------------------------ single-row step
// One block a sequence and head: the block's threads hold the whole state, 4 columns of DV and DK / kGroups
// rows each, so each value is read and written once and both sums over k (k^T S and q^T S) take one pass:
// o = e^g q^T S + (q.k) u needs no second one.  Bound by the state's bytes: 512 sequences of 32 heads of 128 x 128 (2.1 GB read
// and written) take 327 to 338 us, 6.4 to 6.6 TB/s; one takes 4 us, most of it the launch.
constexpr int kStepThreads = 256;

template <int DK, int DV>
__global__ void __launch_bounds__(kStepThreads) gdn_step_kernel(const GdnParams p) {
    constexpr int kCols = DV / 4, kGroups = kStepThreads / kCols, kRows = DK / kGroups;
    __shared__ float s_k[DK], s_q[DK];
    __shared__ float4 s_sum[2][kGroups][kCols];
    __shared__ float s_red[3][DK / 32];
    const int tid = threadIdx.x, hv = blockIdx.x, b = blockIdx.y, hk = hv / (p.v_heads / p.k_heads);
    const int c = tid % kCols, grp = tid / kCols;
    const long long at = static_cast<long long>(b) * p.v_heads + hv;
    const int slot = gdn_slot(p, b);
    if (slot < 0) {
        if (tid < kCols) *reinterpret_cast<uint2*>(p.out + at * DV + c * 4) = uint2{};
        return;
    }
    float4* st = reinterpret_cast<float4*>(p.state + (static_cast<long long>(slot) * p.v_heads + hv) * DK * DV) +
                 grp * kRows * kCols + c;
    float4 s[kRows];
#pragma unroll
    for (int i = 0; i < kRows; ++i) s[i] = st[i * kCols];
    if (tid < DK) {
        const float q = __bfloat162float(p.q[b * p.ldq + hk * DK + tid]), k = __bfloat162float(p.k[b * p.ldk + hk * DK + tid]);
        s_q[tid] = q, s_k[tid] = k;
        const float qq = warp_sum(q * q), kk = warp_sum(k * k), qk = warp_sum(q * k);
        if (tid % 32 == 0) s_red[0][tid / 32] = qq, s_red[1][tid / 32] = kk, s_red[2][tid / 32] = qk;
    }
    __syncthreads();
    float4 ks = {}, qs = {};
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
        const float k = s_k[grp * kRows + i], q = s_q[grp * kRows + i];
        ks.x += k * s[i].x, ks.y += k * s[i].y, ks.z += k * s[i].z, ks.w += k * s[i].w;
        qs.x += q * s[i].x, qs.y += q * s[i].y, qs.z += q * s[i].z, qs.w += q * s[i].w;
    }
    s_sum[0][grp][c] = ks;
    s_sum[1][grp][c] = qs;
    float qq = 0, kk = 0, qk = 0;
#pragma unroll
    for (int i = 0; i < DK / 32; ++i) qq += s_red[0][i], kk += s_red[1][i], qk += s_red[2][i];
    const float rq = p.normalize ? p.scale * gdn_rsqrt(qq) : p.scale;
    const float rk = p.normalize ? gdn_rsqrt(kk) : 1.0f;
    const float decay = expf(p.g[at]), beta = p.beta[at];
    const uint2 vw = *reinterpret_cast<const uint2*>(p.v + b * p.ldv + hv * DV + c * 4);
    __syncthreads();
    ks = s_sum[0][0][c];
#pragma unroll
    for (int i = 1; i < kGroups; ++i) {
        const float4 x = s_sum[0][i][c];
        ks.x += x.x, ks.y += x.y, ks.z += x.z, ks.w += x.w;
    }
    const float f = rk * decay;
    float4 u;                                   // rk u: what k (not normalized) multiplies
    u.x = rk * beta * (__uint_as_float(vw.x << 16) - f * ks.x);
    u.y = rk * beta * (__uint_as_float(vw.x & 0xFFFF0000u) - f * ks.y);
    u.z = rk * beta * (__uint_as_float(vw.y << 16) - f * ks.z);
    u.w = rk * beta * (__uint_as_float(vw.y & 0xFFFF0000u) - f * ks.w);
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
        const float k = s_k[grp * kRows + i];
        s[i].x = decay * s[i].x + k * u.x;
        s[i].y = decay * s[i].y + k * u.y;
        s[i].z = decay * s[i].z + k * u.z;
        s[i].w = decay * s[i].w + k * u.w;
        st[i * kCols] = s[i];
    }
    if (grp == 0) {
        qs = s_sum[1][0][c];
#pragma unroll
        for (int i = 1; i < kGroups; ++i) {
            const float4 x = s_sum[1][i][c];
            qs.x += x.x, qs.y += x.y, qs.z += x.z, qs.w += x.w;
        }
        *reinterpret_cast<uint2*>(p.out + at * DV + c * 4) =
            uint2{bf16x2_rn(f2(rq * (decay * qs.x + qk * u.x), rq * (decay * qs.y + qk * u.y))),
                  bf16x2_rn(f2(rq * (decay * qs.z + qk * u.z), rq * (decay * qs.w + qk * u.w)))};
    }
}

}  // namespace reax
