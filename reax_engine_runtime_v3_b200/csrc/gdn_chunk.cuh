// The gated delta rule by chunks of 64 rows, on tcgen05 tensor cores.
//
// Mathematics.  In a chunk that starts from a state S [dk, dv], let G_i be the running sum of g over its rows, k and q
// the rows' keys and (scaled) queries, and A_ij = beta_i e^(G_i - G_j) k_i.k_j for j < i.  The corrections
// V'_i = beta_i (v_i - k_i^T S_(i-1)) of the recurrence solve (I + A) V' = diag(beta) R with R_j = v_j - e^(G_j) k_j^T S, and
//
//   out_i = e^(G_i) q_i^T S + sum_(j <= i) P_ij V'_j,   P_ij = e^(G_i - G_j) q_i.k_j
//   S    <- e^(G_63) S + sum_j e^(G_63 - G_j) k_j V'_j^T
//
// With T = (I + A)^-1 diag(beta) and W = P T, both found without S, a chunk is a chain of three products:
//
//   [X_k | X_q] = S^T [k | q]^T      ->  R      (rows j of X_k)
//   [V' | Y]    = R^T [T | W]^T      ->  V'     (out = e^G X_q + Y)
//   D           = V'^T diag(..) k    ->  S
//
// Layout.  Everything is transposed so that the 128 TMEM lanes are the columns of the state (dv): S, R and V' are then
// the A operands, in TMEM, and a thread owns one state column (a half of it: two warpgroups share the lanes), which it
// keeps in registers in float32 and reads from and writes to TMEM without any exchange but a row maximum.  The B
// operands k, q, T and W are shared-memory tiles; k serves K-major (X) and MN-major (D) from one copy.
//
// Precision.  The state has to stay a float32 one, and the tensor cores take 16 bits.  An operand is scaled by a power of
// two to a largest value in [2^13, 2^14) in its row and split into two fp16 numbers, hi + lo, with 22 bits; k and q
// have 8 bits and are exact in one.  X_k, V' and D, which the state depends on, take all terms down to 2^-22; X_q and Y
// only reach the bf16 output and take the hi terms.  Sums are float32.
//
// Roles (13 warps): 0-7 carry the state; 8-11 prepare T and W of the chunks ahead; 12 issues the chain's MMAs.
#pragma once

#include <cuda_fp16.h>

#include "common.cuh"
#include "gdn.cuh"

namespace reax {

constexpr int kChunk = 64;
constexpr int kChunkThreads = 13 * 32;
constexpr int kGdnStages = 2;

// TMEM columns.  S hi and lo (64 each) share the columns of D, and V' hi and lo those of X_k: each is written after the
// other has been read.
constexpr uint32_t kTmS = 0, kTmXk = 128, kTmXq = 192, kTmR = 256, kTmY = 320, kTmW = 384, kTmPrep = 448;

struct GdnStage {
    uint8_t kq[2][128 * 128];                 // [half of dk][64 rows of k, then of q][64 fp16], 128-byte swizzle
    uint8_t t_hi[64 * 128], t_lo[64 * 128];   // rows i, columns j of T
    uint8_t w[64 * 128];
    __nv_bfloat16 v[kChunk][128];
    float4 c[kChunk];                         // factors of X_k, V', X_q and Y for each row
    float gamma;
    float pad[255];
};
static_assert(sizeof(GdnStage) % 1024 == 0, "tiles start on swizzle atoms");

struct GdnShared {
    GdnStage stage[kGdnStages];
    uint8_t a21[2][32 * 128];                 // A[32.., ..31] hi and lo: rows of 64 fp16, of which 32 are used
    uint8_t raw[128 * 256];                   // k and q rows as they come
    float a11[32 * 32], a22[32 * 32];         // 16-byte pieces of a row xor-ed with row % 8
    float4 tok[kChunk];                       // G as hi + lo (log2), row scale of k, beta
    float row_q[kChunk];                      // row scale of q
    float a21_inv[32];
    float xch[2][8][32];
    uint64_t full[kGdnStages], empty[kGdnStages], s_ready, r_ready, v_ready, x_done, y_done, d_done, kk_done, z_done;
    uint32_t tmem;
    int abort;
};

static __device__ unsigned g_mixer_status;    // REAX_STATUS_* bits of waits that expired

struct GdnWait {
    volatile int* abort;
    unsigned long long limit_ns;
    // Wait for a phase; once any wait of the block has expired all of them return at once, so that the block runs on to
    // its end (with results that the status word marks as invalid).
    REAX_DEVI void operator()(uint64_t* bar, uint32_t parity, uint32_t bit) const {
        if (mbar_wait_bounded(bar, parity, limit_ns, abort)) return;
        if (!*abort) atomicOr(&g_mixer_status, bit);
        *abort = 1;
    }
};

REAX_DEVI float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Power of two that brings a largest value `m` into [2^13, 2^14), and its inverse.
REAX_DEVI float2 scale_of(float m) {
    const uint32_t e = max(__float_as_uint(m) >> 23, 14u);
    return float2{__uint_as_float((267u - e) << 23), __uint_as_float((e - 13u) << 23)};
}

// (x0, x1) as fp16 pairs hi + lo.
REAX_DEVI void split2(float x0, float x1, uint32_t& hi, uint32_t& lo) {
    const __half2 h = __floats2half2_rn(x0, x1);
    const float2 f = __half22float2(h);
    const __half2 l = __floats2half2_rn(x0 - f.x, x1 - f.y);
    hi = *reinterpret_cast<const uint32_t*>(&h);
    lo = *reinterpret_cast<const uint32_t*>(&l);
}
REAX_DEVI uint32_t half2_bits(float x0, float x1) {
    const __half2 h = __floats2half2_rn(x0, x1);
    return *reinterpret_cast<const uint32_t*>(&h);
}

REAX_DEVI void tmem_st_x16(uint32_t taddr, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}

// MMA with the A operand in TMEM (fp16, two to a column; K = 16 takes 8 columns).
REAX_DEVI void umma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
        "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}
// fp16 operands, float32 sums; b_mn: B is stored with N contiguous.
__host__ __device__ constexpr uint32_t idesc_f16_f32(int M, int N, bool b_mn) {
    return (1u << 4) | (b_mn ? 1u << 16 : 0u) | (static_cast<uint32_t>(N >> 3) << 17) | (static_cast<uint32_t>(M >> 4) << 24);
}
// 128-byte swizzled tile with N contiguous: 64 columns of N to a 128-byte row, 8 rows of K to a 1024-byte atom, the next 64
// columns `lbo` bytes on.
REAX_DEVI uint64_t sw128_mn_desc(uint32_t smem_addr, uint32_t lbo) {
    uint64_t d = sw128_kmajor_desc(smem_addr);
    d &= ~(static_cast<uint64_t>(0x3FFF) << 16);
    return d | static_cast<uint64_t>(lbo >> 4) << 16;
}

REAX_DEVI void cp_async16_zfill(uint32_t dst, const void* src, bool real) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(real ? 16 : 0) : "memory");
}

// One row's solve z (I + a) = p in place, z and p of 32 columns, `a` strictly lower [32][32]: columns from the last to the
// first, each finished value taken out of the ones before it (the row of `a` is the same for all lanes: a broadcast).
REAX_DEVI void solve32(uint64_t (&z)[16], const float* a) {
#pragma unroll
    for (int j = 31; j > 0; --j) {
        const float zj = j % 2 ? f2_hi(z[j / 2]) : f2_lo(z[j / 2]);
        const uint64_t neg = f2(-zj, -zj);
#pragma unroll
        for (int c = 0; c < (j + 3) / 4; ++c) {
            const ulonglong2 x = *reinterpret_cast<const ulonglong2*>(a + j * 32 + ((c ^ (j & 7)) * 4));
            z[2 * c] = fma2_rn(neg, x.x, z[2 * c]);
            if (4 * c + 2 < j) z[2 * c + 1] = fma2_rn(neg, x.y, z[2 * c + 1]);
        }
    }
}

template <int DK, int DV>
__global__ void __launch_bounds__(kChunkThreads, 1) gdn_chunk_kernel(const GdnParams p, unsigned long long limit_ns) {
    extern __shared__ uint8_t smem_raw[];
    GdnShared& sh = *reinterpret_cast<GdnShared*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
    const int hv = blockIdx.x, b = blockIdx.y, hk = hv / (p.v_heads / p.k_heads);
    int r0, r1;
    gdn_rows(p, b, &r0, &r1);
    const int slot = gdn_slot(p, b), rows = r1 - r0, chunks = (rows + kChunk - 1) / kChunk;
    __nv_bfloat16* out = p.out + (static_cast<long long>(r0) * p.v_heads + hv) * DV;
    const long long ldo = static_cast<long long>(p.v_heads) * DV;
    if (slot < 0) {
        for (long long e = tid; e < static_cast<long long>(rows) * (DV / 8); e += kChunkThreads)
            *reinterpret_cast<uint4*>(out + e / (DV / 8) * ldo + e % (DV / 8) * 8) = uint4{};
        return;
    }
    float* state = p.state + (static_cast<long long>(slot) * p.v_heads + hv) * DK * DV;
    if (chunks == 0) {
        if (!p.carry)
            for (int e = tid; e < DK * DV; e += kChunkThreads) state[e] = 0.0f;
        return;
    }

    if (warp == 12) tmem_alloc(&sh.tmem, 512);
    if (tid == 0) {
        for (int i = 0; i < kGdnStages; ++i) mbar_init(&sh.full[i], 128), mbar_init(&sh.empty[i], 256);
        mbar_init(&sh.s_ready, 256), mbar_init(&sh.r_ready, 256), mbar_init(&sh.v_ready, 256);
        mbar_init(&sh.x_done, 1), mbar_init(&sh.y_done, 1), mbar_init(&sh.d_done, 1);
        mbar_init(&sh.kk_done, 1), mbar_init(&sh.z_done, 1);
        sh.abort = 0;
        fence_mbar_init();
    }
    if (DV < 128)
        for (int e = tid; e < kGdnStages * kChunk * 128; e += kChunkThreads)
            sh.stage[e / (kChunk * 128)].v[e / 128 % kChunk][e % 128] = __float2bfloat16_rn(0.0f);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tm = sh.tmem;
    const GdnWait wait{&sh.abort, limit_ns};

    if (warp < 8) {
        // ------------------------------------------------------------------------------------ the state's warps
        const int quarter = warp % 4, half = warp / 4, n = quarter * 32 + lane;
        const uint32_t lanes = tm + (static_cast<uint32_t>(quarter * 32) << 16);
        constexpr int kS = DK / 2;
        float s[kS];
#pragma unroll
        for (int i = 0; i < kS; ++i) s[i] = p.carry && n < DV ? state[(half * kS + i) * DV + n] : 0.0f;
        int turn = 0;
        // Largest of both halves of this thread's row (the two warps of a quarter meet).
        auto row_max = [&](float m) {
            sh.xch[turn][warp][lane] = m;
            named_bar_sync(1 + quarter, 64);
            m = fmaxf(m, sh.xch[turn][warp ^ 4][lane]);
            turn ^= 1;
            return m;
        };
        float xq[32], sq = 0.0f, sr = 0.0f;
        auto output = [&](int c) {
            const GdnStage& st = sh.stage[c & 1];
            uint32_t y[32];
            tmem_ld_x32_sync(lanes + kTmW + half * 32, y);
            const int left = rows - c * kChunk - half * 32;
            __nv_bfloat16* o = out + (static_cast<long long>(c) * kChunk + half * 32) * ldo + n;
#pragma unroll
            for (int i = 0; i < 32; ++i) {
                const float4 f = st.c[half * 32 + i];
                const float x = xq[i] * (f.z * sq) + __uint_as_float(y[i]) * (f.w * sr);
                if (i < left && n < DV) o[i * ldo] = __float2bfloat16_rn(x);
            }
            mbar_arrive(&sh.empty[c & 1]);
        };
        for (int c = 0; c < chunks; ++c) {
            const uint32_t par = c & 1;
            const GdnStage& st = sh.stage[c & 1];
            // S -> two fp16 operands
            float m = 0.0f;
#pragma unroll
            for (int i = 0; i < kS; ++i) m = fmaxf(m, fabsf(s[i]));
            const float2 ss = scale_of(row_max(m));
#pragma unroll
            for (int x = 0; x < kS / 32; ++x) {
                uint32_t hi[16], lo[16];
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    split2(s[x * 32 + 2 * i] * ss.x, s[x * 32 + 2 * i + 1] * ss.x, hi[i], lo[i]);
                tmem_st_x16(lanes + kTmS + half * (kS / 2) + x * 16, hi);
                tmem_st_x16(lanes + kTmS + 64 + half * (kS / 2) + x * 16, lo);
            }
            tmem_wait_st();
            tc_fence_before();
            mbar_arrive(&sh.s_ready);
            if (c > 0) output(c - 1);
            sq = ss.y;
            // X_k -> R
            wait(&sh.full[c & 1], (c >> 1) & 1, kStatusTimeoutFull);
            wait(&sh.x_done, par, kStatusTimeoutAccFull);
            tc_fence_after();
            uint32_t x[32], hi[16], lo[16];
            tmem_ld_x32_sync(lanes + kTmXk + half * 32, x);
            float r[32];
            m = 0.0f;
#pragma unroll
            for (int i = 0; i < 32; ++i) {
                const int j = half * 32 + i;
                r[i] = __bfloat162float(st.v[j][n]) - __uint_as_float(x[i]) * (st.c[j].x * ss.y);
                m = fmaxf(m, fabsf(r[i]));
            }
            const float2 rs = scale_of(row_max(m));
#pragma unroll
            for (int i = 0; i < 16; ++i) split2(r[2 * i] * rs.x, r[2 * i + 1] * rs.x, hi[i], lo[i]);
            tmem_st_x16(lanes + kTmR + half * 16, hi);
            tmem_st_x16(lanes + kTmR + 32 + half * 16, lo);
            tmem_wait_st();
            tc_fence_before();
            mbar_arrive(&sh.r_ready);
            sr = rs.y;
            // V'
            wait(&sh.y_done, par, kStatusTimeoutAccFull);
            tc_fence_after();
            tmem_ld_x32_sync(lanes + kTmY + half * 32, x);
            m = 0.0f;
#pragma unroll
            for (int i = 0; i < 32; ++i) {
                r[i] = __uint_as_float(x[i]) * (st.c[half * 32 + i].y * rs.y);
                m = fmaxf(m, fabsf(r[i]));
            }
            const float2 vs = scale_of(row_max(m));
#pragma unroll
            for (int i = 0; i < 16; ++i) split2(r[2 * i] * vs.x, r[2 * i + 1] * vs.x, hi[i], lo[i]);
            tmem_st_x16(lanes + kTmXk + half * 16, hi);
            tmem_st_x16(lanes + kTmXk + 32 + half * 16, lo);
            tmem_wait_st();
            tc_fence_before();
            mbar_arrive(&sh.v_ready);
            // X_q is overwritten once the next state is handed over
            tmem_ld_x32_sync(lanes + kTmXq + half * 32, x);
#pragma unroll
            for (int i = 0; i < 32; ++i) xq[i] = __uint_as_float(x[i]);
            // D -> S
            wait(&sh.d_done, par, kStatusTimeoutAccFull);
            tc_fence_after();
            const float gamma = st.gamma;
#pragma unroll
            for (int y = 0; y < kS / 32; ++y) {
                tmem_ld_x32_sync(lanes + kTmS + half * kS + y * 32, x);
#pragma unroll
                for (int i = 0; i < 32; ++i) s[y * 32 + i] = gamma * s[y * 32 + i] + vs.y * __uint_as_float(x[i]);
            }
        }
        output(chunks - 1);
        if (n < DV)
#pragma unroll
            for (int i = 0; i < kS; ++i) state[(half * kS + i) * DV + n] = s[i];
    } else if (warp == 12) {
        // ------------------------------------------------------------------------------- issuer of the chain's MMAs
        if (lane == 0) {
            constexpr uint32_t id64 = idesc_f16_f32(128, 64, false), id_d = idesc_f16_f32(128, DK, true);
            for (int c = 0; c < chunks; ++c) {
                const uint32_t par = c & 1;
                GdnStage& st = sh.stage[c & 1];
                const uint32_t kq = smem_u32(st.kq), thi = smem_u32(st.t_hi), tlo = smem_u32(st.t_lo), w = smem_u32(st.w);
                wait(&sh.full[c & 1], (c >> 1) & 1, kStatusTimeoutFull);
                wait(&sh.s_ready, par, kStatusTimeoutEmpty);
                tc_fence_after();
#pragma unroll
                for (int e = 0; e < 2 * (DK / 16); ++e) {
                    const int ks = e % (DK / 16);
                    umma_f16_ts(tm + kTmXk, tm + kTmS + (e / (DK / 16)) * 64 + ks * 8,
                                sw128_kmajor_desc(kq + (ks / 4) * 16384 + (ks % 4) * 32), id64, e > 0);
                }
                umma_commit(&sh.x_done);
#pragma unroll
                for (int ks = 0; ks < DK / 16; ++ks)
                    umma_f16_ts(tm + kTmXq, tm + kTmS + ks * 8, sw128_kmajor_desc(kq + 8192 + (ks / 4) * 16384 + (ks % 4) * 32), id64,
                                ks > 0);
                wait(&sh.r_ready, par, kStatusTimeoutEmpty);
                tc_fence_after();
#pragma unroll
                for (int e = 0; e < 12; ++e) {
                    const int ks = e % 4, term = e / 4;      // hi hi, lo hi, hi lo
                    umma_f16_ts(tm + kTmY, tm + kTmR + (term == 1 ? 32 : 0) + ks * 8,
                                sw128_kmajor_desc((term == 2 ? tlo : thi) + ks * 32), id64, e > 0);
                }
                umma_commit(&sh.y_done);
#pragma unroll
                for (int ks = 0; ks < 4; ++ks)
                    umma_f16_ts(tm + kTmW, tm + kTmR + ks * 8, sw128_kmajor_desc(w + ks * 32), id64, ks > 0);
                wait(&sh.v_ready, par, kStatusTimeoutEmpty);
                tc_fence_after();
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    umma_f16_ts(tm + kTmS, tm + kTmXk + (e / 4) * 32 + (e % 4) * 8, sw128_mn_desc(kq + (e % 4) * 2048, 16384), id_d,
                                e > 0);
                umma_commit(&sh.d_done);
            }
            // TMEM may be freed once the MMAs are done, also after a wait that expired
            mbar_wait_bounded(&sh.d_done, (chunks - 1) & 1, limit_ns, nullptr);
        }
        __syncwarp();
    } else {
        // ---------------------------------------------------------------------------------- T and W of the chunks ahead
        const int t = tid - 256, quarter = warp % 4, i = t % 64;      // lane t of TMEM: row i of k (t < 64) or q
        const bool is_q = t >= 64, upper = (quarter & 1) != 0;        // upper: rows 32.. of the chunk
        const uint32_t lanes = tm + (static_cast<uint32_t>(quarter * 32) << 16);
        const __nv_bfloat16* kg = p.k + static_cast<long long>(r0) * p.ldk + hk * DK;
        const __nv_bfloat16* qg = p.q + static_cast<long long>(r0) * p.ldq + hk * DK;
        const __nv_bfloat16* vg = p.v + static_cast<long long>(r0) * p.ldv + hv * DV;
        constexpr int kPieces = DK / 8;                               // 16-byte pieces of a row
        auto load_kq = [&](int c) {
#pragma unroll 4
            for (int e = t; e < 128 * kPieces; e += 128) {
                const int r = e / kPieces, x = e % kPieces, row = c * kChunk + r % 64;
                const bool real = row < rows;
                const __nv_bfloat16* src = r < 64 ? kg + (real ? row * p.ldk : 0) : qg + (real ? row * p.ldq : 0);
                cp_async16_zfill(smem_u32(sh.raw) + r * (DK * 2) + x * 16, src + x * 8, real);
            }
        };
        load_kq(0);
        for (int c = 0; c < chunks; ++c) {
            const uint32_t par = c & 1;
            GdnStage& st = sh.stage[c & 1];
            if (c >= kGdnStages) wait(&sh.empty[c & 1], ((c >> 1) - 1) & 1, kStatusTimeoutEmpty);
#pragma unroll 4
            for (int e = t; e < kChunk * (DV / 8); e += 128) {
                const int r = e / (DV / 8), x = e % (DV / 8), row = c * kChunk + r;
                const bool real = row < rows;
                cp_async16_zfill(smem_u32(&st.v[r][x * 8]), vg + (real ? row * p.ldv : 0) + x * 8, real);
            }
            // running sums of g in log2 units: multiples of 2^-8 (exact in float32) and the rest, so that differences
            // of far running sums keep their low bits; decays below 2^-128 count as 0
            if (quarter == 0) {
                float hi[2], lo[2], beta[2];
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const int row = c * kChunk + lane * 2 + j;
                    const long long at = (static_cast<long long>(r0) + row) * p.v_heads + hv;
                    const float g = row < rows ? p.g[at] * 1.44269504f : 0.0f;
                    beta[j] = row < rows ? p.beta[at] : 0.0f;
                    const float x = g < -128.0f ? -128.0f : g;
                    hi[j] = rintf(x * 256.0f) * 0.00390625f;
                    lo[j] = x - hi[j];
                }
                float sh_ = hi[0] + hi[1], sl = lo[0] + lo[1];
#pragma unroll
                for (int m = 1; m < 32; m <<= 1) {
                    const float a = __shfl_up_sync(0xFFFFFFFFu, sh_, m), l = __shfl_up_sync(0xFFFFFFFFu, sl, m);
                    if (lane >= m) sh_ += a, sl += l;
                }
                sh.tok[lane * 2 + 1].x = sh_, sh.tok[lane * 2 + 1].y = sl, sh.tok[lane * 2 + 1].w = beta[1];
                sh.tok[lane * 2].x = sh_ - hi[1], sh.tok[lane * 2].y = sl - lo[1], sh.tok[lane * 2].w = beta[0];
                if (lane == 31) st.gamma = ex2(sh_ + sl);
            }
            cp_async_wait_all();
            named_bar_sync(5, 128);
            // k and q rows -> fp16 scaled to [2^13, 2^14): four lanes a row
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int r = quarter * 32 + u * 8 + lane / 4, c4 = lane % 4;
                uint4 w[kPieces / 4];
                uint32_t top = 0;
                uint64_t sum = 0;
#pragma unroll
                for (int x = 0; x < kPieces / 4; ++x) {
                    const int piece = ((x + r) % (kPieces / 4)) * 4 + c4;
                    w[x] = *reinterpret_cast<const uint4*>(sh.raw + r * (DK * 2) + piece * 16);
                    const uint32_t y[4] = {w[x].x, w[x].y, w[x].z, w[x].w};
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        top = __vmaxu2(top, y[j] & 0x7FFF7FFFu);
                        const uint64_t f = bf16x2_to_f2(y[j]);
                        sum = fma2_rn(f, f, sum);
                    }
                }
                top = max(top & 0xFFFFu, top >> 16);
                float sq = f2_lo(sum) + f2_hi(sum);
#pragma unroll
                for (int m = 1; m < 4; m <<= 1) {
                    top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, m));
                    sq += __shfl_xor_sync(0xFFFFFFFFu, sq, m);
                }
                const float2 f = scale_of(__uint_as_float(top << 16));
                const uint64_t f_2 = f2(f.x, f.x);
#pragma unroll
                for (int x = 0; x < kPieces / 4; ++x) {
                    const int piece = ((x + r) % (kPieces / 4)) * 4 + c4;
                    const uint32_t y[4] = {w[x].x, w[x].y, w[x].z, w[x].w};
                    uint32_t o[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const uint64_t g = mul2_rn(bf16x2_to_f2(y[j]), f_2);
                        o[j] = half2_bits(f2_lo(g), f2_hi(g));
                    }
                    *reinterpret_cast<uint4*>(st.kq[piece / 8] + r * 128 + ((piece % 8) ^ (r % 8)) * 16) =
                        uint4{o[0], o[1], o[2], o[3]};
                }
                if (c4 == 0) {
                    const float y = (p.normalize ? rsqrtf(sq + kGdnNormEps) : 1.0f) * f.y;
                    if (r < 64) sh.tok[r].z = y;
                    else sh.row_q[r - 64] = y * p.scale;
                }
            }
            fence_proxy_async_smem();
            named_bar_sync(5, 128);
            if (t == 0) {
                const uint32_t kq = smem_u32(st.kq);
                tc_fence_after();
#pragma unroll
                for (int ks = 0; ks < DK / 16; ++ks) {
                    const uint64_t d = sw128_kmajor_desc(kq + (ks / 4) * 16384 + (ks % 4) * 32);
                    umma_f16(tm + kTmPrep, d, d, idesc_f16_f32(128, 64, false), ks > 0);
                }
                umma_commit(&sh.kk_done);
            }
            if (c + 1 < chunks) load_kq(c + 1);
            const float4 me = sh.tok[i];
            const float mine = is_q ? sh.row_q[i] : me.z * me.w;
            wait(&sh.kk_done, par, kStatusTimeoutAccFull);
            tc_fence_after();
            // this row of A (k) or P (q), in two halves of 32 columns
            uint64_t z1[16], z2[16];
            {
                uint32_t x[32];
                float y[32];
                tmem_ld_x32_sync(lanes + kTmPrep, x);
#pragma unroll
                for (int j = 0; j < 32; ++j) {
                    const float4 o = sh.tok[j];
                    const float d = ex2((me.x - o.x) + (me.y - o.y)) * (o.z * mine) * __uint_as_float(x[j]);
                    y[j] = j < i || (is_q && j == i) ? d : 0.0f;
                }
#pragma unroll
                for (int j = 0; j < 16; ++j) z1[j] = f2(y[2 * j], y[2 * j + 1]);
                if (!is_q) {
                    if (!upper) {
#pragma unroll
                        for (int j = 0; j < 8; ++j)
                            *reinterpret_cast<float4*>(sh.a11 + i * 32 + (j ^ (i & 7)) * 4) =
                                float4{y[4 * j], y[4 * j + 1], y[4 * j + 2], y[4 * j + 3]};
                    } else {
                        float m = 0.0f;
#pragma unroll
                        for (int j = 0; j < 32; ++j) m = fmaxf(m, fabsf(y[j]));
                        const float2 f = scale_of(m);
                        sh.a21_inv[i - 32] = f.y;
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            uint32_t hi[4], lo[4];
#pragma unroll
                            for (int e = 0; e < 4; ++e) split2(y[8 * j + 2 * e] * f.x, y[8 * j + 2 * e + 1] * f.x, hi[e], lo[e]);
                            const int at = (i - 32) * 128 + ((j ^ (i & 7)) * 16);
                            *reinterpret_cast<uint4*>(sh.a21[0] + at) = uint4{hi[0], hi[1], hi[2], hi[3]};
                            *reinterpret_cast<uint4*>(sh.a21[1] + at) = uint4{lo[0], lo[1], lo[2], lo[3]};
                        }
                    }
                }
                if (upper) {
                    tmem_ld_x32_sync(lanes + kTmPrep + 32, x);
#pragma unroll
                    for (int j = 0; j < 32; ++j) {
                        const float4 o = sh.tok[32 + j];
                        const float d = ex2((me.x - o.x) + (me.y - o.y)) * (o.z * mine) * __uint_as_float(x[j]);
                        y[j] = 32 + j < i || (is_q && 32 + j == i) ? d : 0.0f;
                    }
#pragma unroll
                    for (int j = 0; j < 16; ++j) z2[j] = f2(y[2 * j], y[2 * j + 1]);
                    if (!is_q)
#pragma unroll
                        for (int j = 0; j < 8; ++j)
                            *reinterpret_cast<float4*>(sh.a22 + (i - 32) * 32 + (j ^ (i & 7)) * 4) =
                                float4{y[4 * j], y[4 * j + 1], y[4 * j + 2], y[4 * j + 3]};
                }
            }
            if (!is_q) {                       // T starts from the identity
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    z1[j] = f2(2 * j == i ? 1.0f : 0.0f, 2 * j + 1 == i ? 1.0f : 0.0f);
                    z2[j] = f2(32 + 2 * j == i ? 1.0f : 0.0f, 33 + 2 * j == i ? 1.0f : 0.0f);
                }
            } else if (!upper) {
#pragma unroll
                for (int j = 0; j < 16; ++j) z2[j] = 0;
            }
            fence_proxy_async_smem();
            tc_fence_before();
            named_bar_sync(5, 128);
            float z_inv = 0.0f;
            if (upper) {
                // the columns 32.. first, then their product with A[32.., ..31] on the tensor cores
                solve32(z2, sh.a22);
                float y[32], m = 0.0f;
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    y[2 * j] = f2_lo(z2[j]) * sh.a21_inv[2 * j];
                    y[2 * j + 1] = f2_hi(z2[j]) * sh.a21_inv[2 * j + 1];
                    m = fmaxf(m, fmaxf(fabsf(y[2 * j]), fabsf(y[2 * j + 1])));
                }
                const float2 f = scale_of(m);
                z_inv = f.y;
                uint32_t hi[16], lo[16];
#pragma unroll
                for (int j = 0; j < 16; ++j) split2(y[2 * j] * f.x, y[2 * j + 1] * f.x, hi[j], lo[j]);
                tmem_st_x16(lanes + kTmPrep, hi);
                tmem_st_x16(lanes + kTmPrep + 16, lo);
                tmem_wait_st();
                tc_fence_before();
            }
            named_bar_sync(5, 128);
            if (t == 0) {
                tc_fence_after();
#pragma unroll
                for (int e = 0; e < 6; ++e) {
                    const int ks = e % 2, term = e / 2;
                    umma_f16_ts(tm + kTmPrep + 32, tm + kTmPrep + (term == 1 ? 16 : 0) + ks * 8,
                                sw128_mn_desc(smem_u32(sh.a21[term == 2]) + ks * 2048, 4096), idesc_f16_f32(128, 32, true), e > 0);
                }
                umma_commit(&sh.z_done);
            }
            if (upper) {
                wait(&sh.z_done, par, kStatusTimeoutAccFull);
                tc_fence_after();
                uint32_t x[32];
                tmem_ld_x32_sync(lanes + kTmPrep + 32, x);
                tc_fence_before();
#pragma unroll
                for (int j = 0; j < 16; ++j)
                    z1[j] = fma2_rn(f2(-z_inv, -z_inv), f2(__uint_as_float(x[2 * j]), __uint_as_float(x[2 * j + 1])), z1[j]);
            }
            solve32(z1, sh.a11);
            // columns times beta; a row of T in two terms, of W in one
            float m = 0.0f;
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                z1[j] = mul2_rn(z1[j], f2(sh.tok[2 * j].w, sh.tok[2 * j + 1].w));
                z2[j] = mul2_rn(z2[j], f2(sh.tok[32 + 2 * j].w, sh.tok[33 + 2 * j].w));
                m = fmaxf(m, fmaxf(fmaxf(fabsf(f2_lo(z1[j])), fabsf(f2_hi(z1[j]))), fmaxf(fabsf(f2_lo(z2[j])), fabsf(f2_hi(z2[j])))));
            }
            const float2 f = scale_of(m);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                uint32_t hi[4], lo[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint64_t z = j < 4 ? z1[j * 4 + e] : z2[j * 4 + e - 16];
                    split2(f2_lo(z) * f.x, f2_hi(z) * f.x, hi[e], lo[e]);
                }
                const int at = i * 128 + ((j ^ (i & 7)) * 16);
                *reinterpret_cast<uint4*>((is_q ? st.w : st.t_hi) + at) = uint4{hi[0], hi[1], hi[2], hi[3]};
                if (!is_q) *reinterpret_cast<uint4*>(st.t_lo + at) = uint4{lo[0], lo[1], lo[2], lo[3]};
            }
            const float4 last = sh.tok[kChunk - 1];
            if (is_q) {
                st.c[i].z = mine * ex2(me.x + me.y);
                st.c[i].w = f.y;
            } else {
                st.c[i].x = me.z * ex2(me.x + me.y);
                st.c[i].y = me.z * ex2((last.x - me.x) + (last.y - me.y)) * f.y;
            }
            fence_proxy_async_smem();
            mbar_arrive(&sh.full[c & 1]);
            // every lane has read tok, a11 and a22 before the next chunk's are written
            named_bar_sync(5, 128);
        }
        if (t == 0) mbar_wait_bounded(&sh.z_done, (chunks - 1) & 1, limit_ns, nullptr);
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 12) {
        tmem_relinquish();
        tmem_dealloc(tm, 512);
    }
}

constexpr size_t gdn_chunk_smem() { return sizeof(GdnShared) + 1024; }

}  // namespace reax
