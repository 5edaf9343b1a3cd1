// The gated delta rule by chunks of 64 rows, on tcgen05 tensor cores.
//
// Mathematics.  In a chunk that starts from a state S [dk, dv], let G_i be the running sum of g over its rows, k and q
// the rows' keys and (scaled) queries, and A_ij = beta_i e^(G_i - G_j) k_i.k_j for j < i.  The corrections
// V'_i = beta_i (v_i - k_i^T S_(i-1)) of the recurrence solve (I + A) V' = diag(beta) R with R_j = v_j - e^(G_j) k_j^T S, and
//
//   out_i = e^(G_i) q_i^T S + sum_(j <= i) P_ij V'_j,   P_ij = e^(G_i - G_j) q_i.k_j
//   S    <- e^(G_63) S + sum_j e^(G_63 - G_j) k_j V'_j^T
//
// With T = (I + A)^-1 diag(beta) and P, both found without S, a chunk is a chain of three products (and one beside it):
//
//   [X_k | X_q] = S^T [k | q]^T      ->  R      (from X_k)
//   V'          = R^T T^T            ->  V'
//   D           = V'^T diag(..) k    ->  S      and  Y = V'^T P^T, out = e^G X_q + Y
//
// Layout.  Everything is transposed so that the 128 TMEM lanes are the columns of the state (dv): S, R and V' are then
// the A operands, in TMEM, and a thread owns a half of one state column (two warpgroups share the lanes), which it
// keeps in registers in float32 and reads from and writes to TMEM without any exchange but a row maximum.  The B
// operands k, q, T and P are shared-memory tiles; k serves K-major (X) and MN-major (D) from one copy.
//
// Precision.  The state has to stay a float32 one, and the tensor cores take 16 bits.  An operand is scaled by a power of
// two to a largest value in [2^13, 2^14) in its row and split into two fp16 numbers, hi + lo, with 22 bits; k and q
// have 8 bits and are exact in one.  X_k, V' and D, which the state depends on, take all terms down to 2^-22; X_q and Y
// only reach the bf16 output and take the hi terms.  Sums are float32.
//
// Not finite.  The products run over whole chunks, where 0 times NaN would reach the rows before.  So the first kernel finds a
// chunk's first row whose k, g or beta is not finite, leaves the rows from there on out of T (as if their beta were 0) and
// marks them in c_x; the second takes R of the rows from a column's first that is not finite on as 0 (by the mark, by v or by
// the state) and puts NaN into the outputs and the state that follow from it.  A q that is not finite stays in its row.
//
// Two kernels.  What a chunk needs that does not depend on the state (k and q as fp16 tiles, T, P and the rows' factors) is
// found by gdn_tiles_kernel for all chunks at once, a block of four warps for each chunk and key head, and kept in scratch
// memory; gdn_chunk_kernel then carries the states along, a block for each sequence and value head, which reads those tiles
// as they are.  Of one kernel with warps for each part, a chunk took 6.5 us of a block, most of it waiting for the solve of
// the next one, where the second kernel takes 4.0: 8192 rows of one sequence and 32 value heads 860 us then and 590 now,
// 32768 rows of 16 sequences 836 and 776, 4001 of 8 155 and 130, 96 rows 22.5 and 23.2.
//
// What bounds the second: the chain of a chunk.  Its three products take 3700 cycles from operands ready to results ready (of
// which 2500 are MMAs) and the steps between them about 3900.  Sixteen warps of a quarter column each in place of eight of a
// half took as long (645 us for the 8192 rows, 628 then by eight).  With DV = 64 half of the lanes carry zeros and a chunk
// takes as long as with 128 (8192 rows 587 us).  The first (265 us of the 776, 298 alone): four blocks of four warps an SM, which
// its registers and shared memory allow, fill 35% of its issue slots; the rest is waiting for the rows of k below 32, whose solve
// is longest.
//
// Roles of the second (10 warps): 0-7 carry the state; 8 issues the MMAs; 9 loads.
#pragma once

#include <cuda_fp16.h>

#include "common.cuh"
#include "gdn.cuh"

namespace reax {

constexpr int kChunk = 64;
constexpr int kChunkThreads = 10 * 32;
constexpr int kTilesThreads = 4 * 32;
constexpr int kKqSlots = 3;                   // chunks of k and q tiles in flight
constexpr int kGdnSorted = 256;               // sequences up to which blocks take them in the order of their lengths
constexpr float kGdnDown = 0x1p-20f, kGdnUp = 0x1p20f;
constexpr uint32_t kGdnNan = 0x7FFFFFFFu;

// TMEM columns.  S hi and lo (64 each) share the columns of D, and the decayed V' hi and lo those of X_k, V' hi those of R:
// each is written after the other has been read.
constexpr uint32_t kTmS = 0, kTmXk = 128, kTmXq = 192, kTmR = 256, kTmV = 320, kTmY = 384;
// ... and of the first kernel: [k; q] k^T, and the operand and result of a product within the solve.
constexpr uint32_t kTmKk = 0, kTmZ = 64, kTmU = 96;

// Tensor maps of v (boxes of 64 rows of one head) and the output (32 rows of 32 columns).
struct GdnMaps {
    CUtensorMap v, out;
};

// What is found for a chunk and value head: swizzled tiles and the factors of each row.
struct GdnTiles {
    uint8_t t_hi[64 * 128], t_lo[64 * 128];   // rows i, columns j of T
    uint8_t p[64 * 128];                      // of P
    float c_x[kChunk], c_b[kChunk];           // R = c_b v + c_x X_k
    float c_v[kChunk], c_u[kChunk];           // V' decayed to the chunk's end, and for Y
    float c_q[kChunk], c_p[kChunk];           // out = c_q X_q + c_p Y
    float gamma;
    float pad[127];
};
constexpr uint32_t kGdnTilesBytes = 3 * 64 * 128 + 6 * 4 * kChunk + 16;   // what of it is copied
static_assert(sizeof(GdnTiles) % 1024 == 0, "tiles start on swizzle atoms");

// Scratch of one launch of both kernels, for `chunks` chunks from the x0-th on (chunks of the sequences one after the other).
struct GdnScratch {
    uint8_t* kq;                              // [chunks][k_heads][DK / 64][64 rows of k, then of q][64 fp16], 128-byte swizzle
    GdnTiles* tiles;                          // [chunks][v_heads]
    int x0, chunks;
    int heads;                                // value heads of a key head that a block of the first kernel takes
};

struct GdnTilesShared {
    uint8_t kq[2][128 * 128];                 // ... and, once k k^T and q k^T are there, a head's GdnTiles on their way out
    uint8_t a21[2][32 * 128];                 // A[32.., ..31] hi and lo: rows of 64 fp16, of which 32 are used
    float a11[32 * 32], a22[32 * 32];         // -A's diagonal blocks; 16-byte pieces of a row xor-ed with row % 8
    float g_hi[4][kChunk], g_lo[4][kChunk], beta[4][kChunk];   // of four value heads: G in log2, as hi + lo
    float row_k[kChunk], row_q[kChunk];       // scales of the rows of k and q
    int bad_k[2], bad[4];                     // first row of k (of either half) and of four value heads that is not finite, or 64
    uint64_t kk_done, z_done, drained[2];
    uint32_t tmem;
    uint32_t abort;
};

struct GdnShared {
    uint8_t kq[kKqSlots][2][128 * 128];
    GdnTiles tiles[2];
    __nv_bfloat16 v[2][kChunk * 128];         // rows of DV values
    __nv_bfloat16 out[8][32 * 32];            // a warp's 32 rows of 32 output columns
    float xch[2][8][32], mu[8][32];
    uint64_t kq_in[kKqSlots], kq_free[kKqSlots], v_in[2], v_free[2], tiles_in[2], tiles_free[2];
    uint64_t s_ready, r_ready, v_ready, x_done, v_done, d_done, y_done, drained;
    int length[kGdnSorted], sequence, before;
    uint32_t tmem;
    uint32_t abort;
};

static_assert(sizeof(GdnTiles) <= sizeof(GdnTilesShared::kq), "tiles go out by way of k and q");

static __device__ unsigned g_mixer_status;    // REAX_STATUS_* bits of waits that expired

REAX_DEVI uint32_t timer_lo() {
    uint32_t t;
    asm volatile("mov.u32 %0, %%globaltimer_lo;" : "=r"(t));
    return t;
}
// Wait for a phase, for at most limit_ns.  Once a wait of the block has expired all of them return at once, and a role that
// knows of it (`dead`) neither arrives at barriers nor starts copies or MMAs any more, but goes through its loop, so that
// the block ends; the flag then goes to the status word, which says that the results are invalid.
struct GdnWait {
    volatile uint32_t* abort;
    uint32_t limit_ns;
    bool dead = false;
    REAX_DEVI void operator()(uint64_t* bar, uint32_t parity, uint32_t bit) {
        if (mbar_try_wait_suspend(bar, parity, 2000u)) return;
        const uint32_t t0 = timer_lo();
        while (!mbar_try_wait_suspend(bar, parity, 2000u)) {
            if (*abort) {
                dead = true;
                return;
            }
            if (timer_lo() - t0 > limit_ns) *abort = bit;
        }
    }
};
constexpr unsigned long long kDrainNs = 2000000000ull;   // bound of the waits for a block's own copies and MMAs at its end
// Wait for the MMAs that this thread has issued (their TMEM and shared memory may be given back then).
REAX_DEVI void drain_mmas(uint64_t* bar) {
    umma_commit(bar);
    mbar_wait_bounded(bar, 0, kDrainNs, nullptr);
}

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

// One row's solve z (I + a) = p in place, z and p of 32 columns; `neg` holds -a, of which the part below the diagonal is
// used (and zeros on it).  Four columns at a time from the last to the first: solved among themselves, then taken out of
// the columns before them.  The rows of `neg` are the same for all lanes (broadcasts) and do not depend on z, so that
// their loads run ahead of the chain.
REAX_DEVI void solve32(uint64_t (&z)[16], const float* neg) {
#pragma unroll
    for (int b = 7; b >= 0; --b) {
        auto row = [&](int r, int c) {
            return *reinterpret_cast<const ulonglong2*>(neg + (4 * b + r) * 32 + ((c ^ ((4 * b + r) & 7)) * 4));
        };
        auto twice = [](float x) { return f2(x, x); };
        const ulonglong2 a3 = row(3, b), a2 = row(2, b), a1 = row(1, b);
        z[2 * b + 1] = fma2_rn(twice(f2_hi(z[2 * b + 1])), a3.y, z[2 * b + 1]);
        z[2 * b] = fma2_rn(twice(f2_hi(z[2 * b + 1])), a3.x, z[2 * b]);
        z[2 * b] = fma2_rn(twice(f2_lo(z[2 * b + 1])), a2.x, z[2 * b]);
        z[2 * b] = fma2_rn(twice(f2_hi(z[2 * b])), a1.x, z[2 * b]);
#pragma unroll
        for (int c = b - 1; c >= 0; --c)
#pragma unroll
            for (int r = 3; r >= 0; --r) {
                const ulonglong2 x = row(r, c);
                const uint64_t zz = twice(r % 2 ? f2_hi(z[2 * b + r / 2]) : f2_lo(z[2 * b + r / 2]));
                z[2 * c] = fma2_rn(zz, x.x, z[2 * c]);
                z[2 * c + 1] = fma2_rn(zz, x.y, z[2 * c + 1]);
            }
    }
}

// Two float32 of a packed pair, times `f`, as fp16 pairs hi + lo.
REAX_DEVI void split2(uint64_t x, uint64_t f, uint32_t& hi, uint32_t& lo) {
    const uint64_t y = mul2_rn(x, f);
    const __half2 h = __floats2half2_rn(f2_lo(y), f2_hi(y));
    const float2 back = __half22float2(h);
    const uint64_t rest = sub2_rn(y, f2(back.x, back.y));
    const __half2 l = __floats2half2_rn(f2_lo(rest), f2_hi(rest));
    hi = *reinterpret_cast<const uint32_t*>(&h);
    lo = *reinterpret_cast<const uint32_t*>(&l);
}
REAX_DEVI uint32_t half2_of(uint64_t x) { return half2_bits(f2_lo(x), f2_hi(x)); }
REAX_DEVI float max3(float m, uint64_t x) { return fmaxf(m, fmaxf(fabsf(f2_lo(x)), fabsf(f2_hi(x)))); }
// ... that a NaN is not lost in.
REAX_DEVI float max3_nan(float m, uint64_t x) {
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(fabsf(f2_lo(x))), "f"(fabsf(f2_hi(x))));
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(m), "f"(y));
    return y;
}

REAX_DEVI uint64_t u2(uint32_t lo, uint32_t hi) { return (static_cast<uint64_t>(hi) << 32) | lo; }
REAX_DEVI void tmem_st_x8(uint32_t taddr, const uint32_t (&r)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(r[0]), "r"(r[1]),
                 "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
}
REAX_DEVI void tmem_ld_x16_sync(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr)
        : "memory");
}

// Copy `bytes` (a multiple of 16) of this block's shared memory to global memory, in the thread's bulk group.
REAX_DEVI void bulk_store(void* gdst, const void* smem_src, uint32_t bytes) {
    asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(gdst), "r"(smem_u32(smem_src)), "r"(bytes) : "memory");
}

// Chunks of sequence b.
REAX_DEVI int gdn_chunks_of(const GdnParams& p, int b) {
    int lo, hi;
    gdn_rows(p, b, &lo, &hi);
    return (hi - lo + kChunk - 1) / kChunk;
}

// k and q tiles, T, P and factors of chunk x0 + blockIdx.x for the value heads of key head blockIdx.y.  Four blocks share an
// SM: what one waits for (its rows, its products, the solve's chain) the others fill.
template <int DK>
__global__ void __launch_bounds__(kTilesThreads, 4) gdn_tiles_kernel(const __grid_constant__ GdnParams p, const GdnScratch out, uint32_t limit_ns) {
    extern __shared__ uint8_t tiles_smem[];
    // (an offset into the array, not an integer made a pointer: the accesses stay known as shared-memory ones)
    GdnTilesShared& sh = *reinterpret_cast<GdnTilesShared*>(tiles_smem + (-smem_u32(tiles_smem) & 1023u));
    const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32, hk = blockIdx.y;
    const int group = p.v_heads / p.k_heads, head0 = blockIdx.z * out.heads, heads = min(out.heads, group - head0);
    asm volatile("griddepcontrol.launch_dependents;");                // (which wait for the end of this grid)
    // the sequence and its chunk
    int b = -1, c = 0;
    for (int b0 = 0, before = 0; b0 < p.batch; b0 += 32) {
        const int n = b0 + lane < p.batch ? gdn_chunks_of(p, b0 + lane) : 0;
        int upto = n;
#pragma unroll
        for (int m = 1; m < 32; m <<= 1) {
            const int t = __shfl_up_sync(0xFFFFFFFFu, upto, m);
            if (lane >= m) upto += t;
        }
        const int x = out.x0 + static_cast<int>(blockIdx.x);
        const unsigned who = __ballot_sync(0xFFFFFFFFu, before + upto > x);
        if (who) {
            const int l = __ffs(who) - 1;
            b = b0 + l;
            c = x - before - __shfl_sync(0xFFFFFFFFu, upto - n, l);
            break;
        }
        before += __shfl_sync(0xFFFFFFFFu, upto, 31);
    }
    if (b < 0 || gdn_slot(p, b) < 0) return;
    int r0, r1;
    gdn_rows(p, b, &r0, &r1);
    r0 += c * kChunk;
    const int left = r1 - r0;                                         // rows of the chunk, if below 64

    if (warp == 0) {
        tmem_alloc(&sh.tmem, 128);
        tmem_relinquish();                                            // the SM's next block may allocate before this one ends
    }
    if (tid == 0) {
        mbar_init(&sh.kk_done, 1), mbar_init(&sh.z_done, 1), mbar_init(&sh.drained[0], 1), mbar_init(&sh.drained[1], 1);
        sh.abort = 0;
        fence_mbar_init();
    }
    {
        // k and q rows -> fp16, four lanes a row, scaled to a 2-norm in [2^13, 2^14) (a norm below 2^-60, whose square may
        // underflow, counts as 2^-60); rows past the end are zeros.  A lane's pieces of its row come in an order that the
        // row's number turns, so that the eight lanes of a shared-memory pass meet all banks.
        constexpr int kPieces = DK / 8, kTurns = kPieces / 4;
        const int r8 = lane / 4;
        int bad = kChunk;
        uint4 raw[4][kTurns];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int r = warp * 32 + u * 8 + r8;
            const bool real = r % 64 < left;
            const __nv_bfloat16* row = r < 64 ? p.k + static_cast<long long>(r0 + (real ? r : 0)) * p.ldk + hk * DK
                                              : p.q + static_cast<long long>(r0 + (real ? r - 64 : 0)) * p.ldq + hk * DK;
#pragma unroll
            for (int x = 0; x < kTurns; ++x)
                raw[u][x] = real ? *reinterpret_cast<const uint4*>(row + (((x + r8) % kTurns) * 4 + lane % 4) * 8) : uint4{};
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int r = warp * 32 + u * 8 + r8;
            uint64_t sum[2] = {};
#pragma unroll
            for (int x = 0; x < kTurns; ++x) {
                const uint32_t y[4] = {raw[u][x].x, raw[u][x].y, raw[u][x].z, raw[u][x].w};
#pragma unroll
                for (int j = 0; j < 4; ++j) sum[j & 1] = fma2_rn(bf16x2_to_f2(y[j]), bf16x2_to_f2(y[j]), sum[j & 1]);
            }
            sum[0] = add2_rn(sum[0], sum[1]);
            float sq = f2_lo(sum[0]) + f2_hi(sum[0]);
            sq += __shfl_xor_sync(0xFFFFFFFFu, sq, 1);
            sq += __shfl_xor_sync(0xFFFFFFFFu, sq, 2);
            // a row of k that is not finite (its sum of squares is not) is left out
            const bool out_of_k = warp < 2 && !(sq < INFINITY);
            const unsigned who = __ballot_sync(0xFFFFFFFFu, out_of_k);
            if (who) bad = min(bad, warp * 32 + u * 8 + (__ffs(who) - 1) / 4);
            // 2^(k - 1) <= norm < 2^k
            const int k = static_cast<int>((max(__float_as_uint(sq) >> 23, 7u) + 1) >> 1) - 63;
            const float f = __uint_as_float(static_cast<uint32_t>(127 + 14 - k) << 23);
            float back = __uint_as_float(static_cast<uint32_t>(127 - 14 + k) << 23);
            if (p.normalize) back *= rsqrtf(sq + kGdnNormEps);
#pragma unroll
            for (int x = 0; x < kTurns; ++x) {
                const int at = ((x + r8) % kTurns) * 4 + lane % 4;
                if (out_of_k) raw[u][x] = uint4{};
                const uint32_t y[4] = {raw[u][x].x, raw[u][x].y, raw[u][x].z, raw[u][x].w};
                uint32_t o[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) o[j] = half2_of(mul2_rn(bf16x2_to_f2(y[j]), f2(f, f)));
                *reinterpret_cast<uint4*>(sh.kq[at / 8] + r * 128 + ((at % 8) ^ r8) * 16) = uint4{o[0], o[1], o[2], o[3]};
            }
            if (lane % 4 == 0) (r < 64 ? sh.row_k : sh.row_q - 64)[r] = r % 64 >= left || out_of_k ? 0.0f : r < 64 ? back : back * p.scale;
        }
        if (warp < 2 && lane == 0) sh.bad_k[warp] = bad;
        fence_proxy_async_smem();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tm = sh.tmem;
    GdnWait wait{&sh.abort, limit_ns};
    if (tid == 0) {
        const uint64_t d = sw128_kmajor_desc(smem_u32(sh.kq));
#pragma unroll
        for (int ks = 0; ks < DK / 16; ++ks) {
            const uint64_t y = d + (ks / 4) * 1024 + (ks % 4) * 2;
            umma_f16(tm + kTmKk, y, y, idesc_f16_f32(128, 64, false), ks > 0);
        }
        umma_commit(&sh.kk_done);
        if (head0 == 0) {
            bulk_store(out.kq + (static_cast<long long>(blockIdx.x) * p.k_heads + hk) * (DK / 64) * 16384, sh.kq, (DK / 64) * 16384);
            bulk_commit_group();
        }
        bulk_wait_read_all();
    }
    __syncwarp();

    const uint32_t lanes = tm + (static_cast<uint32_t>(warp * 32) << 16);
    const int l = lane;
    const bool is_q = warp >= 2, upper = (warp & 1) != 0;             // warps 0, 1: rows of k; 2, 3: of q; upper: rows 32..
    const int i = upper ? 32 + l : l;                                 // this lane's row
    auto piece = [&](int j) { return (j ^ (l & 7)); };
    const float row_k = sh.row_k[i];
    GdnTiles& st = *reinterpret_cast<GdnTiles*>(sh.kq);
    uint32_t turn = 0;
#pragma unroll 1
    for (int head = 0; head < heads; ++head) {
        if (head % 4 == 0) {
            // running sums of g of four heads, one a warp, in log2 units: multiples of 2^-8 (exact in float32) and the rest,
            // so that differences of far running sums keep their low bits; decays below 2^-128 count as 0
            if (head > 0) __syncthreads();
            if (head + warp < heads) {
                float hi[2], lo[2], be[2], y[2];
                int bad = min(sh.bad_k[0], sh.bad_k[1]);
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const bool real = lane * 2 + j < left;
                    const long long at = (static_cast<long long>(r0) + (real ? lane * 2 + j : 0)) * p.v_heads + hk * group + head0 + head + warp;
                    y[j] = real ? p.g[at] * 1.44269504f : 0.0f;
                    be[j] = real ? p.beta[at] : 0.0f;
                    // (a decay of e^-inf is finite)
                    const unsigned who = __ballot_sync(0xFFFFFFFFu, !(y[j] < 128.0f) || !(fabsf(be[j]) < INFINITY));
                    if (who) bad = min(bad, 2 * (__ffs(who) - 1) + j);
                }
                if (lane == 0) sh.bad[warp] = bad;
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    if (lane * 2 + j >= bad) y[j] = be[j] = 0.0f;
                    const float x = y[j] < -128.0f ? -128.0f : y[j];
                    hi[j] = rintf(x * 256.0f) * 0.00390625f;
                    lo[j] = x - hi[j];
                }
                float sum_h = hi[0] + hi[1], sum_l = lo[0] + lo[1];
#pragma unroll 1
                for (int m = 1; m < 32; m <<= 1) {
                    const float a = __shfl_up_sync(0xFFFFFFFFu, sum_h, m), x = __shfl_up_sync(0xFFFFFFFFu, sum_l, m);
                    if (lane >= m) sum_h += a, sum_l += x;
                }
                *reinterpret_cast<float2*>(sh.g_hi[warp] + 2 * lane) = float2{sum_h - hi[1], sum_h};
                *reinterpret_cast<float2*>(sh.g_lo[warp] + 2 * lane) = float2{sum_l - lo[1], sum_l};
                *reinterpret_cast<float2*>(sh.beta[warp] + 2 * lane) = float2{be[0], be[1]};
            }
            __syncthreads();
            if (head == 0) {
                wait(&sh.kk_done, 0, kStatusTimeoutAccFull);
                tc_fence_after();
            }
        }
        const float *g_hi_s = sh.g_hi[head % 4], *g_lo_s = sh.g_lo[head % 4], *beta_s = sh.beta[head % 4];
        GdnTiles* to = out.tiles + static_cast<long long>(blockIdx.x) * p.v_heads + hk * group + head0 + head;
        {
            const float g_hi = g_hi_s[i], g_lo = g_lo_s[i], beta = beta_s[i];
            // the head before has left the tiles
            if (tid % 64 == 0) bulk_wait_read_all();
            if (is_q) named_bar_sync(6, 64);
            // The row's products with the rows of k before it, with their decays, 8 at a time.  k and q have 2-norms below
            // 2^14, so that products times kGdnDown fit fp16 (with room for a g above 0) and need no look at the row first:
            // the scales of P's columns go with V', those of A[32.., ..31] with what it is multiplied by.
#pragma unroll 1
            for (int o = 0; o < (upper ? 64 : 32); o += 16) {
                uint32_t x[16];
                uint64_t y[8];
                tmem_ld_x16_sync(lanes + kTmKk + o, x);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const uint64_t h = sub2_rn(f2(g_hi, g_hi), *reinterpret_cast<const uint64_t*>(g_hi_s + o + 2 * e));
                    const uint64_t d = add2_rn(h, sub2_rn(f2(g_lo, g_lo), *reinterpret_cast<const uint64_t*>(g_lo_s + o + 2 * e)));
                    y[e] = mul2_rn(f2(ex2(f2_lo(d)), ex2(f2_hi(d))), u2(x[2 * e], x[2 * e + 1]));
                }
                if (is_q) {
#pragma unroll
                    for (int q = 0; q < 2; ++q) {
                        uint32_t hi[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const int at = o + 8 * q + 2 * e;
                            const uint64_t w = mul2_rn(y[4 * q + e], f2(kGdnDown, kGdnDown));
                            hi[e] = half2_bits(at <= i ? f2_lo(w) : 0.0f, at + 1 <= i ? f2_hi(w) : 0.0f);
                        }
                        *reinterpret_cast<uint4*>(st.p + i * 128 + piece(o / 8 + q) * 16) = uint4{hi[0], hi[1], hi[2], hi[3]};
                    }
                } else if (o < 32 && upper) {
#pragma unroll
                    for (int q = 0; q < 2; ++q) {
                        uint32_t hi[4], lo[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) split2(y[4 * q + e], f2(kGdnDown, kGdnDown), hi[e], lo[e]);
                        *reinterpret_cast<uint4*>(sh.a21[0] + l * 128 + piece(o / 8 + q) * 16) = uint4{hi[0], hi[1], hi[2], hi[3]};
                        *reinterpret_cast<uint4*>(sh.a21[1] + l * 128 + piece(o / 8 + q) * 16) = uint4{lo[0], lo[1], lo[2], lo[3]};
                    }
                } else {
                    const float f = -row_k * beta;
                    float* a = (upper ? sh.a22 : sh.a11) + l * 32;
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        y[e] = mul2_rn(y[e], mul2_rn(f2(f, f), *reinterpret_cast<const uint64_t*>(sh.row_k + o + 2 * e)));
#pragma unroll
                    for (int q = 0; q < 4; ++q)
                        *reinterpret_cast<ulonglong2*>(a + piece((o & 31) / 4 + q) * 4) = ulonglong2{y[2 * q], y[2 * q + 1]};
                }
            }
            if (is_q) {
                if (!upper)
#pragma unroll
                    for (int e = 4; e < 8; ++e) *reinterpret_cast<uint4*>(st.p + i * 128 + piece(e) * 16) = uint4{};
                const float f = sh.row_q[i];
                st.c_q[i] = f * ex2(g_hi + g_lo);
                st.c_p[i] = f * kGdnUp;
                if (i == 0) st.gamma = ex2(g_hi_s[kChunk - 1] + g_lo_s[kChunk - 1]);
                fence_proxy_async_smem();
                named_bar_sync(6, 64);
                if (tid == 64 && !wait.dead) {
                    bulk_store(to->p, st.p, sizeof(st.p));
                    bulk_store(to->c_q, st.c_q, kGdnTilesBytes - offsetof(GdnTiles, c_q));
                    bulk_commit_group();
                }
                __syncwarp();
                continue;
            }
            (upper ? sh.a22 : sh.a11)[l * 32 + piece(l / 4) * 4 + l % 4] = 0.0f;
            fence_proxy_async_smem();
            uint64_t z[16], z1[16];                   // T's row: columns ..31 and 32..
#pragma unroll
            for (int j = 0; j < 16; ++j) z[j] = f2(2 * j == l ? 1.0f : 0.0f, 2 * j + 1 == l ? 1.0f : 0.0f), z1[j] = 0;
            named_bar_sync(5, 64);
#pragma unroll 1
            for (int pass = upper ? 0 : 1; pass < 2; ++pass) {
                solve32(z, pass == 0 ? sh.a22 : sh.a11);
                if (pass == 0) {
                    // z (columns 32..) is done; its product with A[32.., ..31] on the tensor cores, then columns ..31
                    uint64_t y[16];
                    float m = 0.0f;
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        y[j] = mul2_rn(z[j], mul2_rn(*reinterpret_cast<const uint64_t*>(beta_s + 32 + 2 * j),
                                                     *reinterpret_cast<const uint64_t*>(sh.row_k + 32 + 2 * j)));
                        m = max3(m, y[j]);
                    }
                    const float2 f = scale_of(m);
                    uint32_t hi[16], lo[16];
#pragma unroll
                    for (int j = 0; j < 16; ++j) split2(y[j], f2(f.x, f.x), hi[j], lo[j]);
                    tmem_st_x16(lanes + kTmZ, hi);
                    tmem_st_x16(lanes + kTmZ + 16, lo);
                    tmem_wait_st();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0 && !wait.dead) {
                        tc_fence_after();
                        const uint64_t hi_desc = sw128_mn_desc(smem_u32(sh.a21[0]), 4096), lo_desc = sw128_mn_desc(smem_u32(sh.a21[1]), 4096);
#pragma unroll 2
                        for (int e = 0; e < 6; ++e) {
                            const int ks = e % 2, term = e / 2;
                            umma_f16_ts(tm + kTmU, tm + kTmZ + (term == 1 ? 16 : 0) + ks * 8, (term == 2 ? lo_desc : hi_desc) + ks * 128,
                                        idesc_f16_f32(128, 32, true), e > 0);
                        }
                        umma_commit(&sh.z_done);
                    }
                    __syncwarp();
                    wait(&sh.z_done, turn & 1, kStatusTimeoutAccFull);
                    tc_fence_after();
                    uint32_t x[32];
                    tmem_ld_x32_sync(lanes + kTmU, x);
                    tc_fence_before();
                    const float g = -f.y * kGdnUp;
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        z1[j] = z[j];
                        z[j] = mul2_rn(u2(x[2 * j], x[2 * j + 1]), mul2_rn(f2(g, g), *reinterpret_cast<const uint64_t*>(sh.row_k + 2 * j)));
                    }
                }
            }
            float m = 0.0f;
#pragma unroll
            for (int j = 0; j < 16; ++j) m = max3(max3(m, z[j]), z1[j]);
            const float2 f = scale_of(m);
            st.c_x[i] = i >= sh.bad[head % 4] ? __uint_as_float(kGdnNan) : -row_k * beta * ex2(g_hi + g_lo);
            st.c_b[i] = beta;
            st.c_v[i] = row_k * ex2((g_hi_s[kChunk - 1] - g_hi) + (g_lo_s[kChunk - 1] - g_lo)) * f.y;
            st.c_u[i] = row_k * f.y;
#pragma unroll 1
            for (int o = 0; o < 8; o += 4) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    uint32_t hi[4], lo[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) split2(z[4 * j + e], f2(f.x, f.x), hi[e], lo[e]);
                    *reinterpret_cast<uint4*>(st.t_hi + i * 128 + piece(o + j) * 16) = uint4{hi[0], hi[1], hi[2], hi[3]};
                    *reinterpret_cast<uint4*>(st.t_lo + i * 128 + piece(o + j) * 16) = uint4{lo[0], lo[1], lo[2], lo[3]};
                }
#pragma unroll
                for (int j = 0; j < 16; ++j) z[j] = z1[j];
            }
            fence_proxy_async_smem();
            named_bar_sync(5, 64);                    // (the next head may have a11, a22 and a21 as well)
            if (tid == 0 && !wait.dead) {
                bulk_store(to->t_hi, st.t_hi, sizeof(st.t_hi) + sizeof(st.t_lo));
                bulk_store(to->c_x, st.c_x, 4 * sizeof(st.c_x));
                bulk_commit_group();
            }
            __syncwarp();
            ++turn;
        }
    }
    if (warp < 2 && lane == 0) drain_mmas(&sh.drained[warp]);
    if (tid % 64 == 0) bulk_wait_all();
    tc_fence_before();
    __syncthreads();
    if (tid == 0 && sh.abort) atomicOr(&g_mixer_status, sh.abort);
    if (warp == 0) tmem_dealloc(tm, 128);
}

template <int DK, int DV>
__global__ void __launch_bounds__(kChunkThreads, 1) gdn_chunk_kernel(const __grid_constant__ GdnParams p,
                                                                     const __grid_constant__ GdnMaps maps, const GdnScratch in,
                                                                     uint32_t limit_ns) {
    extern __shared__ uint8_t smem_raw[];
    GdnShared& sh = *reinterpret_cast<GdnShared*>(smem_raw + (-smem_u32(smem_raw) & 1023u));
    const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
    const int hv = blockIdx.x, hk = hv / (p.v_heads / p.k_heads);
    int r0, r1, b = blockIdx.y;
    if (gridDim.y > 1 && gridDim.y <= kGdnSorted) {
        // blocks start in their order: the longest sequences first, so that no long one is left for the end
        if (tid < p.batch) {
            gdn_rows(p, tid, &r0, &r1);
            sh.length[tid] = r1 - r0;
        }
        __syncthreads();
        if (tid < p.batch) {
            const int mine = sh.length[tid];
            int rank = 0;
            for (int i = 0; i < p.batch; ++i) rank += sh.length[i] > mine || (sh.length[i] == mine && i < tid);
            if (rank == static_cast<int>(blockIdx.y)) sh.sequence = tid;
        }
        __syncthreads();
        b = sh.sequence;
    }
    // chunks of the sequences before
    if (tid == 0) sh.before = 0;
    __syncthreads();
    {
        int n = 0;
        for (int i = tid; i < b; i += kChunkThreads) n += gdn_chunks_of(p, i);
        if (n) atomicAdd(&sh.before, n);
    }
    __syncthreads();
    gdn_rows(p, b, &r0, &r1);
    const int slot = gdn_slot(p, b), all = gdn_chunks_of(p, b);
    // this launch's part of the sequence
    const int first = max(in.x0 - sh.before, 0), chunks = min(all, in.x0 + in.chunks - sh.before) - first;
    const int x_first = sh.before + first - in.x0;                    // its place in the scratch memory
    const bool from_state = p.carry || first > 0;
    r0 += first * kChunk;
    const int rows = min(r1 - r0, chunks * kChunk);
    float* state = p.state + (static_cast<long long>(max(slot, 0)) * p.v_heads + hv) * DK * DV;
    if (slot < 0 || chunks <= 0) {
        asm volatile("griddepcontrol.wait;" ::: "memory");
        if (slot < 0) {
            __nv_bfloat16* o = p.out + (static_cast<long long>(r0) * p.v_heads + hv) * DV;
            for (int e = tid; e < rows * (DV / 8); e += kChunkThreads)
                *reinterpret_cast<uint4*>(o + static_cast<long long>(e / (DV / 8)) * p.v_heads * DV + e % (DV / 8) * 8) = uint4{};
        } else if (all == 0 && !p.carry && in.x0 == 0) {
            for (int e = tid; e < DK * DV; e += kChunkThreads) state[e] = 0.0f;
        }
        return;
    }

    if (warp == 8) tmem_alloc(&sh.tmem, 512);
    if (tid == 0) {
        for (int i = 0; i < kKqSlots; ++i) mbar_init(&sh.kq_in[i], 1), mbar_init(&sh.kq_free[i], 1);
        for (int i = 0; i < 2; ++i) mbar_init(&sh.v_in[i], 1), mbar_init(&sh.v_free[i], 8);
        for (int i = 0; i < 2; ++i) mbar_init(&sh.tiles_in[i], 1), mbar_init(&sh.tiles_free[i], 8);
        mbar_init(&sh.s_ready, 8), mbar_init(&sh.r_ready, 8), mbar_init(&sh.v_ready, 8);
        mbar_init(&sh.x_done, 1), mbar_init(&sh.v_done, 1), mbar_init(&sh.d_done, 1), mbar_init(&sh.y_done, 1);
        mbar_init(&sh.drained, 1);
        sh.abort = 0;
        fence_mbar_init();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tm = sh.tmem;
    asm volatile("griddepcontrol.wait;" ::: "memory");                // the tiles, and all that came before
    GdnWait wait{&sh.abort, limit_ns};
    const int quarter = warp % 4;
    const uint32_t lanes = tm + (static_cast<uint32_t>(quarter * 32) << 16);
    // One arrival for the warp, after what all its lanes have done.
    auto arrive = [&](uint64_t* bar) {
        __syncwarp();
        if (lane == 0 && !wait.dead) mbar_arrive(bar);
    };

    if (warp < 8) {
        // ------------------------------------------------------------------------------------ the state's warps
        const int part = warp / 4, n = quarter * 32 + lane;       // rows 32 part .. of a chunk, S's DK / 2 part ..
        constexpr int kS = DK / 2;
        uint64_t s[kS / 2];
#pragma unroll
        for (int i = 0; i < kS / 2; ++i) {
            const float* at = state + (part * kS + 2 * i) * DV + n;
            s[i] = from_state && n < DV ? f2(at[0], at[DV]) : 0;
        }
        int turn = 0;
        // Largest of both parts of this thread's row (the two warps of a quarter meet).  Both get the same value whatever else has
        // happened, expired waits included: a place is written again only behind the barrier after the one it was read behind.
        auto row_max = [&](float m) {
            float* x = &sh.xch[turn][quarter * 2][lane];
            x[part * 32] = m;
            named_bar_sync(1 + quarter, 64);
            turn ^= 1;
            return fmaxf(x[0], x[32]);
        };
        auto pair_of = [](const float* f) { return *reinterpret_cast<const uint64_t*>(f); };
        const uint16_t* vcol = reinterpret_cast<const uint16_t*>(sh.v[0]) + part * 32 * DV + (n < DV ? n : 0);
        float sq = 0.0f, sv = 0.0f;          // scales of the S behind X_q and the V' behind Y
        int bad = kChunk;                     // the chunk's first row whose R is not finite in this column
#pragma unroll 1
        for (int c = 0;; ++c) {                // (c counts from the first chunk of this launch)
            const uint32_t par = c & 1;
            float2 ss = {};
            if (c < chunks) {
                // S -> two fp16 operands
                float m = 0.0f;
#pragma unroll
                for (int i = 0; i < kS / 2; ++i) m = max3(m, s[i]);
                ss = scale_of(row_max(m));
#pragma unroll
                for (int x = 0; x < kS / 16; ++x) {
                    uint32_t hi[8], lo[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) split2(s[x * 8 + i], f2(ss.x, ss.x), hi[i], lo[i]);
                    tmem_st_x8(lanes + kTmS + part * (kS / 2) + x * 8, hi);
                    tmem_st_x8(lanes + kTmS + 64 + part * (kS / 2) + x * 8, lo);
                }
                tmem_wait_st();
                tc_fence_before();
                arrive(&sh.s_ready);
            }
            if (c > 0) {
                // the rows out of the chunk before, through shared memory: 32 rows of 32 columns a warp
                const GdnTiles& st = sh.tiles[par ^ 1];
                wait(&sh.y_done, par ^ 1, kStatusTimeoutAccFull);
                tc_fence_after();
                if (lane == 0) bulk_wait_read_all();
                __syncwarp();
                uint16_t* o = reinterpret_cast<uint16_t*>(sh.out[warp]) + lane;
#pragma unroll
                for (int e = 0; e < 32; e += 16) {
                    uint32_t x[16], y[16];
                    // (factors first: the compiler must not move a load over a store that it cannot tell apart)
                    uint64_t cq[8], cp[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) cq[i] = pair_of(st.c_q + part * 32 + e + 2 * i), cp[i] = pair_of(st.c_p + part * 32 + e + 2 * i);
                    tmem_ld2_x16_sync(lanes + kTmXq + part * 32 + e, lanes + kTmY + part * 32 + e, x, y);
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const uint64_t z = mul2_rn(u2(x[2 * i], x[2 * i + 1]), mul2_rn(cq[i], f2(sq, sq)));
                        const uint32_t w = bf16x2_rn(fma2_rn(u2(y[2 * i], y[2 * i + 1]), mul2_rn(cp[i], f2(sv, sv)), z));
                        o[(e + 2 * i) * 32] = static_cast<uint16_t>(w);
                        o[(e + 2 * i + 1) * 32] = static_cast<uint16_t>(w >> 16);
                    }
                }
                tc_fence_before();
                arrive(&sh.tiles_free[par ^ 1]);
#pragma unroll 1
                for (int i = max(bad - part * 32, 0); i < 32; ++i) o[i * 32] = kGdnNan >> 16;
                __syncwarp();
                const int row = (c - 1) * kChunk + part * 32, left = rows - row;
                if (quarter * 32 < DV) {
                    if (left >= 32) {
                        fence_proxy_async_smem();
                        __syncwarp();
                        if (lane == 0) {
                            tma_store_2d(&maps.out, sh.out[warp], hv * DV + quarter * 32, r0 + row);
                            bulk_commit_group();
                        }
                    } else {
                        uint16_t* to = reinterpret_cast<uint16_t*>(p.out);
#pragma unroll 1
                        for (int i = 0; i < left; ++i) to[(static_cast<long long>(r0 + row + i) * p.v_heads + hv) * DV + n] = o[i * 32];
                    }
                }
            }
            if (c == chunks) break;
            const GdnTiles& st = sh.tiles[par];
            sq = ss.y;
            // X_k -> R
            wait(&sh.tiles_in[par], (c >> 1) & 1, kStatusTimeoutFull);
            wait(&sh.v_in[par], (c >> 1) & 1, kStatusTimeoutFull);
            wait(&sh.x_done, par, kStatusTimeoutAccFull);
            tc_fence_after();
            uint32_t x[32];
            float m = 0.0f;
            {
                uint64_t r[16];
                tmem_ld_x32_sync(lanes + kTmXk + part * 32, x);
                const uint16_t* v = vcol + par * (kChunk * 128);
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const int at = part * 32 + 2 * i;
                    const uint64_t y = u2(static_cast<uint32_t>(v[2 * i * DV]) << 16, static_cast<uint32_t>(v[(2 * i + 1) * DV]) << 16);
                    r[i] = fma2_rn(u2(x[2 * i], x[2 * i + 1]), mul2_rn(pair_of(st.c_x + at), f2(ss.y, ss.y)), mul2_rn(pair_of(st.c_b + at), y));
                }
                if (rows - c * kChunk < kChunk)            // rows past the end, which the box takes from what follows
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const int left = rows - c * kChunk - part * 32 - 2 * i;
                        r[i] = f2(left > 0 ? f2_lo(r[i]) : 0.0f, left > 1 ? f2_hi(r[i]) : 0.0f);
                    }
                arrive(&sh.v_free[par]);
#pragma unroll
                for (int i = 0; i < 16; ++i) m = max3_nan(m, r[i]);
                float most = row_max(m < INFINITY ? m : INFINITY);
                bad = kChunk;
                if (__any_sync(0xFFFFFFFFu, most == INFINITY)) {      // (in both warps of a quarter)
#pragma unroll
                    for (int i = 15; i >= 0; --i) {
                        if (!(fabsf(f2_hi(r[i])) < INFINITY)) bad = part * 32 + 2 * i + 1;
                        if (!(fabsf(f2_lo(r[i])) < INFINITY)) bad = part * 32 + 2 * i;
                    }
                    bad = kChunk - static_cast<int>(row_max(static_cast<float>(kChunk - bad)));
                    m = 0.0f;
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const int at = part * 32 + 2 * i;
                        r[i] = f2(at < bad ? f2_lo(r[i]) : 0.0f, at + 1 < bad ? f2_hi(r[i]) : 0.0f);
                        m = max3(m, r[i]);
                    }
                    most = row_max(m);
                }
                const float2 rs = scale_of(most);
                sv = rs.y;
#pragma unroll
                for (int e = 0; e < 16; e += 8) {
                    uint32_t hi[8], lo[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) split2(r[e + i], f2(rs.x, rs.x), hi[i], lo[i]);
                    tmem_st_x8(lanes + kTmR + part * 16 + e, hi);
                    tmem_st_x8(lanes + kTmR + 32 + part * 16 + e, lo);
                }
            }
            tmem_wait_st();
            tc_fence_before();
            arrive(&sh.r_ready);
            // V', decayed to the chunk's end for D and as it is for Y
            wait(&sh.v_done, par, kStatusTimeoutAccFull);
            tc_fence_after();
            tmem_ld_x32_sync(lanes + kTmV + part * 32, x);
            float mu = 0.0f;
            m = 0.0f;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int at = part * 32 + 2 * i;
                m = max3(m, mul2_rn(u2(x[2 * i], x[2 * i + 1]), pair_of(st.c_v + at)));
                mu = max3(mu, mul2_rn(u2(x[2 * i], x[2 * i + 1]), pair_of(st.c_u + at)));
            }
            sh.mu[quarter * 2 + part][lane] = mu;                 // read behind row_max's barrier
            const float2 vs = scale_of(row_max(m));
            const float2 us = scale_of(fmaxf(sh.mu[quarter * 2][lane], sh.mu[quarter * 2 + 1][lane]));
#pragma unroll
            for (int e = 0; e < 16; e += 8) {
                uint32_t hi[8], lo[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int at = part * 32 + 2 * (e + i);
                    split2(mul2_rn(u2(x[2 * (e + i)], x[2 * (e + i) + 1]), pair_of(st.c_v + at)), f2(vs.x, vs.x), hi[i], lo[i]);
                }
                tmem_st_x8(lanes + kTmXk + part * 16 + e, hi);
                tmem_st_x8(lanes + kTmXk + 32 + part * 16 + e, lo);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int at = part * 32 + 2 * (e + i);
                    hi[i] = half2_of(mul2_rn(mul2_rn(u2(x[2 * (e + i)], x[2 * (e + i) + 1]), pair_of(st.c_u + at)), f2(us.x, us.x)));
                }
                tmem_st_x8(lanes + kTmR + part * 16 + e, hi);
            }
            tmem_wait_st();
            tc_fence_before();
            arrive(&sh.v_ready);
            // (R's scale is that of V' until here)
            const float back = vs.y * sv, gamma = bad < kChunk ? __uint_as_float(kGdnNan) : st.gamma;
            sv *= us.y;
            // D -> S
#pragma unroll
            for (int i = 0; i < kS / 2; ++i) s[i] = mul2_rn(s[i], f2(gamma, gamma));
            wait(&sh.d_done, par, kStatusTimeoutAccFull);
            tc_fence_after();
#pragma unroll
            for (int y = 0; y < kS / 32; ++y) {
                tmem_ld_x32_sync(lanes + kTmS + part * kS + y * 32, x);
#pragma unroll
                for (int i = 0; i < 16; ++i) s[y * 16 + i] = fma2_rn(f2(back, back), u2(x[2 * i], x[2 * i + 1]), s[y * 16 + i]);
            }
        }
        if (n < DV)
#pragma unroll
            for (int i = 0; i < kS / 2; ++i) {
                float* at = state + (part * kS + 2 * i) * DV + n;
                at[0] = f2_lo(s[i]), at[DV] = f2_hi(s[i]);
            }
        if (lane == 0) bulk_wait_all();
    } else if (warp == 8) {
        // --------------------------------------------------------------------------- issuer of the chain's MMAs
        if (lane == 0) {
            constexpr uint32_t id64 = idesc_f16_f32(128, 64, false);
            constexpr uint32_t id_d = idesc_f16_f32(128, DK, true);
#pragma unroll 1
            for (int c = 0, slot_k = 0; c < chunks; ++c, slot_k = slot_k == kKqSlots - 1 ? 0 : slot_k + 1) {
                const uint32_t par = c & 1;
                GdnTiles& st = sh.tiles[par];
                const uint32_t kq_at = smem_u32(sh.kq[slot_k]);
                const uint64_t kq = sw128_kmajor_desc(kq_at), kmn = sw128_mn_desc(kq_at, 16384);
                const uint64_t thi = sw128_kmajor_desc(smem_u32(st.t_hi)), tlo = sw128_kmajor_desc(smem_u32(st.t_lo));
                const uint64_t pd = sw128_kmajor_desc(smem_u32(st.p));
                wait(&sh.kq_in[slot_k], (c / kKqSlots) & 1, kStatusTimeoutFull);
                wait(&sh.s_ready, par, kStatusTimeoutEmpty);
                if (wait.dead) break;
                tc_fence_after();
                // descriptor addresses count in units of 16 bytes
#pragma unroll
                for (int e = 0; e < 2 * (DK / 16); ++e) {
                    const int ks = e % (DK / 16);
                    umma_f16_ts(tm + kTmXk, tm + kTmS + (e / (DK / 16)) * 64 + ks * 8, kq + (ks / 4) * 1024 + (ks % 4) * 2, id64, e > 0);
                }
                umma_commit(&sh.x_done);
                // the chunk before's X_q has been read
                if (c > 0) wait(&sh.tiles_free[par ^ 1], ((c - 1) >> 1) & 1, kStatusTimeoutEmpty);
                if (wait.dead) break;
                tc_fence_after();
#pragma unroll
                for (int ks = 0; ks < DK / 16; ++ks)
                    umma_f16_ts(tm + kTmXq, tm + kTmS + ks * 8, kq + 512 + (ks / 4) * 1024 + (ks % 4) * 2, id64, ks > 0);
                wait(&sh.tiles_in[par], (c >> 1) & 1, kStatusTimeoutFull);
                wait(&sh.r_ready, par, kStatusTimeoutEmpty);
                if (wait.dead) break;
                tc_fence_after();
#pragma unroll
                for (int e = 0; e < 12; ++e) {
                    const int ks = e % 4, term = e / 4;      // hi hi, lo hi, hi lo
                    umma_f16_ts(tm + kTmV, tm + kTmR + (term == 1 ? 32 : 0) + ks * 8, (term == 2 ? tlo : thi) + ks * 2, id64, e > 0);
                }
                umma_commit(&sh.v_done);
                wait(&sh.v_ready, par, kStatusTimeoutEmpty);
                if (wait.dead) break;
                tc_fence_after();
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    umma_f16_ts(tm + kTmS, tm + kTmXk + (e / 4) * 32 + (e % 4) * 8, kmn + (e % 4) * 128, id_d, e > 0);
                umma_commit(&sh.d_done);
                umma_commit(&sh.kq_free[slot_k]);
#pragma unroll
                for (int ks = 0; ks < 4; ++ks) umma_f16_ts(tm + kTmY, tm + kTmR + ks * 8, pd + ks * 2, id64, ks > 0);
                umma_commit(&sh.y_done);
            }
            drain_mmas(&sh.drained);
        }
        __syncwarp();
    } else if (lane == 0) {
        // ----------------------------------------------------------------------------------------------- loads
        constexpr uint32_t kKqBytes = (DK / 64) * 16384;
        const uint64_t policy = l2_policy_evict_normal();
        int kq_loads = 0, pair_loads = 0;
        auto load_kq = [&](int c) {
            const int slot_k = c % kKqSlots;
            if (c >= kKqSlots) wait(&sh.kq_free[slot_k], (c / kKqSlots - 1) & 1, kStatusTimeoutEmpty);
            if (wait.dead) return;
            ++kq_loads;
            mbar_arrive_expect_tx(&sh.kq_in[slot_k], kKqBytes);
            bulk_load(sh.kq[slot_k], in.kq + (static_cast<long long>(x_first + c) * p.k_heads + hk) * kKqBytes, kKqBytes, &sh.kq_in[slot_k]);
        };
        load_kq(0);
#pragma unroll 1
        for (int c = 0; c < chunks && !wait.dead; ++c) {
            const int par = c & 1;
            if (c + 1 < chunks) load_kq(c + 1);
            if (c > 1) wait(&sh.v_free[par], ((c >> 1) - 1) & 1, kStatusTimeoutEmpty), wait(&sh.tiles_free[par], ((c >> 1) - 1) & 1, kStatusTimeoutEmpty);
            if (wait.dead) break;
            ++pair_loads;
            mbar_arrive_expect_tx(&sh.v_in[par], kChunk * 2 * DV);
            tma_load_2d(sh.v[par], &maps.v, &sh.v_in[par], hv * DV, r0 + c * kChunk, policy);
            mbar_arrive_expect_tx(&sh.tiles_in[par], kGdnTilesBytes);
            bulk_load(&sh.tiles[par], in.tiles + static_cast<long long>(x_first + c) * p.v_heads + hv, kGdnTilesBytes, &sh.tiles_in[par]);
        }
        // no copy may be in flight when the block ends
        for (int c = max(kq_loads - kKqSlots, 0); c < kq_loads; ++c)
            mbar_wait_bounded(&sh.kq_in[c % kKqSlots], (c / kKqSlots) & 1, kDrainNs, nullptr);
        for (int c = max(pair_loads - 2, 0); c < pair_loads; ++c) {
            mbar_wait_bounded(&sh.v_in[c & 1], (c >> 1) & 1, kDrainNs, nullptr);
            mbar_wait_bounded(&sh.tiles_in[c & 1], (c >> 1) & 1, kDrainNs, nullptr);
        }
    }
    tc_fence_before();
    __syncthreads();
    if (tid == 0 && sh.abort) atomicOr(&g_mixer_status, sh.abort);
    if (warp == 8) {
        tmem_relinquish();
        tmem_dealloc(tm, 512);
    }
}

constexpr size_t gdn_chunk_smem() { return sizeof(GdnShared) + 1024; }
constexpr size_t gdn_tiles_smem() { return sizeof(GdnTilesShared) + 1024; }
// A block of the second kernel takes all of its SM's tensor memory and then waits for the first kernel's end, so that no block of
// the first may share an SM with it: it would wait for tensor memory for good.  Their shared memory keeps them apart.
static_assert(gdn_chunk_smem() + gdn_tiles_smem() + 2 * 1024 > 228 * 1024, "blocks of both kernels fit one SM");
static_assert(gdn_chunk_smem() <= 227 * 1024 && 4 * (gdn_tiles_smem() + 1024) <= 228 * 1024, "shared memory of one SM");

}  // namespace reax
