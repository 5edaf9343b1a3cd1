// Attention of few query rows over the paged INT8 cache: a step of the serving loop.
//
// Its floor is the cache's bytes, read once: k and v codes of a page and head are copied into shared memory (16-byte
// pieces xor-ed with their row's number, against bank conflicts), are turned into fp16 in registers (exact: |code| <= 128) and
// multiplied with mma.sync m16n8k16, whose 16 rows hold the query rows and heads that share a cached head.  tcgen05 tiles would be 128 rows high, all but
// a few of them empty; at 16 rows the tensor cores work 24 % of the time.  What bounds it: 64 sequences with 261000 rows keep
// DRAM at 49 % and the issue slots at 53 %.  Outputs of 256 columns take 242 registers, which leaves two warps a scheduler, and a
// warp issues every 3.5 cycles between the latencies of its chain from codes to products.
//
// Scales.  A page's scale of k multiplies its scores.  A page's scale of v (s_v) would multiply the weights, whose fp16
// rounding it must not touch: the running maximum is that of t = score + log2(s_v), the weights are exp2(t - max)
// times 2^14, and the denominator adds them over s_v.
//
// fp16 weights.  A weight below 2^-28 of the largest is subnormal there.  Where a warp meets one, which takes scores that
// differ by more than 19, it multiplies such weights in passes of their own, times 2^29 each, and the outputs so far with
// them: every weight then counts with its 11 bits, down to 2^-115 of the largest.  Peaked scores cost time so: 64 sequences of
// 4078 rows take 125 us where scores have a standard deviation of 1.5, 155 at 3, 200 at 6 and 258 at 12.
//
// Not finite.  A query row that holds a NaN or an infinity gets NaN as its scale, and so does a page with such a scale of k or v
// as its scale of k: the scores that either meets are NaN.  The maximum passes over them (it is never NaN) and the weights'
// comparisons drop them, so the denominator alone carries them to the outputs and the log-sum-exp; 0 is left to rows that
// see nothing.
//
// Loads.  Each warp fetches its own 16 rows of a tile into its own ring with asynchronous 16-byte copies, so that warps never
// wait for one another but to join their parts, and all registers go to eight warps on an SM.  (A fifth warp for the loads
// left 168 of 255 registers and the outputs of 256 columns spilled; boxes of 16 rows by TMA cost about 1100 cycles a tile to
// issue: 141 us for 64 sequences with 261000 rows, where the copies took 134; the call takes 129 to 135 now, 4.0 to 4.1 TB/s.)
//
// Work.  Tiles of 64 cached rows of every (sequence, cached head, 16 query rows) lie on one line, of which each block takes
// an equal part: lengths need not be known on the host and long ones are split by themselves.  A part of an item that
// blocks share goes to the workspace; the last block to add its part joins them in the order of the blocks, so that
// results do not depend on timing.
#pragma once

#include <cuda_fp16.h>

#include "common.cuh"
#include "kv8.cuh"

namespace reax {

constexpr int kStepTile = 64;                 // cached rows a tile: 16 for each of the four warps
constexpr int kStepRows = 16;                 // query rows x heads of an item
constexpr int kAttendStepThreads = 4 * 32;
constexpr int kStepBlocksPerSm = 2;

template <int D>
struct StepShared {
    static constexpr int kStages = D == 256 ? 2 : 4;
    uint8_t kv[kStages][4][2][16 * D];        // a warp's 16 rows of codes of k and v
    float o[2][kStepRows][D + 16];            // outputs of warps 0 and 1, and of 2 and 3 (columns in the order of step_col)
    __half q[kStepRows][D + 8];
    float q_scale[kStepRows];
    float4 meta[kStages][4];                  // of each 16 rows: scale of k, log2 and inverse of that of v, 1 if in the cache
    float stat[2][4][kStepRows];
    long long sum[4];
    int last;
};

struct StepWork {
    int* counters;                            // [blocks]
    float* stats;                             // [blocks][2][2][kStepRows]: maximum and denominator
    float* parts;                             // [blocks][2][kStepRows][D]
};

// Where a sequence's rows are, how many tiles it has, and how many items a cached head.
struct StepSeq {
    int lo, rows, len, tiles, items;
    StepSeq() = default;
    REAX_DEVI StepSeq(const Kv8Attend& a, int b) {
        int hi;
        kv8_span(a.cu, b, a.rows, &lo, &hi);
        rows = hi - lo;
        len = min(max(a.lengths[b], 0), a.capacity);
        tiles = max((len + kStepTile - 1) / kStepTile, 1);
        items = (rows * a.group + kStepRows - 1) / kStepRows;
    }
    REAX_DEVI long long units(int heads) const { return static_cast<long long>(heads) * items * tiles; }
};

// A place on the line of tiles.
struct StepCursor {
    int b, h, item, x;
    StepSeq s;
    // The next tile; false at the line's end.
    REAX_DEVI bool next(const Kv8Attend& a) {
        if (++x < s.tiles) return true;
        x = 0;
        if (++item < s.items) return true;
        item = 0;
        if (++h < a.c.heads) return true;
        h = 0;
        while (++b < a.batch) {
            s = StepSeq(a, b);
            if (s.items > 0) return true;
        }
        return false;
    }
};

// Offset of byte `x` of row `r` in a swizzled tile of 16 rows of D bytes.
template <int D>
REAX_DEVI int step_at(int r, int x) {
    if (D == 64) return r * 64 + (((x / 16) ^ ((r / 2) & 3)) * 16) + x % 16;
    return (x / 128) * (16 * 128) + r * 128 + ((((x / 16) & 7) ^ (r & 7)) * 16) + x % 16;
}

// Place of column `col` in a row of parts: pieces of 4 columns in an order that spreads a warp's pieces over the banks.
REAX_DEVI int step_col(int col) { return ((col / 4) ^ ((col / 32) & 3)) * 4 + col % 4; }

REAX_DEVI void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Two codes (as bytes b + 128 in bytes `sel` of x) as fp16: 0x64 in the high byte makes 1024 + b + 128.
template <uint32_t SEL>
REAX_DEVI uint32_t codes_half2(uint32_t x) {
    const uint32_t y = __byte_perm(x, 0x64646464u, SEL);
    const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&y), __floats2half2_rn(1152.0f, 1152.0f));
    return *reinterpret_cast<const uint32_t*>(&h);
}

REAX_DEVI float ex2f(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
REAX_DEVI float lg2f(float x) {
    float y;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Clears the counters before a step whose workspace may hold anything; the step, a dependent launch, waits for it.
__global__ void __launch_bounds__(kAttendStepThreads) kv8_clear_kernel(const StepWork work, int blocks) {
    asm volatile("griddepcontrol.launch_dependents;");
    for (int i = threadIdx.x; i < blocks; i += kAttendStepThreads) work.counters[i] = 0;
}

constexpr uint32_t kNanBits = 0x7FFFFFFFu;

// A page's scale of k, NaN where it or the page's scale of v is not finite.
REAX_DEVI float kv8_score_scale(float k_scale, float v_scale) { return __fmaf_rn(0.0f, v_scale, __fmaf_rn(0.0f, k_scale, k_scale)); }
// A row's factor from its denominator: 0 where that is (nothing seen), NaN where that is.
REAX_DEVI float kv8_inverse(float x, float den) { return den == 0.0f ? 0.0f : x / den; }
// ... and its log-sum-exp.
REAX_DEVI float kv8_lse(float reference, float den) { return den == 0.0f ? -INFINITY : 0.69314718f * (reference + log2f(den)); }

template <int D>
__global__ void __launch_bounds__(kAttendStepThreads, kStepBlocksPerSm)
    kv8_step_kernel(const __grid_constant__ Kv8Attend a, const StepWork work) {
    using Shared = StepShared<D>;
    constexpr int kStages = Shared::kStages;
    extern __shared__ uint8_t step_smem[];
    Shared& sh = *reinterpret_cast<Shared*>(step_smem + (-smem_u32(step_smem) & 1023u));
    const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
    const int heads = a.c.heads, page = a.c.page, shift = __ffs(page) - 1;

    // this block's part [u0, u1) of the line of tiles
    long long sum = 0;
    for (int b = tid; b < a.batch; b += kAttendStepThreads) sum += StepSeq(a, b).units(heads);
#pragma unroll
    for (int m = 16; m > 0; m >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, m);
    if (lane == 0) sh.sum[warp] = sum;
    __syncthreads();
    long long total = 0;
#pragma unroll
    for (int i = 0; i < kAttendStepThreads / 32; ++i) total += sh.sum[i];
    const long long each = max((total + gridDim.x - 1) / gridDim.x, 2ll);
    const long long u0 = min(each * blockIdx.x, total), u1 = min(u0 + each, total);
    if (u0 >= u1) {
        asm volatile("griddepcontrol.wait;" ::: "memory");
        return;
    }
    // the tile u0 (each warp looks for itself)
    StepCursor at_u;
    long long u = u0, start = 0;              // start: tiles of the sequences before
    for (int b0 = 0; b0 < a.batch; b0 += 32) {
        const long long n = b0 + lane < a.batch ? StepSeq(a, b0 + lane).units(heads) : 0;
        long long upto = n;
#pragma unroll
        for (int m = 1; m < 32; m <<= 1) {
            const long long t = __shfl_up_sync(0xFFFFFFFFu, upto, m);
            if (lane >= m) upto += t;
        }
        const unsigned who = __ballot_sync(0xFFFFFFFFu, start + upto > u0);
        if (who) {
            const int l = __ffs(who) - 1;
            at_u.b = b0 + l;
            start += __shfl_sync(0xFFFFFFFFu, upto - n, l);
            break;
        }
        start += __shfl_sync(0xFFFFFFFFu, upto, 31);
    }
    at_u.s = StepSeq(a, at_u.b);
    at_u.x = static_cast<int>((u0 - start) % at_u.s.tiles);
    at_u.item = static_cast<int>((u0 - start) / at_u.s.tiles % at_u.s.items);
    at_u.h = static_cast<int>((u0 - start) / at_u.s.tiles / at_u.s.items);
    // Loads of this warp's rows, kStages tiles ahead.  `ahead` is the tile to be loaded next and `id` its page (looked up one
    // load earlier); the scales of the tile loaded last arrive in registers and are put down at the next load.
    StepCursor ahead = at_u;
    long long left = u1 - u0;                 // tiles not loaded yet
    int id = -1, fill = 0, put = -1;
    float ks = 0.0f, vs = 1.0f;
    bool in = false;
    auto look_up = [&]() {
        const int row = ahead.x * kStepTile + warp * 16;
        id = row < ahead.s.len ? a.tables[static_cast<long long>(ahead.b) * a.table_ld + (row >> shift)] : -1;
    };
    auto put_down = [&]() {
        if (put >= 0 && lane == 0) {
            const float v = fmaxf(vs, 1e-30f);
            sh.meta[put][warp] = float4{kv8_score_scale(ks, vs), lg2f(v), __fdividef(1.0f, v), in ? 1.0f : 0.0f};
        }
        put = -1;
    };
    auto load = [&]() {
        put_down();
        if (left > 0) {
            in = id >= 0 && id < a.c.pages;
            ks = 0.0f, vs = 1.0f;
            if (in) {
                const long long at = static_cast<long long>(id) * heads + ahead.h;
                ks = a.c.k_scale[at];
                vs = a.c.v_scale[at];
                const long long first = ((at << shift) + ((ahead.x * kStepTile + warp * 16) & (page - 1))) * D + lane * 16;
#pragma unroll
                for (int e = 0; e < 16 * D; e += 512) {
                    const int to = step_at<D>((e + lane * 16) / D, (e + lane * 16) % D);
                    cp_async16_cg(sh.kv[fill][warp][0] + to, a.c.k + first + e);
                    cp_async16_cg(sh.kv[fill][warp][1] + to, a.c.v + first + e);
                }
            }
            put = fill;
            if (++fill == kStages) fill = 0;
            if (--left > 0 && ahead.next(a)) look_up();
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    look_up();
#pragma unroll 1
    for (int i = 0; i < kStages; ++i) load();
    asm volatile("griddepcontrol.wait;" ::: "memory");        // the counters are clear (what comes before that, comes before the inputs)
    put_down();
    __syncwarp();

    {
        // ----------------------------------------------------------------------------------------------- products
        const int g = lane / 4, q = lane % 4;
        const int perm = g ^ ((g & 1) << 2);                          // cached row of score column g: no bank conflicts
        const int v0 = 2 * q, v1 = (2 * q + 1) ^ 4;                   // cached rows behind weights 2q and 2q + 1
        int stage = 0;
        while (u < u1) {
            const StepSeq& s = at_u.s;
            const int b = at_u.b, h = at_u.h, at = at_u.item * kStepRows, from = at_u.x;
            const int to = static_cast<int>(min(static_cast<long long>(s.tiles), from + (u1 - u)));
            const long long item_start = u - from;
            // query rows -> fp16, scaled by a power of two to a largest value in [2^13, 2^14)
            __syncthreads();
#pragma unroll 1
            for (int r = warp; r < kStepRows; r += 4) {
                const bool real = at + r < s.rows * a.group;
                const __nv_bfloat16* src = a.q + static_cast<long long>(s.lo + (real ? (at + r) / a.group : 0)) * a.ldq +
                                           (h * a.group + (real ? (at + r) % a.group : 0)) * D;
                float x[D / 32], m = 0.0f;
                bool finite = true;
#pragma unroll
                for (int i = 0; i < D / 64; ++i) {
                    const uint32_t w = real ? *reinterpret_cast<const uint32_t*>(src + i * 64 + lane * 2) : 0u;
                    x[2 * i] = __uint_as_float(w << 16), x[2 * i + 1] = __uint_as_float(w & 0xFFFF0000u);
                    m = fmaxf(m, fmaxf(fabsf(x[2 * i]), fabsf(x[2 * i + 1])));
                    finite = finite && fabsf(x[2 * i]) < INFINITY && fabsf(x[2 * i + 1]) < INFINITY;
                }
                m = warp_max(m);
                finite = __all_sync(0xFFFFFFFFu, finite);
                const uint32_t e = max(__float_as_uint(m) >> 23, 14u);
                const float f = __uint_as_float((267u - e) << 23);
#pragma unroll
                for (int i = 0; i < D / 64; ++i)
                    *reinterpret_cast<__half2*>(&sh.q[r][i * 64 + lane * 2]) = __floats2half2_rn(x[2 * i] * f, x[2 * i + 1] * f);
                if (lane == 0) sh.q_scale[r] = finite ? __uint_as_float((e - 13u) << 23) * a.scale * 1.44269504f : __uint_as_float(kNanBits);
            }
            __syncthreads();
            const float qs[2] = {sh.q_scale[g], sh.q_scale[g + 8]};
            int seen[2];                      // cached rows that query rows g and g + 8 see
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int r = at + g + 8 * i;
                seen[i] = r < s.rows * a.group ? min(s.len, a.lengths[b] - s.rows + r / a.group + 1) : 0;
            }
            float o[D / 8][4], top[2] = {-INFINITY, -INFINITY}, den[2] = {};
#pragma unroll
            for (int i = 0; i < D / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
#pragma unroll 1
            for (int x = from; x < to; ++x) {
                asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");
                __syncwarp();
                const float4 meta = sh.meta[stage][warp];
                const uint8_t* kt = sh.kv[stage][warp][0];
                const uint8_t* vt = sh.kv[stage][warp][1];
                // scores of 16 query rows and this warp's 16 cached rows
                float c[2][4] = {};
#pragma unroll
                for (int ch = 0; ch < D / 64; ++ch) {
                    uint4 qa[2][2];           // rows g and g + 8: the 16 values that meet the 16 codes below
#pragma unroll
                    for (int i = 0; i < 2; ++i)
#pragma unroll
                        for (int e = 0; e < 2; ++e)
                            qa[i][e] = *reinterpret_cast<const uint4*>(&sh.q[g + 8 * i][ch * 64 + q * 16 + e * 8]);
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
                        const uint4 w = *reinterpret_cast<const uint4*>(kt + step_at<D>(t * 8 + perm, ch * 64 + q * 16));
                        const uint32_t code[4] = {w.x ^ 0x80808080u, w.y ^ 0x80808080u, w.z ^ 0x80808080u, w.w ^ 0x80808080u};
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const uint4 &lo = qa[0][k / 2], &hi = qa[1][k / 2];
                            const uint32_t fa[4] = {k % 2 ? lo.z : lo.x, k % 2 ? hi.z : hi.x, k % 2 ? lo.w : lo.y, k % 2 ? hi.w : hi.y};
                            mma16816(c[t], fa, codes_half2<0x4140>(code[k]), codes_half2<0x4342>(code[k]));
                        }
                    }
                }
                const int first = x * kStepTile + warp * 16;
                // (`top` is the maximum less 14: weights up to 2^14, so that those down to 2^-28 of the largest are normal fp16)
                float p[2][4], m[2] = {top[0], top[1]};
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int at_row = first + t * 8 + (e % 2 ? v1 : v0);
                        p[t][e] = at_row < seen[e / 2] && meta.w > 0.0f ? c[t][e] * (qs[e / 2] * meta.x) + meta.y : -INFINITY;
                        m[e / 2] = fmaxf(m[e / 2], p[t][e] - 14.0f);
                    }
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    m[i] = fmaxf(m[i], __shfl_xor_sync(0xFFFFFFFFu, m[i], 1));
                    m[i] = fmaxf(m[i], __shfl_xor_sync(0xFFFFFFFFu, m[i], 2));
                }
                if (__any_sync(0xFFFFFFFFu, m[0] > top[0] || m[1] > top[1])) {
                    const float f0 = top[0] == -INFINITY ? 0.0f : ex2f(top[0] - m[0]), f1 = top[1] == -INFINITY ? 0.0f : ex2f(top[1] - m[1]);
                    den[0] *= f0, den[1] *= f1;
#pragma unroll
                    for (int i = 0; i < D / 8; ++i) o[i][0] *= f0, o[i][1] *= f0, o[i][2] *= f1, o[i][3] *= f1;
                    top[0] = m[0], top[1] = m[1];
                }
                float add[2] = {};
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        p[t][e] = p[t][e] == -INFINITY ? 0.0f : ex2f(p[t][e] - top[e / 2]);
                        add[e / 2] += p[t][e];
                    }
                den[0] += add[0] * meta.z, den[1] += add[1] * meta.z;
                float least = 0.0f;           // the smallest weight above 0
                {
                    float y = 1.0f;
#pragma unroll
                    for (int t = 0; t < 2; ++t)
#pragma unroll
                        for (int e = 0; e < 4; ++e) y = p[t][e] > 0.0f ? fminf(y, p[t][e]) : y;
                    least = y;
                }
                float upto = INFINITY, down_to = 0x1p-14f, times = 1.0f;
#pragma unroll 1
                for (int pass = 0;; ++pass) {
                    uint32_t pa[4];
#pragma unroll
                    for (int t = 0; t < 2; ++t)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const float y0 = p[t][2 * e], y1 = p[t][2 * e + 1];
                            const __half2 y = __floats2half2_rn(y0 < upto && y0 >= down_to ? y0 * times : 0.0f,
                                                                y1 < upto && y1 >= down_to ? y1 * times : 0.0f);
                            pa[2 * t + e] = *reinterpret_cast<const uint32_t*>(&y);
                        }
                // output: lane column g of tile e stands for value W g + e (of each 8 W values)
                constexpr int W = D == 64 ? 8 : 16;
#pragma unroll
                for (int blk = 0; blk < D / (8 * W); ++blk) {
                    uint32_t w[4][W / 4];
#pragma unroll
                    for (int t = 0; t < 4; ++t) {
                        const int r = (t / 2) * 8 + (t % 2 ? v1 : v0);
                        const uint8_t* src = vt + step_at<D>(r, blk * 8 * W + g * W);
                        if constexpr (W == 16) {
                            const uint4 y = *reinterpret_cast<const uint4*>(src);
                            w[t][0] = y.x, w[t][1] = y.y, w[t][2] = y.z, w[t][3] = y.w;
                        } else {
                            const uint2 y = *reinterpret_cast<const uint2*>(src);
                            w[t][0] = y.x, w[t][1] = y.y;
                        }
                    }
#pragma unroll
                    for (int e = 0; e < W / 4; ++e) {
                        // rows 2q, 2q + 1 of bytes 0, 1 and of bytes 2, 3; then those 8 rows on
                        const uint32_t x0 = __byte_perm(w[0][e], w[1][e], 0x5140) ^ 0x80808080u, x1 = __byte_perm(w[0][e], w[1][e], 0x7362) ^ 0x80808080u;
                        const uint32_t y0 = __byte_perm(w[2][e], w[3][e], 0x5140) ^ 0x80808080u, y1 = __byte_perm(w[2][e], w[3][e], 0x7362) ^ 0x80808080u;
                        float(*d)[4] = o + blk * W + e * 4;
                        mma16816(d[0], pa, codes_half2<0x4140>(x0), codes_half2<0x4140>(y0));
                        mma16816(d[1], pa, codes_half2<0x4342>(x0), codes_half2<0x4342>(y0));
                        mma16816(d[2], pa, codes_half2<0x4140>(x1), codes_half2<0x4140>(y1));
                        mma16816(d[3], pa, codes_half2<0x4342>(x1), codes_half2<0x4342>(y1));
                    }
                }
                    const bool more = __any_sync(0xFFFFFFFFu, least < down_to) && pass < 3;
                    if (!more && pass == 0) break;
                    const float f = more ? 0x1p29f : 1.0f / times;
#pragma unroll
                    for (int i = 0; i < D / 8; ++i) o[i][0] *= f, o[i][1] *= f, o[i][2] *= f, o[i][3] *= f;
                    if (!more) break;
                    upto = down_to, down_to *= 0x1p-29f, times *= 0x1p29f;
                }
                __syncwarp();
                load();
                __syncwarp();
                if (++stage == kStages) stage = 0;
            }
            u += to - from;
            at_u.x = to - 1;
            const bool whole = to - from == s.tiles;
            const int tiles = s.tiles;
            // the four warps' parts -> one, in the warps' order
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                den[i] += __shfl_xor_sync(0xFFFFFFFFu, den[i], 1);
                den[i] += __shfl_xor_sync(0xFFFFFFFFu, den[i], 2);
                if (q == 0) sh.stat[0][warp][g + 8 * i] = top[i], sh.stat[1][warp][g + 8 * i] = den[i];
            }
            __syncthreads();
            float f[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                float m = sh.stat[0][0][g + 8 * i];
#pragma unroll
                for (int w = 1; w < 4; ++w) m = fmaxf(m, sh.stat[0][w][g + 8 * i]);
                f[i] = top[i] == -INFINITY ? 0.0f : ex2f(top[i] - m);
            }
            constexpr int W = D == 64 ? 8 : 16;
            const int live = min(kStepRows, s.rows * a.group - at);
#pragma unroll 1
            for (int w = 0; w < 2; ++w) {
                if (warp % 2 == w) {
#pragma unroll
                    for (int r = 0; r < 2; ++r)
                        if (g + 8 * r < live)
#pragma unroll
                            for (int blk = 0; blk < D / (8 * W); ++blk)
#pragma unroll
                                for (int e = 0; e < 2; ++e)
#pragma unroll
                                    for (int j = 0; j < W; j += 4) {
                                        const float(*x)[4] = o + blk * W + j;
                                        const int k = 2 * r + e;
                                        float4& y = *reinterpret_cast<float4*>(&sh.o[warp / 2][g + 8 * r][step_col(blk * 8 * W + (2 * q + e) * W + j)]);
                                        float4 z = w == 0 ? float4{} : y;
                                        z.x += x[0][k] * f[r], z.y += x[1][k] * f[r], z.z += x[2][k] * f[r], z.w += x[3][k] * f[r];
                                        y = z;
                                    }
                }
                __syncthreads();
            }
            // row r's maximum and denominator, over the warps
            auto row_stat = [&](int r, float* m, float* d) {
                *m = sh.stat[0][0][r];
#pragma unroll
                for (int w = 1; w < 4; ++w) *m = fmaxf(*m, sh.stat[0][w][r]);
                *d = 0.0f;
#pragma unroll
                for (int w = 0; w < 4; ++w)
                    *d += sh.stat[1][w][r] * (sh.stat[0][w][r] == -INFINITY ? 0.0f : ex2f(sh.stat[0][w][r] - *m));
            };
            auto write_row = [&](int r, float m, float d, const float (&y)[D / 32]) {
                const int i = (at + r) / a.group, hq = h * a.group + (at + r) % a.group;
                const long long row = static_cast<long long>(s.lo + i) * heads * a.group + hq;
                const float inv = kv8_inverse(1.0f, d);
#pragma unroll
                for (int e = 0; e < D / 64; ++e)
                    *reinterpret_cast<uint32_t*>(a.out + row * D + e * 64 + lane * 2) = bf16x2_rn(f2(y[2 * e] * inv, y[2 * e + 1] * inv));
                if (lane == 0 && a.lse) a.lse[row] = kv8_lse(m, d);
            };
            auto two_columns = [&](int r, int col) {
                const float2 x = *reinterpret_cast<const float2*>(&sh.o[0][r][step_col(col)]), y = *reinterpret_cast<const float2*>(&sh.o[1][r][step_col(col)]);
                return float2{x.x + y.x, x.y + y.y};
            };
            if (whole) {
#pragma unroll 1
                for (int r = warp; r < live; r += 4) {
                    float m, d, y[D / 32];
                    row_stat(r, &m, &d);
#pragma unroll
                    for (int e = 0; e < D / 64; ++e) {
                        const float2 z = two_columns(r, e * 64 + lane * 2);
                        y[2 * e] = z.x, y[2 * e + 1] = z.y;
                    }
                    write_row(r, m, d, y);
                }
                if (u < u1) at_u.next(a);
                continue;
            }
            // a part: into the workspace; blocks w0 .. w1 share the item, the first of them in its slot 1, the others in 0
            const int w0 = static_cast<int>(item_start / each), w1 = static_cast<int>((item_start + tiles - 1) / each);
            const int mine = static_cast<int>(blockIdx.x), part = 2 * mine + (mine == w0 ? 1 : 0);
#pragma unroll 1
            for (int r = warp; r < live; r += 4) {
                float m, d;
                row_stat(r, &m, &d);
                if (lane == 0) {
                    __stcg(&work.stats[(part * 2 + 0) * kStepRows + r], m);
                    __stcg(&work.stats[(part * 2 + 1) * kStepRows + r], d);
                }
#pragma unroll
                for (int e = 0; e < D / 64; ++e)
                    __stcg(reinterpret_cast<float2*>(work.parts + (static_cast<long long>(part) * kStepRows + r) * D + e * 64 + lane * 2),
                           two_columns(r, e * 64 + lane * 2));
            }
            __threadfence();
            __syncthreads();
            if (tid == 0) {
                const int before_me = atomicAdd(&work.counters[w0], 1);
                sh.last = before_me == w1 - w0;
                if (sh.last) work.counters[w0] = 0;
                __threadfence();
            }
            __syncthreads();
            if (sh.last) {
#pragma unroll 1
                for (int r = warp; r < live; r += 4) {
                    float m = -INFINITY, d = 0.0f, y[D / 32] = {};
                    float2 z[16][D / 64];
                    auto fetch = [&](int first) {             // 16 parts (past the end: factor 0)
#pragma unroll
                        for (int i = 0; i < 16; ++i)
#pragma unroll
                            for (int e = 0; e < D / 64; ++e) {
                                const int w = min(first + i, w1), slot = 2 * w + (w == w0);
                                z[i][e] = __ldcg(reinterpret_cast<const float2*>(
                                    work.parts + (static_cast<long long>(slot) * kStepRows + r) * D + e * 64 + lane * 2));
                            }
                    };
                    fetch(w0);
                    for (int w = w0 + lane; w <= w1; w += 32) m = fmaxf(m, __ldcg(&work.stats[(2 * w + (w == w0)) * 2 * kStepRows + r]));
                    m = warp_max(m);
                    // 32 parts at a time: a lane has the factor of one
#pragma unroll 1
                    for (int first = w0; first <= w1; first += 32) {
                        float f_lane = 0.0f, d_lane = 0.0f;
                        if (first + lane <= w1) {
                            const int slot = 2 * (first + lane) + (first + lane == w0);
                            const float mw = __ldcg(&work.stats[slot * 2 * kStepRows + r]);
                            f_lane = mw == -INFINITY ? 0.0f : ex2f(mw - m);
                            d_lane = f_lane * __ldcg(&work.stats[(slot * 2 + 1) * kStepRows + r]);
                        }
                        d += warp_sum(d_lane);
                        const int n_parts = min(32, w1 - first + 1);
#pragma unroll 1
                        for (int i0 = 0; i0 < n_parts; i0 += 16) {
#pragma unroll
                            for (int i = 0; i < 16; ++i) {
                                const float fw = __shfl_sync(0xFFFFFFFFu, f_lane, i0 + i);
#pragma unroll
                                for (int e = 0; e < D / 64; ++e) y[2 * e] += fw * z[i][e].x, y[2 * e + 1] += fw * z[i][e].y;
                            }
                            if (first + i0 + 16 <= w1) fetch(first + i0 + 16);
                        }
                    }
                    write_row(r, m, d, y);
                }
            }
            if (u < u1) at_u.next(a);
        }
    }
}

}  // namespace reax
