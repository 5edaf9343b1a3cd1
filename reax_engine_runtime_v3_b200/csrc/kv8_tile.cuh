// Attention of many query rows over the paged INT8 cache (a prompt's chunk), on tcgen05 tensor cores.
//
// A block takes 128 query rows (rows x heads that share a cached head) and goes through the cache in tiles of 64 rows with a
// running maximum and denominator.  Codes come through TMA, are turned into fp16 (k) or bf16 (v), both exact, by warps of
// their own into swizzled tiles, and serve as the B operands: K-major for the scores S = Q K^T, MN-major for O += P V.  q and P are the A
// operands, in TMEM, where O stays in float32.
//
// Precision.  q becomes fp16 times a power of two for each row (its 8 bits fit); with it k can be fp16, which takes half the
// instructions of bf16 to make from codes.  A weight is split into two bf16 numbers, hi + lo (cut, not rounded: 2^-15), whose exponents reach as far as
// float32's: a single bf16 would lose half the output's bits again, and fp16 the weights below 2^-28 of the largest.
//
// What bounds it: at 256 values a head a tile takes about 2650 cycles (1.55 us), of which the tensor cores work 2000 (128 x 64
// scores cost 1000: an MMA of N = 64 takes 60 cycles with its A operand in TMEM, and twice that with q read from shared memory
// beside the conversion's traffic, so q lives in TMEM; O costs another 1000 with both terms).  The softmax's chain from a
// tile's scores to its weights takes 2600, the codes' conversion 2500.  The roles overlap.
//
// Values that are not finite go as in the step form: a NaN as the scale of the row or of the page's scores, carried to the
// outputs by the denominator.
//
// Scaling O (in TMEM) costs as much as a tile, so the reference that the exponents are taken from moves only when a maximum
// exceeds it by 8 (in log2): weights stay below 2^8, which bf16 holds as well as any.
//
// Work.  The tiles of all items lie on one line, of which each block takes an equal part; parts of items that blocks share are
// joined by a second kernel, in the blocks' order.  2048 rows of four prompts (19676 tiles) take 267 to 292 us; a block for each item
// had left the longest for the end (510 us), and one sequence of 65536 cached rows and 16 new ones to four blocks (2305 us,
// now 73).
//
// Roles (17 warps): 0-7 softmax (thread = row and half of the columns), 8 loads, 12 MMAs of the scores, 16 those of O, the
// others codes to 16 bits.  Waiting for and issuing both sorts of MMA takes one warp 3350 cycles a tile.  The two, and the
// loads, share a scheduler with softmax warps alone.
#pragma once

#include "common.cuh"
#include "gdn_chunk.cuh"
#include "kv8.cuh"
#include "kv8_step.cuh"

namespace reax {

constexpr int kTileRows = 128, kTileCols = 64;
constexpr int kAttendTileThreads = 17 * 32;
constexpr int kConverters = 6;                // warps
constexpr uint32_t kTmO = 0, kTmQ = 256, kTmScore = 384, kTmWeight = 448;

constexpr int kTileSeqs = 256;                // sequences counted at a time

struct Kv8Maps {
    CUtensorMap k, v;                         // rows of D bytes, boxes of min(D, 128) bytes by 16 rows
};

template <int D>
struct TileShared {
    uint8_t k[2][kTileCols * D * 2], v[2][kTileCols * D * 2];   // [D / 64][64 rows][64 values], 128-byte swizzle
    uint8_t codes[2][2][kTileCols * D];       // of k and v as they come, two tiles: 16 rows after 16 rows
    float xch[2][8][32];
    long long units[kTileSeqs];               // tiles of the sequences, for one cached head
    uint64_t in[2][2], in_free[2][2], k_full[2], v_full[2], k_free[2], v_free[2], s_full, s_free, p_full, pv_done, drained[2];
    uint32_t tmem;
    uint32_t abort;
    bool more[2];                             // a tile's outputs are added to those of the item's tiles before
};

// fp32 sums of bf16 operands; b_mn: B is stored with N contiguous.
__host__ __device__ constexpr uint32_t idesc_bf16_ts(int M, int N, bool b_mn) {
    return idesc_bf16_f32(M, N) | (b_mn ? 1u << 16 : 0u);
}

// Two codes (as bytes c + 128 of x, picked by SEL into 16-bit lanes) as bf16 times 2^-6: the bits c + 128 are (c + 128) 2^-133
// there, subnormal or not, so that one multiplication by 2^127 and a subtraction give them, exactly.
constexpr float kCodeUp = 64.0f;
template <uint32_t SEL>
REAX_DEVI uint32_t codes_bf162(uint32_t x) {
    const uint32_t y = __byte_perm(x, 0u, SEL);
    uint32_t z;
    asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(z) : "r"(y), "r"(0x7F007F00u), "r"(0xC000C000u));
    return z;
}

// What the blocks leave for the join: the item that block i begins and others go on with, and the parts of both ends of each
// block's stretch (0: of an item that it goes on with, 1: of one that it begins and does not end).
struct TileRest {
    int lo, first, live, h, parts;            // parts: blocks that have one (0: no such item)
};
struct TileWork {
    TileRest* rest;                           // [blocks]
    float* stats;                             // [blocks][2][2][kTileRows]: reference and denominator
    float* sums;                              // [blocks][2][D][kTileRows]
};

struct TileSeq {
    int lo, rows, len, before, items;         // `before`: rows that its first query row sees, less one
    TileSeq() = default;
    REAX_DEVI TileSeq(const Kv8Attend& a, int b) {
        int hi;
        kv8_span(a.cu, b, a.rows, &lo, &hi);
        rows = hi - lo;
        const int all = max(a.lengths[b], 0);
        len = min(all, a.capacity);
        before = all - rows;
        items = (rows * a.group + kTileRows - 1) / kTileRows;
    }
    // Rows that see nothing take one tile too (a masked one).
    REAX_DEVI int tiles(const Kv8Attend& a, int item) const {
        const int last = min((item + 1) * kTileRows, rows * a.group) - 1;
        return max((min(len, before + last / a.group + 1) + kTileCols - 1) / kTileCols, 1);
    }
};

// A place on the line of items: of the cached heads one after the other, in each those of the sequences.  An item is as long
// as its tiles and kItemTiles more, which come first and stand for the time that it takes to begin and end one (its rows
// of q, its outputs; measured 9 us, at 256 values a head): 2048 rows of four prompts took 290 us where only tiles are counted
// and 270 with it, side by side.
constexpr int kItemTiles = 5;
struct TileCursor {
    long long end;                            // the item's on the line
    int h, b, item, x, to, tiles;             // [x, to): this block's of its tiles
    TileSeq s;
    REAX_DEVI void take(long long from, long long u1) {
        x = static_cast<int>(max(tiles - (end - from), 0ll));
        to = static_cast<int>(tiles - max(end - u1, 0ll));
    }
    // The next item of which this block has tiles.
    REAX_DEVI bool next(const Kv8Attend& a, long long u1) {
        if (end + kItemTiles >= u1) return false;
        if (++item >= s.items) {
            item = 0;
            do {
                if (++b == a.batch) b = 0, ++h;
                s = TileSeq(a, b);
            } while (s.items == 0);
        }
        tiles = s.tiles(a, item);
        end += kItemTiles + tiles;
        take(0, u1);
        x = 0;
        return true;
    }
};

REAX_DEVI long long warp_sum_ll(long long v) {
#pragma unroll
    for (int m = 16; m > 0; m >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, m);
    return v;
}
// Takes from `rest` what lies before the first lane whose running sum of `n` exceeds it, and gives that lane, or -1.
REAX_DEVI int warp_find(long long n, long long* rest, int lane) {
    long long upto = n;
#pragma unroll
    for (int m = 1; m < 32; m <<= 1) {
        const long long t = __shfl_up_sync(0xFFFFFFFFu, upto, m);
        if (lane >= m) upto += t;
    }
    const unsigned who = __ballot_sync(0xFFFFFFFFu, upto > *rest);
    const int l = who ? __ffs(who) - 1 : 31;
    *rest -= __shfl_sync(0xFFFFFFFFu, who ? upto - n : upto, l);
    return who ? l : -1;
}

template <int D>
__global__ void __launch_bounds__(kAttendTileThreads, 1)
    kv8_tile_kernel(const __grid_constant__ Kv8Attend a, const __grid_constant__ Kv8Maps maps, const TileWork work, uint32_t limit_ns) {
    extern __shared__ uint8_t tile_smem[];
    TileShared<D>& sh = *reinterpret_cast<TileShared<D>*>(tile_smem + (-smem_u32(tile_smem) & 1023u));
    const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32, quarter = warp % 4;
    const int heads = a.c.heads, page = a.c.page, shift = __ffs(page) - 1;
    asm volatile("griddepcontrol.launch_dependents;");        // (the join, which waits for the end of this grid)
    // this block's stretch [u0, u1) of the line, and what it begins with
    long long u0 = 0, u1 = 0, all = 0;
    int blocks = 0, n = 0;                                    // n: its tiles
    TileCursor start;
    {
        auto count = [&](int b0) {
            __syncthreads();
            for (int b = b0 + warp; b < min(a.batch, b0 + kTileSeqs); b += kAttendTileThreads / 32) {
                const TileSeq s(a, b);
                long long n = 0;
                for (int i = lane; i < s.items; i += 32) n += kItemTiles + s.tiles(a, i);
                n = warp_sum_ll(n);
                if (lane == 0) sh.units[b - b0] = n;
            }
            __syncthreads();
        };
        long long head = 0;
        for (int b0 = 0; b0 < a.batch; b0 += kTileSeqs) {
            count(b0);
            long long n = 0;
            for (int i = lane; i < min(a.batch - b0, kTileSeqs); i += 32) n += sh.units[i];
            head += warp_sum_ll(n);
        }
        all = head * heads;
        blocks = static_cast<int>(min(static_cast<long long>(gridDim.x), all / (kItemTiles + 1)));   // (each gets a tile)
        if (tid == 0) work.rest[blockIdx.x].parts = 0;
        if (static_cast<int>(blockIdx.x) >= blocks) return;
        u0 = all * blockIdx.x / blocks, u1 = all * (blockIdx.x + 1) / blocks;
        start.h = static_cast<int>(u0 / head);
        long long rest = u0 - start.h * head;
        int b = -1;
        for (int b0 = 0; b < 0; b0 += kTileSeqs) {
            if (a.batch > kTileSeqs) count(b0);
            for (int i = 0; i < min(a.batch - b0, kTileSeqs) && b < 0; i += 32) {
                const int l = warp_find(b0 + i + lane < a.batch && i + lane < kTileSeqs ? sh.units[i + lane] : 0, &rest, lane);
                if (l >= 0) b = b0 + i + l;
            }
        }
        start.b = b;
        start.s = TileSeq(a, b);
        int item = -1;
        for (int i = 0; item < 0; i += 32) {
            const int l = warp_find(i + lane < start.s.items ? kItemTiles + start.s.tiles(a, i + lane) : 0, &rest, lane);
            if (l >= 0) item = i + l;
        }
        start.item = item;
        start.tiles = start.s.tiles(a, item);
        start.end = u0 - rest + kItemTiles + start.tiles;
        start.take(u0, u1);
        TileCursor at = start;
        do n += at.to - at.x;
        while (at.next(a, u1));
    }

    if (warp == 12) tmem_alloc(&sh.tmem, 512);
    if (tid == 0) {
        for (int i = 0; i < 2; ++i) {
            for (int e = 0; e < 2; ++e) mbar_init(&sh.in[i][e], 1), mbar_init(&sh.in_free[i][e], kConverters);
            mbar_init(&sh.k_full[i], kConverters), mbar_init(&sh.v_full[i], kConverters);
            mbar_init(&sh.k_free[i], 1), mbar_init(&sh.v_free[i], 1);
        }
        mbar_init(&sh.s_full, 1), mbar_init(&sh.s_free, 8), mbar_init(&sh.p_full, 8), mbar_init(&sh.pv_done, 1), mbar_init(&sh.drained[0], 1), mbar_init(&sh.drained[1], 1);
        sh.abort = 0;
        fence_mbar_init();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tm = sh.tmem;
    GdnWait wait{&sh.abort, limit_ns};
    const uint32_t lanes = tm + (static_cast<uint32_t>(quarter * 32) << 16);
    auto arrive = [&](uint64_t* bar) {
        __syncwarp();
        if (lane == 0 && !wait.dead) mbar_arrive(bar);
    };

    if (warp < 8) {
        // ------------------------------------------------------------------------------------------------- softmax
        const int half = warp / 4, r = quarter * 32 + lane;
        int turn = 0;
        auto row_max = [&](float m) {
            float* x = &sh.xch[turn][quarter * 2][lane];
            x[half * 32] = m;
            named_bar_sync(1 + quarter, 64);
            turn ^= 1;
            return fmaxf(x[0], x[32]);
        };
        int t0 = 0;                           // tiles so far
#pragma unroll 1
        for (TileCursor at = start;;) {
            const TileSeq& seq = at.s;
            const int first = at.item * kTileRows, live = min(kTileRows, seq.rows * a.group - first);
            const int to = at.to;
            const int32_t* table = a.tables + static_cast<long long>(at.b) * a.table_ld;
            float scale = a.scale * 1.44269504f;
            {
                // q's row, half of it, into TMEM: two values a column, scaled to a largest in [2^13, 2^14)
                const int i = first + min(r, live - 1);
                const __nv_bfloat16* src = a.q + (static_cast<long long>(seq.lo) + i / a.group) * a.ldq + (at.h * a.group + i % a.group) * D + half * (D / 2);
                uint32_t top = 0;
                uint4 y[D / 16];
#pragma unroll
                for (int e = 0; e < D / 16; ++e) y[e] = *reinterpret_cast<const uint4*>(src + e * 8);
#pragma unroll
                for (int e = 0; e < D / 16; ++e)
                    top = __vmaxu2(__vmaxu2(top, y[e].x & 0x7FFF7FFFu), __vmaxu2(y[e].y & 0x7FFF7FFFu, __vmaxu2(y[e].z & 0x7FFF7FFFu, y[e].w & 0x7FFF7FFFu)));
                // (a NaN counts as an infinity, which the maximum keeps)
                const float most = row_max(__uint_as_float(min(max(top & 0xFFFFu, top >> 16), 0x7F80u) << 16));
                const float2 f = scale_of(most);
                scale = most < INFINITY ? scale * f.y : __uint_as_float(kNanBits);
#pragma unroll
                for (int e = 0; e < D / 16; e += 4) {
                    uint32_t w[16];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const uint4 z = y[e + j];
                        w[4 * j] = half2_of(mul2_rn(bf16x2_to_f2(z.x), f2(f.x, f.x))), w[4 * j + 1] = half2_of(mul2_rn(bf16x2_to_f2(z.y), f2(f.x, f.x)));
                        w[4 * j + 2] = half2_of(mul2_rn(bf16x2_to_f2(z.z), f2(f.x, f.x))), w[4 * j + 3] = half2_of(mul2_rn(bf16x2_to_f2(z.w), f2(f.x, f.x)));
                    }
                    tmem_st_x16(lanes + kTmQ + half * (D / 4) + e * 4, w);
                }
                tmem_wait_st();
                tc_fence_before();
                arrive(&sh.s_free);
            }
            const int seen = r < live ? min(seq.len, seq.before + (first + r) / a.group + 1) : 0;
            const int least = min(seq.len, seq.before + first / a.group + 1);     // what the first row sees
            float ref = -INFINITY, den = 0.0f;
            // scales of this half's two runs of 16 rows: pages looked up two tiles ahead, scales fetched one ahead
            int id[2];
            float ks[2], vs[2];
            bool in[2];
            auto look_up = [&](int x) {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int row = x * kTileCols + half * 32 + e * 16;
                    id[e] = x < to && row < seq.len ? table[row >> shift] : -1;
                }
            };
            auto fetch = [&]() {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    in[e] = id[e] >= 0 && id[e] < a.c.pages;
                    const long long scales = static_cast<long long>(in[e] ? id[e] : 0) * heads + at.h;
                    ks[e] = in[e] ? a.c.k_scale[scales] : 0.0f;
                    vs[e] = in[e] ? a.c.v_scale[scales] : 1.0f;
                }
            };
            look_up(at.x);
            fetch();
            look_up(at.x + 1);
#pragma unroll 1
            for (int x = at.x; x < to; ++x, ++t0) {
                const float v[2] = {fmaxf(vs[0], 1e-30f), fmaxf(vs[1], 1e-30f)}, inv[2] = {__fdividef(1.0f, v[0]), __fdividef(1.0f, v[1])};
                const float f[2] = {kv8_score_scale(ks[0], vs[0]) * scale, kv8_score_scale(ks[1], vs[1]) * scale}, add[2] = {lg2f(v[0]), lg2f(v[1])};
                const bool plain = in[0] && in[1] && x * kTileCols + half * 32 + 32 <= least;
                const bool have[2] = {in[0], in[1]};
                fetch();
                look_up(x + 2);
                wait(&sh.s_full, t0 & 1, kStatusTimeoutAccFull);
                tc_fence_after();
                uint32_t c[32];
                tmem_ld_x32_sync(lanes + kTmScore + half * 32, c);
                tc_fence_before();
                if (x + 1 < to) arrive(&sh.s_free);
                uint64_t t[16];
                float m = -INFINITY;
#pragma unroll
                for (int i = 0; i < 16; ++i) t[i] = fma2_rn(u2(c[2 * i], c[2 * i + 1]), f2(f[i / 8], f[i / 8]), f2(add[i / 8], add[i / 8]));
                if (!plain) {
                    const int col = x * kTileCols + half * 32;
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        t[i] = f2(col + 2 * i < seen && have[i / 8] ? f2_lo(t[i]) : -INFINITY, col + 2 * i + 1 < seen && have[i / 8] ? f2_hi(t[i]) : -INFINITY);
                }
#pragma unroll
                for (int i = 0; i < 16; ++i) m = fmaxf(m, fmaxf(f2_lo(t[i]), f2_hi(t[i])));
                m = row_max(m);
                // a new reference where the maximum is well above the old one; O is scaled then
                const bool move = m > ref + 8.0f;           // (true from -inf)
                if (__any_sync(0xFFFFFFFFu, move)) {
                    const float to = move ? m : ref, g = ref == -INFINITY ? 0.0f : ex2(ref - to);
                    if (x > at.x) {
                        wait(&sh.pv_done, (t0 - 1) & 1, kStatusTimeoutAccFull);
                        tc_fence_after();
#pragma unroll 1
                        for (int e = half * (D / 2); e < (half + 1) * (D / 2); e += 16) {
                            uint32_t o[16];
                            tmem_ld_x16_sync(lanes + kTmO + e, o);
#pragma unroll
                            for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * g);
                            tmem_st_x16(lanes + kTmO + e, o);
                        }
                        tmem_wait_st();
                    }
                    den *= g;
                    ref = to;
                }
                const float base = ref == -INFINITY ? 0.0f : ref;
                uint64_t sum[2] = {};
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const uint64_t y = sub2_rn(t[i], f2(base, base));
                    t[i] = f2(ex2(f2_lo(y)), ex2(f2_hi(y)));
                    sum[i / 8] = add2_rn(sum[i / 8], t[i]);
                }
                den += (f2_lo(sum[0]) + f2_hi(sum[0])) * inv[0] + (f2_lo(sum[1]) + f2_hi(sum[1])) * inv[1];
                // P's place is free once O has taken the tile before
                if (x > at.x) wait(&sh.pv_done, (t0 - 1) & 1, kStatusTimeoutAccFull);
                tc_fence_after();
#pragma unroll
                for (int e = 0; e < 32; e += 16) {
                    uint32_t hi[8], lo[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        // upper halves, and upper halves of what they leave
                        const uint32_t y0 = static_cast<uint32_t>(t[e / 2 + i]), y1 = static_cast<uint32_t>(t[e / 2 + i] >> 32);
                        hi[i] = __byte_perm(y0, y1, 0x7632);
                        const uint64_t rest = sub2_rn(t[e / 2 + i], u2(y0 & 0xFFFF0000u, y1 & 0xFFFF0000u));
                        lo[i] = __byte_perm(static_cast<uint32_t>(rest), static_cast<uint32_t>(rest >> 32), 0x7632);
                    }
                    tmem_st_x8(lanes + kTmWeight + half * 16 + e / 2, hi);
                    tmem_st_x8(lanes + kTmWeight + 32 + half * 16 + e / 2, lo);
                }
                tmem_wait_st();
                tc_fence_before();
                if (tid == 0) sh.more[t0 & 1] = x > at.x;
                arrive(&sh.p_full);
            }
            // out
            sh.xch[turn][quarter * 2 + half][lane] = den;
            named_bar_sync(1 + quarter, 64);
            den = sh.xch[turn][quarter * 2][lane] + sh.xch[turn][quarter * 2 + 1][lane];
            turn ^= 1;
            wait(&sh.pv_done, (t0 - 1) & 1, kStatusTimeoutAccFull);
            tc_fence_after();
            if (at.x > 0 || to < at.tiles) {
                // a part: columns of 128 rows
                const long long place = 2 * static_cast<long long>(blockIdx.x) + (at.x == 0);
                float* sums = work.sums + place * D * kTileRows + r;
#pragma unroll 2
                for (int e = half * (D / 2); e < (half + 1) * (D / 2); e += 32) {
                    uint32_t o[32];
                    tmem_ld_x32_sync(lanes + kTmO + e, o);
#pragma unroll
                    for (int j = 0; j < 32; ++j) sums[(e + j) * kTileRows] = __uint_as_float(o[j]);
                }
                if (half == 0) work.stats[place * 2 * kTileRows + r] = ref, work.stats[(place * 2 + 1) * kTileRows + r] = den;
                if (tid == 0 && at.x == 0) {
                    // the last block that has a part of it
                    work.rest[blockIdx.x] = {seq.lo, first, live, at.h, static_cast<int>((at.end * blocks - 1) / all) - static_cast<int>(blockIdx.x) + 1};
                }
            } else {
                const float scale_out = kv8_inverse(kCodeUp, den);
                const int i = first + r;
                const long long row = (static_cast<long long>(seq.lo) + i / a.group) * heads * a.group + at.h * a.group + i % a.group;
#pragma unroll 2
                for (int e = half * (D / 2); e < (half + 1) * (D / 2); e += 16) {
                    uint32_t o[16], w[8];
                    tmem_ld_x16_sync(lanes + kTmO + e, o);
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        w[j] = bf16x2_rn(f2(__uint_as_float(o[2 * j]) * scale_out, __uint_as_float(o[2 * j + 1]) * scale_out));
                    if (r < live) {
                        *reinterpret_cast<uint4*>(a.out + row * D + e) = uint4{w[0], w[1], w[2], w[3]};
                        *reinterpret_cast<uint4*>(a.out + row * D + e + 8) = uint4{w[4], w[5], w[6], w[7]};
                    }
                }
                if (a.lse && half == 0 && r < live) a.lse[row] = kv8_lse(ref, den);
            }
            if (!at.next(a, u1)) break;
        }
    } else if (warp == 12) {
        // ---------------------------------------------------------------------------------------- MMAs of the scores
        if (lane == 0) {
            constexpr uint32_t id_s = idesc_f16_f32(128, kTileCols, false);
#pragma unroll 1
            for (int t = 0; t < n; ++t) {
                const int buf = t & 1;
                const uint64_t kd = sw128_kmajor_desc(smem_u32(sh.k[buf]));
                wait(&sh.k_full[buf], (t >> 1) & 1, kStatusTimeoutFull);
                wait(&sh.s_free, t & 1, kStatusTimeoutAccEmpty);       // (an item's first: q is there)
                if (wait.dead) break;
                tc_fence_after();
#pragma unroll
                for (int ks = 0; ks < D / 16; ++ks)
                    umma_f16_ts(tm + kTmScore, tm + kTmQ + ks * 8, kd + (ks / 4) * (kTileCols * 8) + (ks % 4) * 2, id_s, ks > 0);
                umma_commit(&sh.s_full);
                umma_commit(&sh.k_free[buf]);
            }
            drain_mmas(&sh.drained[0]);
        }
        __syncwarp();
    } else if (warp == 16) {
        // ----------------------------------------------------------------------------------------------- MMAs of O
        if (lane == 0) {
            constexpr uint32_t id_o = idesc_bf16_ts(128, D, true);
#pragma unroll 1
            for (int t = 0; t < n; ++t) {
                const int buf = t & 1;
                const uint64_t vd = sw128_mn_desc(smem_u32(sh.v[buf]), kTileCols * 128);
                wait(&sh.v_full[buf], (t >> 1) & 1, kStatusTimeoutFull);
                wait(&sh.p_full, t & 1, kStatusTimeoutEmpty);
                if (wait.dead) break;
                tc_fence_after();
                const bool more = sh.more[buf];
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    umma_f16_ts(tm + kTmO, tm + kTmWeight + (e / 4) * 32 + (e % 4) * 8, vd + (e % 4) * 128, id_o, more || e > 0);
                umma_commit(&sh.pv_done);
                umma_commit(&sh.v_free[buf]);
            }
            drain_mmas(&sh.drained[1]);
        }
        __syncwarp();
    } else if (warp == 8) {
        // --------------------------------------------------------------------------------------------------- loads
        const uint64_t policy = l2_policy_evict_normal();
        int id = -1, loads[2] = {};
        TileCursor at = start;
        auto look_up = [&]() {                // lane l < 4: rows 16 l .. of the tile
            const int row = at.x * kTileCols + lane * 16;
            id = lane < 4 && row < at.s.len ? a.tables[static_cast<long long>(at.b) * a.table_ld + (row >> shift)] : -1;
        };
        look_up();
#pragma unroll 1
        for (int t = 0; t < n; ++t) {
            const bool in = id >= 0 && id < a.c.pages;
            const int from = (id * heads + at.h) * page + ((at.x * kTileCols + lane * 16) & (page - 1)), buf = t & 1;
            const uint32_t have = __popc(__ballot_sync(0xFFFFFFFFu, in));
#pragma unroll 1
            for (int e = 0; e < 2; ++e) {     // k, then v
                if (t > 1) wait(&sh.in_free[buf][e], ((t >> 1) - 1) & 1, kStatusTimeoutEmpty);
                wait.dead = __any_sync(0xFFFFFFFFu, wait.dead);
                if (lane == 0 && !wait.dead) {
                    fence_proxy_async_smem();
                    mbar_arrive_expect_tx(&sh.in[buf][e], have * 16 * D);
                }
                __syncwarp();
                loads[e] += !wait.dead;
                if (in && !wait.dead)
#pragma unroll
                    for (int d = 0; d < D; d += 128)
                        tma_load_2d(sh.codes[buf][e] + lane * 16 * D + d * 16, e ? &maps.v : &maps.k, &sh.in[buf][e], d, from, policy);
                __syncwarp();
            }
            if (t + 1 < n) {
                if (++at.x == at.to) at.next(a, u1);
                look_up();
            }
        }
        // no copy may be in flight when the block ends
        if (lane == 0)
            for (int e = 0; e < 2; ++e)
                for (int x = max(loads[e] - 2, 0); x < loads[e]; ++x) mbar_wait_bounded(&sh.in[x & 1][e], (x >> 1) & 1, kDrainNs, nullptr);
        __syncwarp();
    } else {
        // ------------------------------------------------------------------------------------------- codes to bf16
        const int begin = warp < 12 ? warp - 9 : warp - 10;
        constexpr int step = kConverters;
        // this lane's place in 8 rows of 64 codes as they come, and in the tile
        const int from = D == 64 ? step_at<64>(lane % 8, lane / 8 * 16) : (lane % 8) * 128 + ((lane / 8) ^ (lane % 8)) * 16;
        const int into = (lane % 8) * 128 + ((lane / 8 * 2) ^ (lane % 8)) * 16;
#pragma unroll 1
        for (int t = 0; t < n; ++t) {
            const int buf = t & 1;
#pragma unroll 1
            for (int e = 0; e < 2; ++e) {
                wait(&sh.in[buf][e], (t >> 1) & 1, kStatusTimeoutFull);
                // K's place is free once the scores of the tile before last are there, V's once O has taken it
                if (t > 1) wait(e ? &sh.v_free[buf] : &sh.k_free[buf], ((t >> 1) - 1) & 1, kStatusTimeoutEmpty);
                uint8_t* to = e ? sh.v[buf] : sh.k[buf];
                // 8 rows by 4 pieces of 16 codes a warp and turn
                auto convert = [&](auto pair) {
                    // (the loads first: the compiler must not move one over a store that it cannot tell apart)
                    constexpr int kAll = (kTileCols / 8) * (D / 64), kEach = (kAll + step - 1) / step;
                    {
                        uint4 y[kEach];
#pragma unroll
                        for (int n = 0; n < kEach; ++n) {
                            const int u = min(begin + n * step, kAll - 1), rb = u / (D / 64), pb = u % (D / 64);
                            y[n] = *reinterpret_cast<const uint4*>(
                                D == 64 ? sh.codes[buf][e] + rb * 512 + from
                                        : sh.codes[buf][e] + (rb / 2) * (16 * D) + (rb % 2) * 1024 + (pb / 2) * 2048 + (from ^ (pb % 2 * 64)));
                        }
#pragma unroll
                        for (int n = 0; n < kEach; ++n) {
                            const int u = begin + n * step, rb = u / (D / 64), pb = u % (D / 64);
                            if (u >= kAll) break;
                            uint8_t* row = to + pb * (kTileCols * 128) + rb * 1024;
                            uint32_t w[8];
                            pair(y[n].x, w[0], w[1]), pair(y[n].y, w[2], w[3]), pair(y[n].z, w[4], w[5]), pair(y[n].w, w[6], w[7]);
                            *reinterpret_cast<uint4*>(row + into) = uint4{w[0], w[1], w[2], w[3]};
                            *reinterpret_cast<uint4*>(row + (into ^ 16)) = uint4{w[4], w[5], w[6], w[7]};
                        }
                    }
                };
                if (e)
                    convert([](uint32_t x, uint32_t& lo, uint32_t& hi) {
                        lo = codes_bf162<0x4140>(x ^ 0x80808080u), hi = codes_bf162<0x4342>(x ^ 0x80808080u);
                    });
                else
                    convert([](uint32_t x, uint32_t& lo, uint32_t& hi) {
                        lo = codes_half2<0x4140>(x ^ 0x80808080u), hi = codes_half2<0x4342>(x ^ 0x80808080u);
                    });
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0 && !wait.dead) {
                    mbar_arrive(&sh.in_free[buf][e]);
                    mbar_arrive(e ? &sh.v_full[buf] : &sh.k_full[buf]);
                }
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (tid == 0 && sh.abort) atomicOr(&g_mixer_status, sh.abort);
    if (warp == 12) {
        tmem_relinquish();
        tmem_dealloc(tm, 512);
    }
}

// The join of items that blocks share.  A unit of it is 32 rows of some columns; 2, 4 or 8 warps (by the number of parts, so
// that neither a few long items nor many short ones leave warps without work) take the parts in turn for 16 columns, and
// their sums are added in the warps' order.
constexpr int kJoinThreads = 8 * 32, kJoinBlocksPerSm = 4, kJoinCols = 16, kMostTileBlocks = 256;
template <int D>
__global__ void __launch_bounds__(kJoinThreads) kv8_join_kernel(const __grid_constant__ Kv8Attend a, const TileWork work, int blocks) {
    __shared__ int upto[kMostTileBlocks];                     // units of the blocks' items, added up
    __shared__ float xch[8][2 + kJoinCols][32];
    const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
    auto ways_of = [](int parts) { return parts > 4 ? 8 : parts > 2 ? 4 : 2; };
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (warp == 0) {
        int before = 0;
        for (int i = lane; i - lane < blocks; i += 32) {
            const int parts = i < blocks ? work.rest[i].parts : 0;
            int n = parts ? (work.rest[i].live + 31) / 32 * (D / kJoinCols / (8 / ways_of(parts))) : 0;
#pragma unroll
            for (int m = 1; m < 32; m <<= 1) {
                const int t = __shfl_up_sync(0xFFFFFFFFu, n, m);
                if (lane >= m) n += t;
            }
            if (i < blocks) upto[i] = before + n;
            before += __shfl_sync(0xFFFFFFFFu, n, 31);
        }
    }
    __syncthreads();
    const int units = upto[blocks - 1];
#pragma unroll 1
    for (int u = blockIdx.x; u < units; u += gridDim.x) {
        int i = 0;                                            // the first with upto[i] > u
#pragma unroll
        for (int m = kMostTileBlocks / 2; m > 0; m >>= 1)
            if (i + m <= blocks && upto[i + m - 1] <= u) i += m;
        const TileRest rest = work.rest[i];
        const int ways = ways_of(rest.parts), across = D / kJoinCols / (8 / ways), slice = warp % ways;
        const int unit = u - (i ? upto[i - 1] : 0), r = unit / across * 32 + lane;
        const int col = (unit % across * (8 / ways) + warp / ways) * kJoinCols;
        float top = -INFINITY, den = 0.0f, o[kJoinCols] = {};
#pragma unroll 2
        for (int p = slice; p < rest.parts; p += ways) {
            const long long place = 2 * (static_cast<long long>(i) + p) + (p == 0);
            const float ref = work.stats[place * 2 * kTileRows + r], d = work.stats[(place * 2 + 1) * kTileRows + r];
            float y[kJoinCols];
#pragma unroll
            for (int e = 0; e < kJoinCols; ++e) y[e] = work.sums[(place * D + col + e) * kTileRows + r];
            const float m = fmaxf(top, ref), base = m == -INFINITY ? 0.0f : m, f0 = ex2f(top - base), f1 = ex2f(ref - base);
            top = m;
            den = den * f0 + d * f1;
#pragma unroll
            for (int e = 0; e < kJoinCols; ++e) o[e] = o[e] * f0 + y[e] * f1;
        }
        __syncthreads();                                      // the unit before has been read
        xch[warp][0][lane] = top, xch[warp][1][lane] = den;
#pragma unroll
        for (int e = 0; e < kJoinCols; ++e) xch[warp][2 + e][lane] = o[e];
        __syncthreads();
        if (slice > 0 || r >= rest.live) continue;
        for (int w = 1; w < ways; ++w) {
            const float ref = xch[warp + w][0][lane], m = fmaxf(top, ref), base = m == -INFINITY ? 0.0f : m;
            const float f0 = ex2f(top - base), f1 = ex2f(ref - base);
            top = m;
            den = den * f0 + xch[warp + w][1][lane] * f1;
#pragma unroll
            for (int e = 0; e < kJoinCols; ++e) o[e] = o[e] * f0 + xch[warp + w][2 + e][lane] * f1;
        }
        const float scale = kv8_inverse(kCodeUp, den);
        const int y = rest.first + r;
        const long long row = (static_cast<long long>(rest.lo) + y / a.group) * a.c.heads * a.group + rest.h * a.group + y % a.group;
        uint32_t w[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e] = bf16x2_rn(f2(o[2 * e] * scale, o[2 * e + 1] * scale));
        *reinterpret_cast<uint4*>(a.out + row * D + col) = uint4{w[0], w[1], w[2], w[3]};
        *reinterpret_cast<uint4*>(a.out + row * D + col + 8) = uint4{w[4], w[5], w[6], w[7]};
        if (a.lse && col == 0) a.lse[row] = kv8_lse(top, den);
    }
}

}  // namespace reax
