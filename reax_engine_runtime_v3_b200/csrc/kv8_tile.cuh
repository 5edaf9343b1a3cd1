// Attention of many query rows over the paged INT8 cache (a prompt's chunk), on tcgen05 tensor cores.
//
// A block takes 128 query rows (rows x heads that share a cached head) and goes through the cache in tiles of 64 rows with a
// running maximum and denominator.  Codes come through TMA, are turned into bf16 (exact) by warps of their own into
// swizzled tiles, and serve as the B operands: K-major for the scores S = Q K^T, MN-major for O += P V.  S and P alternate
// between two places in TMEM, where O stays in float32.
//
// Precision.  q is bf16 as it comes.  A weight is split into two bf16 numbers, hi + lo (2^-17), whose exponents reach as far as
// float32's: a single bf16 would lose half the output's bits again, and fp16 the weights below 2^-28 of the largest.
//
// What bounds it: 64 x 128 scores cost 1024 tensor cycles at 256 values a head (N = 64 runs at half rate), O 1024 with
// both terms, and the softmax, the split and the codes' conversion about as much on the other pipes; the roles overlap.
//
// Scaling O (in TMEM) costs as much as a tile, so the reference that the exponents are taken from moves only when a maximum
// exceeds it by 8 (in log2): weights stay below 2^8, which bf16 holds as well as any.
//
// Roles (16 warps): 0-7 softmax (thread = row and half of the columns), 8-11 and 14-15 codes to bf16, 12 MMAs, 13 loads.
#pragma once

#include "common.cuh"
#include "gdn_chunk.cuh"
#include "kv8.cuh"
#include "kv8_step.cuh"

namespace reax {

constexpr int kTileRows = 128, kTileCols = 64;
constexpr int kAttendTileThreads = 16 * 32;
constexpr int kConverters = 6;                // warps
constexpr uint32_t kTmO = 0, kTmScore = 256, kTmWeight = 384;

template <int D>
struct TileShared {
    uint8_t q[kTileRows * D * 2];             // [D / 64][128 rows][64 values], 128-byte swizzle
    uint8_t k[2][kTileCols * D * 2], v[2][kTileCols * D * 2];
    uint8_t codes[2][kTileCols * D];          // of k and v as they come: 16 rows after 16 rows
    float xch[2][8][32];
    uint64_t in[2], in_free[2], k_full[2], v_full[2], s_full[2], s_free[2], p_full[2], pv_done[2];
    uint32_t tmem;
    uint32_t abort;
};

// fp32 sums of bf16 operands; b_mn: B is stored with N contiguous.
__host__ __device__ constexpr uint32_t idesc_bf16_ts(int M, int N, bool b_mn) {
    return idesc_bf16_f32(M, N) | (b_mn ? 1u << 16 : 0u);
}

// Two codes (bytes of x picked by SEL into 16-bit lanes) as bf16: 128 + (c & 127) less 128 or 256.
template <uint32_t SEL>
REAX_DEVI uint32_t codes_bf162(uint32_t x) {
    const uint32_t y = __byte_perm(x, 0u, SEL);
    const uint32_t a = (y & 0x007F007Fu) | 0x43004300u, b = (y & 0x00800080u) | 0x43004300u;
    const __nv_bfloat162 h = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
    return *reinterpret_cast<const uint32_t*>(&h);
}

template <int D>
__global__ void __launch_bounds__(kAttendTileThreads, 1)
    kv8_tile_kernel(const __grid_constant__ Kv8Attend a, const __grid_constant__ Kv8Maps maps, uint32_t limit_ns) {
    // The array starts on a swizzle atom (256 columns leave no room to round its address up); checked all the same.
    extern __shared__ __align__(1024) uint8_t tile_smem[];
    TileShared<D>& sh = *reinterpret_cast<TileShared<D>*>(tile_smem);
    if (smem_u32(tile_smem) & 1023u) {
        if (threadIdx.x == 0) atomicOr(&g_mixer_status, static_cast<unsigned>(kStatusPlanLimit));
        return;
    }
    const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32, quarter = warp % 4;
    const int heads = a.c.heads, page = a.c.page, h = blockIdx.y;
    // the sequence and the 128 rows of block x: items of the sequences one after the other
    int b = -1, item = 0;
    for (int b0 = 0, before = 0; b0 < a.batch; b0 += 32) {
        int n = 0;
        if (b0 + lane < a.batch) {
            int lo, hi;
            kv8_span(a.cu, b0 + lane, a.rows, &lo, &hi);
            n = ((hi - lo) * a.group + kTileRows - 1) / kTileRows;
        }
        int upto = n;
#pragma unroll
        for (int m = 1; m < 32; m <<= 1) {
            const int t = __shfl_up_sync(0xFFFFFFFFu, upto, m);
            if (lane >= m) upto += t;
        }
        const unsigned who = __ballot_sync(0xFFFFFFFFu, before + upto > static_cast<int>(blockIdx.x));
        if (who) {
            const int l = __ffs(who) - 1;
            b = b0 + l;
            item = static_cast<int>(blockIdx.x) - before - __shfl_sync(0xFFFFFFFFu, upto - n, l);
            break;
        }
        before += __shfl_sync(0xFFFFFFFFu, upto, 31);
    }
    if (b < 0) return;
    const StepSeq seq(a, b);
    const int first = item * kTileRows, live = min(kTileRows, seq.rows * a.group - first);
    // the last row sees the most
    const int most = min(seq.len, a.lengths[b] - seq.rows + (first + live - 1) / a.group + 1);
    const int tiles = most > 0 ? (most + kTileCols - 1) / kTileCols : 0;
    const int32_t* table = a.tables + static_cast<long long>(b) * a.table_ld;
    if (tiles == 0) {                         // rows that see nothing
        for (int e = tid; e < live * (D / 8); e += kAttendTileThreads) {
            const int r = first + e / (D / 8);
            const long long row = (static_cast<long long>(seq.lo) + r / a.group) * heads * a.group + h * a.group + r % a.group;
            *reinterpret_cast<uint4*>(a.out + row * D + e % (D / 8) * 8) = uint4{};
            if (a.lse && e % (D / 8) == 0) a.lse[row] = -INFINITY;
        }
        return;
    }

    if (warp == 12) tmem_alloc(&sh.tmem, 512);
    if (tid == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(&sh.in[i], 1), mbar_init(&sh.in_free[i], kConverters);
            mbar_init(&sh.k_full[i], kConverters), mbar_init(&sh.v_full[i], kConverters);
            mbar_init(&sh.s_full[i], 1), mbar_init(&sh.s_free[i], 8), mbar_init(&sh.p_full[i], 8), mbar_init(&sh.pv_done[i], 1);
        }
        sh.abort = 0;
        fence_mbar_init();
    }
    // q
    for (int e = tid; e < kTileRows * (D / 8); e += kAttendTileThreads) {
        const int r = e / (D / 8), x = e % (D / 8), i = first + r;
        uint4 w = {};
        if (r < live) w = *reinterpret_cast<const uint4*>(a.q + (static_cast<long long>(seq.lo) + i / a.group) * a.ldq +
                                                        (h * a.group + i % a.group) * D + x * 8);
        *reinterpret_cast<uint4*>(sh.q + (x / 8) * (kTileRows * 128) + r * 128 + ((x % 8) ^ (r % 8)) * 16) = w;
    }
    fence_proxy_async_smem();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tm = sh.tmem;
    const GdnWait wait{&sh.abort, limit_ns};
    const uint32_t lanes = tm + (static_cast<uint32_t>(quarter * 32) << 16);
    auto arrive = [&](uint64_t* bar) {
        __syncwarp();
        if (lane == 0) mbar_arrive(bar);
    };

    if (warp < 8) {
        // ------------------------------------------------------------------------------------------------- softmax
        const int half = warp / 4, r = quarter * 32 + lane;
        const int seen = r < live ? min(seq.len, a.lengths[b] - seq.rows + (first + r) / a.group + 1) : 0;
        const int least = min(seq.len, a.lengths[b] - seq.rows + first / a.group + 1);     // what the first row sees
        const float scale = a.scale * 1.44269504f;
        float ref = -INFINITY, den = 0.0f;
        int turn = 0;
        auto row_max = [&](float m) {
            float* x = &sh.xch[turn][quarter * 2][lane];
            x[half * 32] = m;
            named_bar_sync(1 + quarter, 64);
            turn ^= 1;
            return fmaxf(x[0], x[32]);
        };
        // scales of this half's two runs of 16 rows: pages looked up two tiles ahead, scales fetched one ahead
        int id[2];
        float ks[2], vs[2];
        bool in[2];
        auto look_up = [&](int x) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int row = x * kTileCols + half * 32 + e * 16;
                id[e] = x < tiles && row < seq.len ? table[row / page] : -1;
            }
        };
        auto fetch = [&]() {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                in[e] = id[e] >= 0 && id[e] < a.c.pages;
                const long long at = static_cast<long long>(in[e] ? id[e] : 0) * heads + h;
                ks[e] = in[e] ? a.c.k_scale[at] : 0.0f;
                vs[e] = in[e] ? fmaxf(a.c.v_scale[at], 1e-30f) : 1.0f;
            }
        };
        look_up(0);
        fetch();
        look_up(1);
#pragma unroll 1
        for (int x = 0; x < tiles; ++x) {
            const int buf = x & 1;
            const uint32_t par = (x >> 1) & 1;
            const float f[2] = {ks[0] * scale, ks[1] * scale}, inv[2] = {1.0f / vs[0], 1.0f / vs[1]}, add[2] = {lg2f(vs[0]), lg2f(vs[1])};
            const bool plain = in[0] && in[1] && x * kTileCols + half * 32 + 32 <= least;
            const bool have[2] = {in[0], in[1]};
            fetch();
            look_up(x + 2);
            wait(&sh.s_full[buf], par, kStatusTimeoutAccFull);
            tc_fence_after();
            uint32_t c[32];
            tmem_ld_x32_sync(lanes + kTmScore + buf * kTileCols + half * 32, c);
            tc_fence_before();
            arrive(&sh.s_free[buf]);
            float t[32], m = -INFINITY;
#pragma unroll
            for (int i = 0; i < 32; ++i) t[i] = fmaf(__uint_as_float(c[i]), f[i / 16], add[i / 16]);
            if (!plain) {
                const int col = x * kTileCols + half * 32;
#pragma unroll
                for (int i = 0; i < 32; ++i) t[i] = col + i < seen && have[i / 16] ? t[i] : -INFINITY;
            }
#pragma unroll
            for (int i = 0; i < 32; i += 2) m = fmaxf(m, fmaxf(t[i], t[i + 1]));
            m = row_max(m);
            // a new reference where the maximum is well above the old one; O is scaled then
            const bool move = m > ref + 8.0f;           // (true from -inf)
            if (__any_sync(0xFFFFFFFFu, move)) {
                const float to = move ? m : ref, g = ref == -INFINITY ? 0.0f : ex2(ref - to);
                if (x > 0) {
                    wait(&sh.pv_done[buf ^ 1], ((x - 1) >> 1) & 1, kStatusTimeoutAccFull);
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
            float sum[2] = {};
#pragma unroll
            for (int i = 0; i < 32; ++i) {
                t[i] = ex2(t[i] - base);
                sum[i / 16] += t[i];
            }
            den += sum[0] * inv[0] + sum[1] * inv[1];
            // P's place is free once O has taken the tile before last
            if (x > 1) wait(&sh.pv_done[buf], ((x >> 1) - 1) & 1, kStatusTimeoutAccFull);
            tc_fence_after();
#pragma unroll
            for (int e = 0; e < 32; e += 16) {
                uint32_t hi[8], lo[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const uint64_t y = f2(t[e + 2 * i], t[e + 2 * i + 1]);
                    hi[i] = bf16x2_rn(y);
                    lo[i] = bf16x2_rn(sub2_rn(y, bf16x2_to_f2(hi[i])));
                }
                tmem_st_x8(lanes + kTmWeight + buf * 64 + half * 16 + e / 2, hi);
                tmem_st_x8(lanes + kTmWeight + buf * 64 + 32 + half * 16 + e / 2, lo);
            }
            tmem_wait_st();
            tc_fence_before();
            arrive(&sh.p_full[buf]);
        }
        // out
        sh.xch[turn][quarter * 2 + half][lane] = den;
        named_bar_sync(1 + quarter, 64);
        den = sh.xch[turn][quarter * 2][lane] + sh.xch[turn][quarter * 2 + 1][lane];
        wait(&sh.pv_done[(tiles - 1) & 1], ((tiles - 1) >> 1) & 1, kStatusTimeoutAccFull);
        tc_fence_after();
        const float scale_out = den > 0.0f ? 1.0f / den : 0.0f;
        const int i = first + r;
        const long long row = (static_cast<long long>(seq.lo) + i / a.group) * heads * a.group + h * a.group + i % a.group;
#pragma unroll 1
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
        if (a.lse && half == 0 && r < live) a.lse[row] = den > 0.0f ? 0.69314718f * (ref + log2f(den)) : -INFINITY;
    } else if (warp == 12) {
        // ---------------------------------------------------------------------------------------------------- MMAs
        if (lane == 0) {
            constexpr uint32_t id_s = idesc_bf16_ts(128, kTileCols, false), id_o = idesc_bf16_ts(128, D, true);
            const uint64_t qd = sw128_kmajor_desc(smem_u32(sh.q));
#pragma unroll 1
            for (int x = 0; x <= tiles; ++x) {
                if (x < tiles) {
                    const int buf = x & 1;
                    const uint64_t kd = sw128_kmajor_desc(smem_u32(sh.k[buf]));
                    wait(&sh.k_full[buf], (x >> 1) & 1, kStatusTimeoutFull);
                    if (x > 1) wait(&sh.s_free[buf], ((x >> 1) - 1) & 1, kStatusTimeoutAccEmpty);
                    tc_fence_after();
#pragma unroll 1
                    for (int ks = 0; ks < D / 16; ++ks)
                        umma_f16(tm + kTmScore + buf * kTileCols, qd + (ks / 4) * (kTileRows * 8) + (ks % 4) * 2,
                                 kd + (ks / 4) * (kTileCols * 8) + (ks % 4) * 2, id_s, ks > 0);
                    umma_commit(&sh.s_full[buf]);
                }
                if (x > 0) {
                    const int y = x - 1, buf = y & 1;
                    const uint64_t vd = sw128_mn_desc(smem_u32(sh.v[buf]), kTileCols * 128);
                    wait(&sh.v_full[buf], (y >> 1) & 1, kStatusTimeoutFull);
                    wait(&sh.p_full[buf], (y >> 1) & 1, kStatusTimeoutEmpty);
                    tc_fence_after();
#pragma unroll 1
                    for (int e = 0; e < 8; ++e)
                        umma_f16_ts(tm + kTmO, tm + kTmWeight + buf * 64 + (e / 4) * 32 + (e % 4) * 8, vd + (e % 4) * 128, id_o,
                                    y > 0 || e > 0);
                    umma_commit(&sh.pv_done[buf]);
                }
            }
            // TMEM may be freed once the MMAs are done, also after a wait that expired
            mbar_wait_bounded(&sh.pv_done[(tiles - 1) & 1], ((tiles - 1) >> 1) & 1, limit_ns, nullptr);
        }
        __syncwarp();
    } else if (warp == 13) {
        // --------------------------------------------------------------------------------------------------- loads
        const uint64_t policy = l2_policy_evict_normal();
        int id = -1;
        auto look_up = [&](int x) {           // lane l < 4: rows 16 l .. of the tile
            const int row = x * kTileCols + lane * 16;
            id = x < tiles && lane < 4 && row < seq.len ? table[row / page] : -1;
        };
        look_up(0);
#pragma unroll 1
        for (int x = 0; x < tiles; ++x) {
            const bool in = id >= 0 && id < a.c.pages;
            const int at = (id * heads + h) * page + (x * kTileCols + lane * 16) % page;
            const uint32_t have = __popc(__ballot_sync(0xFFFFFFFFu, in));
#pragma unroll 1
            for (int e = 0; e < 2; ++e) {     // k, then v
                if (x > 0) wait(&sh.in_free[e], (x - 1) & 1, kStatusTimeoutEmpty);
                if (lane == 0) {
                    fence_proxy_async_smem();
                    mbar_arrive_expect_tx(&sh.in[e], have * 16 * D);
                }
                __syncwarp();
                if (in)
#pragma unroll
                    for (int d = 0; d < D; d += 128)
                        tma_load_2d(sh.codes[e] + lane * 16 * D + d * 16, e ? &maps.v : &maps.k, &sh.in[e], d, at, policy);
                __syncwarp();
            }
            look_up(x + 1);
        }
        if (lane == 0) {
            mbar_wait_bounded(&sh.in[0], (tiles - 1) & 1, limit_ns, nullptr);
            mbar_wait_bounded(&sh.in[1], (tiles - 1) & 1, limit_ns, nullptr);
        }
        __syncwarp();
    } else {
        // ------------------------------------------------------------------------------------------- codes to bf16
        const int w = warp < 12 ? warp - 8 : warp - 10;
#pragma unroll 1
        for (int x = 0; x < tiles; ++x) {
            const int buf = x & 1;
#pragma unroll 1
            for (int e = 0; e < 2; ++e) {
                wait(&sh.in[e], x & 1, kStatusTimeoutFull);
                // K's place is free once the scores of the tile before last are there, V's once O has taken it
                if (x > 1) wait(e ? &sh.pv_done[buf] : &sh.s_full[buf], ((x >> 1) - 1) & 1, kStatusTimeoutEmpty);
                uint8_t* to = e ? sh.v[buf] : sh.k[buf];
                // 8 rows by 4 pieces of 16 codes a warp and turn
#pragma unroll 2
                for (int u = w; u < (kTileCols / 8) * (D / 64); u += kConverters) {
                    const int r = u / (D / 64) * 8 + lane % 8, p = u % (D / 64) * 4 + lane / 8;
                    const uint4 y = *reinterpret_cast<const uint4*>(sh.codes[e] + (r / 16) * 16 * D + step_at<D>(r % 16, p * 16));
                    uint8_t* row = to + (p / 4) * (kTileCols * 128) + r * 128;
                    const int at = (p % 4) * 2;
                    *reinterpret_cast<uint4*>(row + ((at ^ (r % 8)) * 16)) =
                        uint4{codes_bf162<0x4140>(y.x), codes_bf162<0x4342>(y.x), codes_bf162<0x4140>(y.y), codes_bf162<0x4342>(y.y)};
                    *reinterpret_cast<uint4*>(row + (((at + 1) ^ (r % 8)) * 16)) =
                        uint4{codes_bf162<0x4140>(y.z), codes_bf162<0x4342>(y.z), codes_bf162<0x4140>(y.w), codes_bf162<0x4342>(y.w)};
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(&sh.in_free[e]);
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

}  // namespace reax
