// A paged INT8 cache of keys and values, and attention over it.
//
// Page p of head h holds `page` rows of D codes (codes [pages, heads, page, D]) and one scale
// (scales [pages, heads]); a code c stands for c * scale.  Sequence b's row i lies in page
// tables[b, i / page], place i % page.
#pragma once

#include "common.cuh"

namespace reax {

struct Kv8Cache {
    int8_t* k;
    int8_t* v;
    float* k_scale;
    float* v_scale;
    int pages, heads, page, dim;
};

struct Kv8Append {
    Kv8Cache c;
    const __nv_bfloat16* k;   // [rows, heads, dim], row stride ldk
    const __nv_bfloat16* v;
    long long ldk, ldv;
    const int32_t* tables;    // [batch, table_ld]
    const int32_t* lengths;   // [batch]: rows cached before this call
    const int32_t* cu;        // [batch + 1] (NULL: one row a sequence)
    int rows, batch, table_ld;
};

REAX_DEVI void kv8_span(const int32_t* cu, int b, int rows, int* lo, int* hi) {
    int l = cu ? cu[b] : b, h = cu ? cu[b + 1] : b + 1;
    *lo = min(max(l, 0), rows);
    *hi = min(max(h, *lo), rows);
}

REAX_DEVI float warp_max(float v) {
#pragma unroll
    for (int m = 16; m > 0; m >>= 1) v = fmaxf(v, __shfl_xor_sync(0xFFFFFFFFu, v, m));
    return v;
}

// |x| of a bf16 pair's two values, infinities and NaN left out.
REAX_DEVI float absmax_finite(float m, uint32_t w) {
    const uint32_t a = (w << 16) & 0x7FFF0000u, b = w & 0x7FFF0000u;
    if (a < 0x7F800000u) m = fmaxf(m, __uint_as_float(a));
    if (b < 0x7F800000u) m = fmaxf(m, __uint_as_float(b));
    return m;
}

// rint(x / scale) kept in [-127, 127]; NaN gives 0.
REAX_DEVI int kv8_code(float x, float scale) {
    const float q = rintf(__fdiv_rn(x, scale));
    return q != q ? 0 : static_cast<int>(fminf(fmaxf(q, -127.0f), 127.0f));
}

// (Not inlined: it is rare, and the division is long.)
__device__ __noinline__ uint32_t kv8_codes_divided(float x0, float x1, float x2, float x3, float scale) {
    return (kv8_code(x0, scale) & 0xFF) | (kv8_code(x1, scale) & 0xFF) << 8 | (kv8_code(x2, scale) & 0xFF) << 16 |
           static_cast<uint32_t>(kv8_code(x3, scale)) << 24;
}

// The codes of 4 values.  x times the scale's inverse is within 127 * 2^-22 of x / scale, so that it rounds to the same whole
// number unless it lies that near to a half; those few, and what is not finite, take the division.
REAX_DEVI uint32_t kv8_codes(float x0, float x1, float x2, float x3, float scale, float inv) {
    constexpr float kRound = 12582912.0f;     // 1.5 * 2^23: a sum with it is rounded to a whole number, in its low bits
    const float x[4] = {x0, x1, x2, x3};
    uint32_t c[4];
    bool sure = true;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float t = __fmaf_rn(x[i], inv, kRound);
        sure = sure && fabsf(__fmaf_rn(x[i], inv, kRound - t)) <= 0.4999f;
        c[i] = __float_as_uint(t);
    }
    if (!sure) return kv8_codes_divided(x0, x1, x2, x3, scale);
    return __byte_perm(__byte_perm(c[0], c[1], 0x0040), __byte_perm(c[2], c[3], 0x0040), 0x5410);
}

// One block writes the new rows of one page, one head, of k (blockIdx.z = 0) or v (1).  Block x is the x-th
// page touched, counted over the sequences in order: a warp's prefix sum over the batch finds whose it is,
// so the host need not know the lengths.  Bound by bytes in the long run (rows read once, in registers for both the page's
// maximum and its codes): 8192 rows of 4 heads of 256 take 21 us to append and 12 to read back, where their bytes take 8 each:
// two rounds of blocks here and a search for each row there, chains of loads that need each other.
constexpr int kAppendThreads = 256;

__global__ void __launch_bounds__(kAppendThreads) kv8_append_kernel(const Kv8Append a) {
    __shared__ int s_seq, s_page;
    __shared__ float s_max[kAppendThreads / 32];
    const int tid = threadIdx.x, lane = tid % 32;
    if (tid < 32) {
        int before = 0, seq = -1, page = 0;
        for (int b0 = 0; b0 < a.batch; b0 += 32) {
            int n = 0, first = 0;
            if (b0 + lane < a.batch) {
                int lo, hi;
                kv8_span(a.cu, b0 + lane, a.rows, &lo, &hi);
                const int len = max(a.lengths[b0 + lane], 0);
                first = len / a.c.page;
                n = hi > lo ? (len + hi - lo - 1) / a.c.page - first + 1 : 0;
            }
            int sum = n;
#pragma unroll
            for (int m = 1; m < 32; m <<= 1) {
                const int t = __shfl_up_sync(0xFFFFFFFFu, sum, m);
                if (lane >= m) sum += t;
            }
            const int x = static_cast<int>(blockIdx.x) - before;
            const bool mine = x >= sum - n && x < sum;
            const unsigned who = __ballot_sync(0xFFFFFFFFu, mine);
            if (who) {
                const int l = __ffs(who) - 1;
                seq = b0 + l;
                page = __shfl_sync(0xFFFFFFFFu, first + x - (sum - n), l);
                break;
            }
            before += __shfl_sync(0xFFFFFFFFu, sum, 31);
        }
        if (lane == 0) s_seq = seq, s_page = page;
    }
    __syncthreads();
    const int b = s_seq, pg = s_page;
    if (b < 0 || pg >= a.table_ld) return;
    const int id = a.tables[static_cast<long long>(b) * a.table_ld + pg];
    int lo, hi;
    kv8_span(a.cu, b, a.rows, &lo, &hi);
    const int len = max(a.lengths[b], 0), h = blockIdx.y, dim = a.c.dim;
    const int from = max(len - pg * a.c.page, 0);                     // places of the page held before
    const int to = min(len + hi - lo - pg * a.c.page, a.c.page);
    const bool is_v = blockIdx.z != 0;
    const long long ld = is_v ? a.ldv : a.ldk;
    const __nv_bfloat16* src = (is_v ? a.v : a.k) + (lo + static_cast<long long>(pg) * a.c.page + from - len) * ld + h * dim;
    const int per_row = dim / 8, row_shift = __ffs(per_row) - 1, total = (to - from) * per_row;       // pieces of 8 values
    constexpr int kHeld = 64 * 256 / 8 / kAppendThreads;              // a whole page of the largest size
    uint4 x[kHeld];                                                   // (asked for before the page's number is looked at)
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
        const int e = tid + i * kAppendThreads;
        x[i] = e < total ? *reinterpret_cast<const uint4*>(src + (e >> row_shift) * ld + (e & (per_row - 1)) * 8) : uint4{};
    }
    if (id < 0 || id >= a.c.pages) return;
    const long long at = static_cast<long long>(id) * a.c.heads + h;
    int8_t* dst = (is_v ? a.c.v : a.c.k) + at * a.c.page * dim;
    float* scale = (is_v ? a.c.v_scale : a.c.k_scale) + at;
    const float was = from > 0 ? *scale : 0.0f;
    float m = 0.0f;
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
        const int e = tid + i * kAppendThreads;
        if (e < total) {
            m = absmax_finite(absmax_finite(absmax_finite(absmax_finite(m, x[i].x), x[i].y), x[i].z), x[i].w);
        }
    }
    m = warp_max(m);
    if (lane == 0) s_max[tid / 32] = m;
    __syncthreads();
    m = s_max[0];
#pragma unroll
    for (int i = 1; i < kAppendThreads / 32; ++i) m = fmaxf(m, s_max[i]);
    const float now = fmaxf(was, __fdiv_rn(fmaxf(m, 1e-12f), 127.0f));
    if (tid == 0) *scale = now;
    const float inv = __frcp_rn(now);
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
        const int e = tid + i * kAppendThreads;
        if (e < total) {
            auto lo = [](uint32_t w) { return __uint_as_float(w << 16); };
            auto hi = [](uint32_t w) { return __uint_as_float(w & 0xFFFF0000u); };
            *reinterpret_cast<uint2*>(dst + (from + (e >> row_shift)) * dim + (e & (per_row - 1)) * 8) =
                uint2{kv8_codes(lo(x[i].x), hi(x[i].x), lo(x[i].y), hi(x[i].y), now, inv),
                      kv8_codes(lo(x[i].z), hi(x[i].z), lo(x[i].w), hi(x[i].w), now, inv)};
        }
    }
    if (now > was && from > 0) {
        const float r = __fdiv_rn(was, now);
        uint32_t* old = reinterpret_cast<uint32_t*>(dst);
        for (int e = tid; e < from * dim / 4; e += kAppendThreads) {
            const uint32_t w = old[e];
            uint32_t o = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float f = static_cast<float>(static_cast<int8_t>(w >> (8 * j)));
                o |= (static_cast<uint32_t>(static_cast<int>(rintf(__fmul_rn(f, r)))) & 0xFFu) << (8 * j);
            }
            old[e] = o;
        }
    }
}

// ------------------------------------------------------------------------------------------------- read back
struct Kv8Read {
    Kv8Cache c;
    const int32_t* tables;
    const int32_t* starts;    // [batch]: first cached row read
    const int32_t* cu;        // [batch + 1]: rows read, packed
    __nv_bfloat16* k;         // [rows, heads, dim]
    __nv_bfloat16* v;
    int rows, batch, table_ld;
};

// A warp a row, 16 codes a lane and turn; row r of the output belongs to the last sequence that starts at or before it.
__global__ void __launch_bounds__(256) kv8_read_kernel(const Kv8Read a) {
    const int lane = threadIdx.x % 32, shift = __ffs(a.c.page) - 1, dim_shift = __ffs(a.c.dim) - 1;
    const bool is_v = blockIdx.y != 0;
    const int8_t* codes = is_v ? a.c.v : a.c.k;
    const float* scales = is_v ? a.c.v_scale : a.c.k_scale;
    __nv_bfloat16* out = is_v ? a.v : a.k;
    const int width = a.c.heads << dim_shift;
    for (int r = blockIdx.x * 8 + threadIdx.x / 32; r < a.rows; r += gridDim.x * 8) {
        int lo = 0, hi = a.batch;                                     // cu[lo] <= r < cu[hi]
        if (a.batch > 1) {
            // 32 places at a time: the lanes' comparisons narrow the range to a 32nd
            while (hi - lo > 1) {
                const int step = (hi - lo + 31) / 32, at = lo + lane * step;
                const unsigned below = __ballot_sync(0xFFFFFFFFu, at < hi && (lane == 0 || a.cu[at] <= r));
                const int last = 31 - __clz(below);
                hi = min(hi, lo + (last + 1) * step);
                lo += last * step;
            }
        }
        const int place = a.starts[lo] + r - a.cu[lo];
        int id = -1;
        if (place >= 0 && r < a.cu[a.batch] && (place >> shift) < a.table_ld)
            id = a.tables[static_cast<long long>(lo) * a.table_ld + (place >> shift)];
        const bool in = id >= 0 && id < a.c.pages;
        const long long first = static_cast<long long>(in ? id : 0) * a.c.heads;
        for (int x = lane * 16; x < width; x += 512) {
            const int h = x >> dim_shift;
            uint4 o[2] = {};
            if (in) {
                const uint4 w = *reinterpret_cast<const uint4*>(codes + (((first + h) << shift) + (place & (a.c.page - 1))) * a.c.dim +
                                                                (x & (a.c.dim - 1)));
                const float s = scales[first + h];
                const uint32_t c[4] = {w.x, w.y, w.z, w.w};
                uint32_t y[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const uint32_t b = c[j / 2] >> (16 * (j % 2));
                    y[j] = bf16x2_rn(f2(static_cast<int8_t>(b) * s, static_cast<int8_t>(b >> 8) * s));
                }
                o[0] = uint4{y[0], y[1], y[2], y[3]}, o[1] = uint4{y[4], y[5], y[6], y[7]};
            }
            uint4* to = reinterpret_cast<uint4*>(out + static_cast<long long>(r) * width + x);
            to[0] = o[0], to[1] = o[1];
        }
    }
}

// ------------------------------------------------------------------------------------------------- attention
struct Kv8Attend {
    Kv8Cache c;
    const __nv_bfloat16* q;   // [rows, heads * group, dim], row stride ldq
    long long ldq;
    const int32_t* tables;
    const int32_t* lengths;   // [batch]: rows cached, the new ones among them
    const int32_t* cu;        // [batch + 1] (NULL: one row a sequence)
    __nv_bfloat16* out;       // [rows, heads * group, dim]
    float* lse;               // [rows, heads * group] or NULL
    int rows, batch, table_ld, group;
    int capacity;             // rows that a table has places for, at most 2^31 - 64
    float scale;
};

}  // namespace reax
