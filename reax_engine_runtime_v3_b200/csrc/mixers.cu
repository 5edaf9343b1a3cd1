// C ABI of the token mixers: the gated delta rule and the paged INT8 cache with its attention
// (declarations and contracts: include/reax_b200.h).  As in abi.cu, nothing here allocates or synchronizes.
#include <algorithm>
#include <atomic>
#include <type_traits>
#include <utility>

#include "abi_shared.h"
#include "gdn.cuh"
#include "gdn_chunk.cuh"
#include "kv8.cuh"
#include "kv8_step.cuh"
#include "kv8_tile.cuh"
#include "reax_b200.h"

namespace {

using reax_abi::fail;

constexpr int kGridYz = 65535;

bool aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }

// (`dependent`: the kernel may start while the one before it on the stream still runs, and waits for its end itself)
template <bool dependent = false, typename... P>
int launch(const char* what, void (*kernel)(P...), dim3 grid, int threads, size_t smem, void* stream, const P&... p) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads, 1, 1);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = static_cast<cudaStream_t>(stream);
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = dependent ? 1 : 0;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, p...);
    return e == cudaSuccess ? REAX_OK : reax_abi::cuda_fail(e, what);
}

int check_gdn(const char* who, const reax::GdnParams& p, int Dk, int Dv) {
    if (p.rows < 0 || p.batch < 0 || p.k_heads <= 0 || p.v_heads <= 0 || p.v_heads % p.k_heads || p.n_slots < 0)
        return fail(REAX_ERR_INVALID, "%s: rows %d, batch %d, heads %d and %d (the second a multiple of the first), "
                    "slots %d", who, p.rows, p.batch, p.k_heads, p.v_heads, p.n_slots);
    if ((Dk != 64 && Dk != 128) || (Dv != 64 && Dv != 128))
        return fail(REAX_ERR_INVALID, "%s: head widths %d and %d: each must be 64 or 128", who, Dk, Dv);
    if (p.ldq < static_cast<long long>(p.k_heads) * Dk || p.ldk < static_cast<long long>(p.k_heads) * Dk ||
        p.ldv < static_cast<long long>(p.v_heads) * Dv)
        return fail(REAX_ERR_INVALID, "%s: a row stride is shorter than its row", who);
    if (p.v_heads > kGridYz || p.batch > kGridYz)
        return fail(REAX_ERR_INVALID, "%s: at most %d heads and sequences", who, kGridYz);
    if (p.rows == 0 || p.batch == 0) return REAX_OK;
    if (!p.q || !p.k || !p.v || !p.g || !p.beta || !p.state || !p.out)
        return fail(REAX_ERR_INVALID, "%s: NULL pointer", who);
    if (!aligned(p.q, 16) || !aligned(p.k, 16) || !aligned(p.v, 16) || !aligned(p.state, 16) || !aligned(p.out, 16) ||
        p.ldq % 8 || p.ldk % 8 || p.ldv % 8)
        return fail(REAX_ERR_ALIGN, "%s: q, k, v, state and out must be 16-byte aligned, row strides multiples of 8", who);
    return REAX_OK;
}

#define REAX_GDN_DISPATCH(Dk, Dv, X)               \
    (Dk == 128 ? (Dv == 128 ? X(128, 128) : X(128, 64)) : (Dv == 128 ? X(64, 128) : X(64, 64)))

// Shared memory of a kernel above the default limit, set once for each device.
constexpr int kMaxDevices = 64;
int allow_smem(const void* kernel, std::atomic<bool> (&done)[kMaxDevices], size_t bytes) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return reax_abi::cuda_fail(e, "cudaGetDevice");
    if (dev >= kMaxDevices) return fail(REAX_ERR_DEVICE, "device ordinal %d out of range", dev);
    if (done[dev].load(std::memory_order_acquire)) return REAX_OK;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes));
    if (e != cudaSuccess) return reax_abi::cuda_fail(e, "cudaFuncSetAttribute(shared memory)");
    done[dev].store(true, std::memory_order_release);
    return REAX_OK;
}

// The bound of device-side waits for kernels that keep it in 32 bits (at most 4 s).
uint32_t wait_ns() { return static_cast<uint32_t>(std::min(reax_abi::wait_timeout_ns(), 4000000000ull)); }

// Chunks that `rows` rows of `batch` sequences can have at most, and how many of them one launch takes (the scratch memory of
// a launch is kept to about 1.5 GB; longer batches take several).
long long gdn_most_chunks(int rows, int batch) { return static_cast<long long>(rows) / reax::kChunk + std::min(rows, batch); }
size_t gdn_chunk_bytes(int k_heads, int v_heads, int Dk) {
    return static_cast<size_t>(v_heads) * sizeof(reax::GdnTiles) + static_cast<size_t>(k_heads) * (Dk / 64) * 16384;
}
long long gdn_slab(int rows, int batch, int k_heads, int v_heads, int Dk) {
    const long long cap = static_cast<long long>((1536ull << 20) / gdn_chunk_bytes(k_heads, v_heads, Dk));
    return std::min(gdn_most_chunks(rows, batch), std::max(cap, 16ll));
}

template <int DK, int DV>
int gdn_chunks(const char* who, const reax::GdnParams& p, void* workspace, int sms, void* stream) {
    static std::atomic<bool> done[kMaxDevices], tiles_done[kMaxDevices];
    int rc = allow_smem(reinterpret_cast<const void*>(reax::gdn_chunk_kernel<DK, DV>), done, reax::gdn_chunk_smem());
    if (rc == REAX_OK) rc = allow_smem(reinterpret_cast<const void*>(reax::gdn_tiles_kernel<DK>), tiles_done, reax::gdn_tiles_smem());
    reax::GdnMaps maps;
    if (rc == REAX_OK) rc = reax_abi::encode_rows(&maps.v, p.v, p.v_heads * DV, p.rows, p.ldv, DV, reax::kChunk);
    if (rc == REAX_OK)
        rc = reax_abi::encode_rows(&maps.out, p.out, p.v_heads * DV, p.rows, static_cast<long long>(p.v_heads) * DV, 32, 32);
    const long long most = gdn_most_chunks(p.rows, p.batch), slab = gdn_slab(p.rows, p.batch, p.k_heads, p.v_heads, DK);
    reax::GdnScratch scratch;
    scratch.tiles = static_cast<reax::GdnTiles*>(workspace);
    scratch.kq = static_cast<uint8_t*>(workspace) + static_cast<size_t>(slab) * p.v_heads * sizeof(reax::GdnTiles);
    for (long long x = 0; x < most && rc == REAX_OK; x += slab) {
        scratch.x0 = static_cast<int>(x);
        scratch.chunks = static_cast<int>(std::min(slab, most - x));
        // A block takes the value heads of a key head one after the other, which saves their common products; where all blocks
        // find room at once, four to an SM, more blocks of fewer heads are the shorter way.
        const int group = p.v_heads / p.k_heads;
        const int parts = static_cast<int>(std::clamp(4ll * sms / (static_cast<long long>(scratch.chunks) * p.k_heads), 1ll, static_cast<long long>(group)));
        scratch.heads = (group + parts - 1) / parts;
        rc = launch(who, reax::gdn_tiles_kernel<DK>, dim3(scratch.chunks, p.k_heads, (group + scratch.heads - 1) / scratch.heads), reax::kTilesThreads,
                    reax::gdn_tiles_smem(), stream, p, scratch, wait_ns());
        if (rc == REAX_OK)
            rc = launch<true>(who, reax::gdn_chunk_kernel<DK, DV>, dim3(p.v_heads, p.batch), reax::kChunkThreads, reax::gdn_chunk_smem(), stream, p,
                        maps, scratch, wait_ns());
    }
    return rc;
}

int check_cache(const char* who, const reax::Kv8Cache& c) {
    if (c.pages < 0 || c.heads <= 0 || c.heads > kGridYz)
        return fail(REAX_ERR_INVALID, "%s: %d pages of %d heads", who, c.pages, c.heads);
    if ((c.page != 16 && c.page != 32 && c.page != 64) || (c.dim != 64 && c.dim != 128 && c.dim != 256))
        return fail(REAX_ERR_INVALID, "%s: pages of %d rows must have 16, 32 or 64, heads of %d values 64, 128 or 256", who,
                    c.page, c.dim);
    if (!c.k || !c.v || !c.k_scale || !c.v_scale) return fail(REAX_ERR_INVALID, "%s: NULL pointer in the cache", who);
    if (!aligned(c.k, 16) || !aligned(c.v, 16)) return fail(REAX_ERR_ALIGN, "%s: codes must be 16-byte aligned", who);
    return REAX_OK;
}

int check_rows(const char* who, const int32_t* tables, const int32_t* lengths, const int32_t* cu, int rows, int batch,
               int table_ld) {
    if (rows < 0 || batch < 0 || table_ld < 0) return fail(REAX_ERR_INVALID, "%s: negative size", who);
    if (rows == 0 || batch == 0) return REAX_OK;
    if (!tables || !lengths) return fail(REAX_ERR_INVALID, "%s: NULL pointer", who);
    if (!cu && rows != batch)
        return fail(REAX_ERR_INVALID, "%s: %d rows for %d sequences: without cu_seqlens each has one", who, rows, batch);
    return REAX_OK;
}

// Workspace of the attention: counters (zero between calls), then the parts of items that blocks share.
struct AttendWorkspace {
    reax::StepWork step;
    reax::TileWork tile;
    size_t bytes;
    AttendWorkspace(void* base, int sms) {
        char* p = static_cast<char*>(base);
        size_t at = 0;
        auto take = [&](auto*& to, size_t n) {
            to = reinterpret_cast<std::remove_reference_t<decltype(to)>>(p + at);
            at += (n * sizeof(*to) + 255) / 256 * 256;
        };
        const size_t blocks = static_cast<size_t>(sms) * reax::kStepBlocksPerSm;
        take(step.counters, blocks);
        const size_t shared = at;
        take(step.stats, blocks * 2 * 2 * reax::kStepRows);
        take(step.parts, blocks * 2 * reax::kStepRows * 256);
        bytes = at;
        at = shared;
        take(tile.rest, sms);
        take(tile.stats, static_cast<size_t>(sms) * 2 * 2 * reax::kTileRows);
        take(tile.sums, static_cast<size_t>(sms) * 2 * reax::kTileRows * 256);
        bytes = std::max(bytes, at);
    }
};

// Rows x heads of a sequence up to which the step form is used: it reads the cache once for each 16 of them.  Measured (us on
// the device, by it / by the form for many rows, 4 cached heads):
//   values a head                            64          128          256
//   64 sequences of 4096 rows, 16:      78 / 152     92 / 164    144 / 208
//                              32:     134 / 153    162 / 165    253 / 207
//   16 sequences of 1024 rows, 16:      18 / 26      21 / 28      31 / 35
//                              32:      26 / 26      30 / 29      42 / 36
//   one of 65536 rows,         16:      46 / 51      52 / 55      73 / 67
//                              32:      53 / 52      62 / 56      91 / 69
//   one of 4096 rows,          16:      19 / 21      21 / 22      26 / 26
//                              32:      19 / 21      22 / 22      29 / 27
constexpr int kStepMostRows = reax::kStepRows;

template <int D>
int attend_tiles(const char* who, const reax::Kv8Attend& a, const reax::Kv8Maps& maps, void* workspace, int sms, void* stream) {
    static std::atomic<bool> done[kMaxDevices];
    constexpr size_t smem = sizeof(reax::TileShared<D>) + 1024;
    static_assert(smem <= 227 * 1024, "shared memory of one block");
    int rc = allow_smem(reinterpret_cast<const void*>(reax::kv8_tile_kernel<D>), done, smem);
    if (rc != REAX_OK) return rc;
    const reax::TileWork work = AttendWorkspace(workspace, sms).tile;
    const int blocks = std::min(sms, reax::kMostTileBlocks);
    rc = launch(who, reax::kv8_tile_kernel<D>, dim3(blocks), reax::kAttendTileThreads, smem, stream, a, maps, work, wait_ns());
    if (rc != REAX_OK) return rc;
    return launch<true>(who, reax::kv8_join_kernel<D>, dim3(sms * reax::kJoinBlocksPerSm), reax::kJoinThreads, 0, stream, a, work, blocks);
}

template <int D>
int attend_step(const char* who, const reax::Kv8Attend& a, void* workspace, int sms, void* stream) {
    static std::atomic<bool> done[kMaxDevices];
    constexpr size_t smem = sizeof(reax::StepShared<D>) + 1024;
    int rc = allow_smem(reinterpret_cast<const void*>(reax::kv8_step_kernel<D>), done, smem);
    if (rc != REAX_OK) return rc;
    const reax::StepWork work = AttendWorkspace(workspace, sms).step;
    const int blocks = sms * reax::kStepBlocksPerSm;
    // A captured call clears its counters: whether the zeroing of the workspace, or the call before on the capturing stream, runs
    // before the replay is not known here.  The attention begins meanwhile (one row over 4097: 18.2 us on the device without
    // it, 19.5 with it, 22.7 with a cudaMemsetAsync).
    cudaStreamCaptureStatus capture;
    const cudaError_t e = cudaStreamIsCapturing(static_cast<cudaStream_t>(stream), &capture);
    if (e != cudaSuccess) return reax_abi::cuda_fail(e, who);
    if (capture == cudaStreamCaptureStatusNone)
        return launch(who, reax::kv8_step_kernel<D>, dim3(blocks), reax::kAttendStepThreads, smem, stream, a, work);
    rc = launch(who, reax::kv8_clear_kernel, dim3(1), reax::kAttendStepThreads, 0, stream, work, blocks);
    if (rc != REAX_OK) return rc;
    return launch<true>(who, reax::kv8_step_kernel<D>, dim3(blocks), reax::kAttendStepThreads, smem, stream, a, work);
}

}  // namespace

extern "C" {

size_t reax_gdn_workspace_bytes(int rows, int batch, int k_heads, int v_heads, int Dk) {
    if (rows <= 0 || batch <= 0 || k_heads <= 0 || v_heads <= 0 || (Dk != 64 && Dk != 128)) return 0;
    return static_cast<size_t>(gdn_slab(rows, batch, k_heads, v_heads, Dk)) * gdn_chunk_bytes(k_heads, v_heads, Dk);
}

int reax_gdn_prefill(const void* q, const void* k, const void* v, const float* g, const float* beta, float* state,
                     const int32_t* cu_seqlens, const int32_t* slots, void* out, int rows, int batch, int k_heads,
                     int v_heads, int Dk, int Dv, int n_slots, long long ldq, long long ldk, long long ldv, float scale,
                     int normalize, int carry, void* workspace, size_t workspace_bytes, void* stream) {
    using bf16 = __nv_bfloat16;
    const reax::GdnParams p = {static_cast<const bf16*>(q), static_cast<const bf16*>(k), static_cast<const bf16*>(v), g,
                               beta, state, cu_seqlens, slots, static_cast<bf16*>(out), ldq, ldk, ldv, rows, batch, k_heads,
                               v_heads, n_slots, scale, normalize, carry};
    int rc = check_gdn("reax_gdn_prefill", p, Dk, Dv), sms = 0;
    if (rc != REAX_OK || rows == 0 || batch == 0) return rc;
    if (!cu_seqlens && batch != 1)
        return fail(REAX_ERR_INVALID, "reax_gdn_prefill: %d sequences need cu_seqlens", batch);
    if ((rc = reax_abi::current_sms(&sms)) != REAX_OK) return rc;
    const size_t need = reax_gdn_workspace_bytes(rows, batch, k_heads, v_heads, Dk);
    if (!workspace || workspace_bytes < need)
        return fail(REAX_ERR_WORKSPACE, "reax_gdn_prefill: workspace of %zu bytes, needs reax_gdn_workspace_bytes() = %zu", workspace_bytes, need);
    if (!aligned(workspace, 128)) return fail(REAX_ERR_ALIGN, "reax_gdn_prefill: the workspace must be 128-byte aligned");
#define X(K, V) gdn_chunks<K, V>("reax_gdn_prefill", p, workspace, sms, stream)
    return REAX_GDN_DISPATCH(Dk, Dv, X);
#undef X
}

int reax_mixer_status(unsigned* status, int clear, void* stream) {
    if (!status) return fail(REAX_ERR_INVALID, "reax_mixer_status: NULL pointer");
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    unsigned zero = 0;
    cudaError_t e = cudaMemcpyFromSymbolAsync(status, reax::g_mixer_status, sizeof(unsigned), 0, cudaMemcpyDeviceToHost, s);
    if (e == cudaSuccess && clear)
        e = cudaMemcpyToSymbolAsync(reax::g_mixer_status, &zero, sizeof(unsigned), 0, cudaMemcpyHostToDevice, s);
    if (e == cudaSuccess) e = cudaStreamSynchronize(s);
    return e == cudaSuccess ? REAX_OK : reax_abi::cuda_fail(e, "reax_mixer_status");
}

int reax_gdn_decode(const void* q, const void* k, const void* v, const float* g, const float* beta, float* state,
                    const int32_t* slots, void* out, int batch, int k_heads, int v_heads, int Dk, int Dv, int n_slots,
                    long long ldq, long long ldk, long long ldv, float scale, int normalize, void* stream) {
    using bf16 = __nv_bfloat16;
    const reax::GdnParams p = {static_cast<const bf16*>(q), static_cast<const bf16*>(k), static_cast<const bf16*>(v), g,
                               beta, state, nullptr, slots, static_cast<bf16*>(out), ldq, ldk, ldv, batch, batch, k_heads,
                               v_heads, n_slots, scale, normalize, 1};
    int rc = check_gdn("reax_gdn_decode", p, Dk, Dv), sms = 0;
    if (rc != REAX_OK || batch == 0) return rc;
    if ((rc = reax_abi::current_sms(&sms)) != REAX_OK) return rc;
#define X(K, V) reax::gdn_step_kernel<K, V>
    return launch("reax_gdn_decode", REAX_GDN_DISPATCH(Dk, Dv, X), dim3(v_heads, batch), reax::kStepThreads, 0, stream, p);
#undef X
}

int reax_kv8_append(const void* k, const void* v, int8_t* k_codes, int8_t* v_codes, float* k_scales, float* v_scales,
                    const int32_t* tables, const int32_t* lengths, const int32_t* cu_seqlens, int rows, int batch,
                    int table_ld, int pages, int heads, int page, int dim, long long ldk, long long ldv, void* stream) {
    const char* who = "reax_kv8_append";
    using bf16 = __nv_bfloat16;
    const reax::Kv8Append a = {{k_codes, v_codes, k_scales, v_scales, pages, heads, page, dim},
                               static_cast<const bf16*>(k), static_cast<const bf16*>(v), ldk, ldv, tables, lengths,
                               cu_seqlens, rows, batch, table_ld};
    int rc = check_rows(who, tables, lengths, cu_seqlens, rows, batch, table_ld), sms = 0;
    if (rc != REAX_OK || rows == 0 || batch == 0) return rc;
    if ((rc = check_cache(who, a.c)) != REAX_OK) return rc;
    if (!k || !v) return fail(REAX_ERR_INVALID, "%s: NULL pointer", who);
    if (ldk < static_cast<long long>(heads) * dim || ldv < static_cast<long long>(heads) * dim)
        return fail(REAX_ERR_INVALID, "%s: a row stride is shorter than its row", who);
    if (!aligned(k, 16) || !aligned(v, 16) || ldk % 8 || ldv % 8)
        return fail(REAX_ERR_ALIGN, "%s: k and v must be 16-byte aligned, row strides multiples of 8", who);
    if ((rc = reax_abi::current_sms(&sms)) != REAX_OK) return rc;
    // n new rows touch at most (n - 1) / page + 2 pages: the most that any split of `rows` over the batch gives
    const long long most = cu_seqlens ? static_cast<long long>(rows) / page + 2ll * std::min(rows, batch) : batch;
    return launch(who, reax::kv8_append_kernel, dim3(static_cast<unsigned>(most), heads, 2), reax::kAppendThreads, 0, stream,
                  a);
}

int reax_kv8_read(const int8_t* k_codes, const int8_t* v_codes, const float* k_scales, const float* v_scales,
                  const int32_t* tables, const int32_t* starts, const int32_t* cu_seqlens, void* k, void* v, int rows,
                  int batch, int table_ld, int pages, int heads, int page, int dim, void* stream) {
    const char* who = "reax_kv8_read";
    const reax::Kv8Read a = {{const_cast<int8_t*>(k_codes), const_cast<int8_t*>(v_codes), const_cast<float*>(k_scales),
                              const_cast<float*>(v_scales), pages, heads, page, dim},
                             tables, starts, cu_seqlens, static_cast<__nv_bfloat16*>(k), static_cast<__nv_bfloat16*>(v), rows,
                             batch, table_ld};
    int rc = check_rows(who, tables, starts, cu_seqlens, rows, batch, table_ld), sms = 0;
    if (rc != REAX_OK || rows == 0 || batch == 0) return rc;
    if ((rc = check_cache(who, a.c)) != REAX_OK) return rc;
    if (!cu_seqlens || !k || !v) return fail(REAX_ERR_INVALID, "%s: NULL pointer", who);
    if (!aligned(k, 16) || !aligned(v, 16)) return fail(REAX_ERR_ALIGN, "%s: k and v must be 16-byte aligned", who);
    if ((rc = reax_abi::current_sms(&sms)) != REAX_OK) return rc;
    return launch(who, reax::kv8_read_kernel, dim3(std::min((rows + 7) / 8, sms * 8), 2), 256, 0,
                  stream, a);
}

size_t reax_kv8_workspace_bytes(int device) {
    const int sms = reax_abi::device_sms(device);
    return sms < 0 ? 0 : AttendWorkspace(nullptr, sms).bytes;
}

int reax_kv8_attend(const void* q, const int8_t* k_codes, const int8_t* v_codes, const float* k_scales,
                    const float* v_scales, const int32_t* tables, const int32_t* lengths, const int32_t* cu_seqlens,
                    void* out, float* lse, int rows, int max_rows, int batch, int table_ld, int pages, int heads, int group,
                    int page, int dim, long long ldq, float scale, void* workspace, size_t workspace_bytes, void* stream) {
    const char* who = "reax_kv8_attend";
    const int capacity = static_cast<int>(std::min(std::max(table_ld, 0) * static_cast<long long>(page), 0x7FFFFFC0ll));
    const reax::Kv8Attend a = {{const_cast<int8_t*>(k_codes), const_cast<int8_t*>(v_codes), const_cast<float*>(k_scales),
                                const_cast<float*>(v_scales), pages, heads, page, dim},
                               static_cast<const __nv_bfloat16*>(q), ldq, tables, lengths, cu_seqlens,
                               static_cast<__nv_bfloat16*>(out), lse, rows, batch, table_ld, group, capacity, scale};
    int rc = check_rows(who, tables, lengths, cu_seqlens, rows, batch, table_ld), sms = 0;
    if (rc != REAX_OK || rows == 0 || batch == 0) return rc;
    if ((rc = check_cache(who, a.c)) != REAX_OK) return rc;
    if (!q || !out) return fail(REAX_ERR_INVALID, "%s: NULL pointer", who);
    if (group <= 0 || heads * static_cast<long long>(group) > kGridYz)
        return fail(REAX_ERR_INVALID, "%s: %d query heads a cached head, %d cached heads", who, group, heads);
    if (ldq < static_cast<long long>(heads) * group * dim) return fail(REAX_ERR_INVALID, "%s: row stride shorter than a row", who);
    if (!aligned(q, 16) || !aligned(out, 16) || ldq % 8)
        return fail(REAX_ERR_ALIGN, "%s: q and out must be 16-byte aligned, the row stride a multiple of 8", who);
    if ((rc = reax_abi::current_sms(&sms)) != REAX_OK) return rc;
    if (!workspace || workspace_bytes < AttendWorkspace(nullptr, sms).bytes)
        return fail(REAX_ERR_WORKSPACE, "%s: workspace of %zu bytes, needs reax_kv8_workspace_bytes() = %zu", who, workspace_bytes,
                    AttendWorkspace(nullptr, sms).bytes);
    if (!aligned(workspace, 256)) return fail(REAX_ERR_ALIGN, "%s: the workspace must be 256-byte aligned", who);
    if (static_cast<long long>(max_rows) * group > kStepMostRows) {
        const long long pool = static_cast<long long>(pages) * heads * page;
        if (pool > 0x7FFFFFFF) return fail(REAX_ERR_INVALID, "%s: the pool has 2^31 rows or more", who);
        reax::Kv8Maps maps;
        if ((rc = reax_abi::encode_codes(&maps.k, k_codes, dim, std::max(pool, 16ll), 16)) != REAX_OK) return rc;
        if ((rc = reax_abi::encode_codes(&maps.v, v_codes, dim, std::max(pool, 16ll), 16)) != REAX_OK) return rc;
        if (dim == 64) return attend_tiles<64>(who, a, maps, workspace, sms, stream);
        if (dim == 128) return attend_tiles<128>(who, a, maps, workspace, sms, stream);
        return attend_tiles<256>(who, a, maps, workspace, sms, stream);
    }
    if (dim == 64) return attend_step<64>(who, a, workspace, sms, stream);
    if (dim == 128) return attend_step<128>(who, a, workspace, sms, stream);
    return attend_step<256>(who, a, workspace, sms, stream);
}

}  // extern "C"
