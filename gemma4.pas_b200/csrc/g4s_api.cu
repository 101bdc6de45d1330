// g4s_api.cu -- C ABI of the sampler: context, argument checks, row routing,
// kernel launches.  See include/g4sampler.h for the contract.
#include <cuda_runtime.h>

#include <algorithm>

#include <dlfcn.h>
#include <nccl.h>

#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <cstring>
#include <initializer_list>
#include <chrono>
#include <string>
#include <thread>

#include "g4s_kernels.cuh"
#include "g4sampler.h"

namespace g4s {
constexpr int KMAX_ = 256;
constexpr int NCH_MAX_ = 1024;
constexpr int STREAM_MIN_CHUNK_ = 8192;  // shortest chunk given to it (four tiles)
constexpr int STREAM_MIN_ROWS_ = 64;     // fewer rows: the chunk kernel's shorter chunks win (B = 32 measured)
constexpr int LK_SLOTS = 16;
constexpr int PSLOTS = 4;  // per-row params staging slots
}  // namespace g4s

using namespace g4s;

struct g4s_ctx {
    int device = -1;
    int max_rows = 0;
    int max_vocab = 0;
    uint32_t flags = 0;
    int sm_count = 0;
    bool cluster_ok = false;  // the single-row cluster kernel can be scheduled
    cudaStream_t stream = nullptr;
    // workspace (one allocation)
    void *ws = nullptr;
    size_t ws_bytes = 0;
    int64_t lists_cap = 0;  // per-chunk candidate lists available
    uint64_t *cand = nullptr;
    int32_t *cand_cnt = nullptr;
    uint32_t *counters_topk = nullptr;
    float4 *istat = nullptr;
    int persist[2][2] = {{0, 0}, {0, 0}};  // full-path streaming CTAs per SM [dtype][vec]
    int persist_tab = 0;                   // the same for the bf16 softcap-table variant
    float *sc_tab = nullptr;               // bf16 softcap table (workspace), built for sc_tab_cap
    float sc_tab_cap = 0.0f;               // softcap the table holds (0: not built)
    float *e_tab = nullptr;                // bf16 weight table of one (softcap, 1/T) (workspace)
    float e_tab_cap = 0.0f, e_tab_invt = 0.0f;  // what it holds (cap 0: not built)
    int persist_etab = 0;                  // CTAs per SM of the weight-table kernel
    ShardTarget *shard_tgt = nullptr;      // [max_rows] sharded full-vocabulary draws (workspace)
    RowStat *rowstat = nullptr;
    int32_t *lk_idx = nullptr;
    float *lk_val = nullptr;
    g4s_params *params_dev = nullptr;
    // per-row params staging: a ring of PSLOTS pinned slots and device slots,
    // so the host can enqueue a few calls ahead of the GPU
    g4s_params *params_pinned = nullptr;
    cudaEvent_t params_ev[4] = {nullptr, nullptr, nullptr, nullptr};
    bool params_ev_pending[4] = {false, false, false, false};
    int params_slot = 0;
    // vocabulary-sharded mode (g4s_shard_init)
    void *nccl_comm = nullptr;
    int shard_world = 0, shard_rank = 0, shard_vocab = 0, shard_slice = 0;
    int64_t shard_timeout_ms = G4S_SHARD_TIMEOUT_MS_DEFAULT;  // host deadline of rendezvous and waits
    cudaEvent_t shard_ev = nullptr;                           // g4s_shard_wait's marker
    uint64_t *sh_send = nullptr;  // [max_rows][KMAX] this rank's lists, then [max_rows] counts
    uint64_t *sh_recv = nullptr;  // [world][max_rows][KMAX], then [world][max_rows] counts
    int32_t *sh_off = nullptr;    // [max_rows] packed list offsets of a g4s_shard_sample step
    // LM head workspace (first g4s_lmhead_sample call): fp32 logits and fp16 hidden
    float *lm_logits = nullptr;
    void *lm_xh = nullptr;
    float4 *beam_stat = nullptr;  // [max_rows][beam_items(max_vocab)] item statistics of g4s_beam_select
    int4 *pg_copies = nullptr;  // [max_rows] page copies a g4s_pages_fork lists, and their count
    int *pg_n_copies = nullptr;
    int *dev_err = nullptr;  // device error flag in the workspace (a bounded wait that ran out), read by g4s_device_status
    int64_t wait_limit = 0;  // g4s_set_wait_limit (test hook; 0 = the kernels' own limits)
    size_t lm_logits_n = 0, lm_xh_n = 0;
    void *lm_fused = nullptr;  // fused LM head: candidates, counts, thresholds, sample logits
    size_t lm_fused_n = 0;
    // g4s_sample_host staging
    void *h_logits = nullptr;
    double *h_u = nullptr;
    int32_t *h_tok = nullptr;
    std::string err;
};

static thread_local std::string g_create_err;

static int32_t fail(g4s_ctx *ctx, int32_t code, const char *fmt, ...)
{
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof(buf), fmt, ap);
    va_end(ap);
    if (ctx) ctx->err = buf;
    else g_create_err = buf;
    return code;
}

// Makes the context's device current for the duration of a call.
struct DeviceGuard {
    int prev = -1;
    bool ok = true;
    explicit DeviceGuard(int dev)
    {
        if (cudaGetDevice(&prev) != cudaSuccess) prev = -1;
        if (prev != dev) ok = cudaSetDevice(dev) == cudaSuccess;
    }
    ~DeviceGuard()
    {
        int cur = -1;
        if (prev >= 0 && cudaGetDevice(&cur) == cudaSuccess && cur != prev) cudaSetDevice(prev);
    }
};

static int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

static bool create_param_events(g4s_ctx *ctx)
{
    for (int k = 0; k < PSLOTS; k++)
        if (cudaEventCreateWithFlags(&ctx->params_ev[k], cudaEventDisableTiming) != cudaSuccess) return false;
    return true;
}

// Chunk size for a call: 2048 ids (8 per thread) when big chunks would leave
// the GPU under two CTAs per SM, else 8192 ids (32 per thread).
static int choose_ept(const g4s_ctx *ctx, int rows, int vocab)
{
    const int64_t big = ceil_div(vocab, 8192);
    if ((int64_t)rows * big < 2LL * ctx->sm_count && ceil_div(vocab, 2048) <= NCH_MAX_) return 8;
    return 32;
}

// Top-K chunking of a call: the streaming pass (long chunks, a running
// threshold, bulk copies: 16-byte aligned rows) for batches of 64 rows or more
// where big chunks would be chosen, split so that the grid fills the resident
// CTA slots once; the chunks of choose_ept otherwise.
struct TopkChunks {
    int chunk, nch;
    bool stream;
};
static TopkChunks choose_topk_chunks(const g4s_ctx *ctx, int rows, int vocab, bool vec)
{
    const int ept = choose_ept(ctx, rows, vocab);
    if (ept == 32 && vec && vocab >= STREAM_MIN_CHUNK_ && rows >= STREAM_MIN_ROWS_) {
        const int64_t slots = (int64_t)topk_stream_blocks_per_sm() * ctx->sm_count;
        const int64_t splits = std::max<int64_t>(1, slots / rows);
        int64_t chunk = ceil_div(ceil_div(vocab, splits), STREAM_TILE) * STREAM_TILE;
        if (chunk < STREAM_MIN_CHUNK_) chunk = STREAM_MIN_CHUNK_;
        return {(int)chunk, (int)ceil_div(vocab, chunk), true};
    }
    return {ept * 256, (int)ceil_div(vocab, ept * 256), false};
}

// NCCL, loaded on first use of the sharded API (the rest of the library does
// not depend on it).  A process that already holds libnccl.so.2 (PyTorch's,
// for instance) shares that copy.
struct NcclApi {
    bool tried = false, ok = false;
    std::string why;
    ncclResult_t (*GetUniqueId)(ncclUniqueId *) = nullptr;
    ncclResult_t (*CommInitRankConfig)(ncclComm_t *, int, ncclUniqueId, int, ncclConfig_t *) = nullptr;
    ncclResult_t (*CommGetAsyncError)(ncclComm_t, ncclResult_t *) = nullptr;
    ncclResult_t (*CommDestroy)(ncclComm_t) = nullptr;
    ncclResult_t (*CommAbort)(ncclComm_t) = nullptr;
    ncclResult_t (*AllGather)(const void *, void *, size_t, ncclDataType_t, ncclComm_t, cudaStream_t) = nullptr;
    ncclResult_t (*AllReduce)(const void *, void *, size_t, ncclDataType_t, ncclRedOp_t, ncclComm_t, cudaStream_t) = nullptr;
    ncclResult_t (*GroupStart)() = nullptr;
    ncclResult_t (*GroupEnd)() = nullptr;
    const char *(*GetErrorString)(ncclResult_t) = nullptr;
};
static NcclApi g_nccl;

static bool nccl_load()
{
    if (g_nccl.tried) return g_nccl.ok;
    g_nccl.tried = true;
    void *h = dlopen("libnccl.so.2", RTLD_NOW | RTLD_LOCAL);
    if (!h) h = dlopen("libnccl.so", RTLD_NOW | RTLD_LOCAL);
    if (!h) {
        g_nccl.why = std::string("cannot load libnccl.so.2: ") + dlerror();
        return false;
    }
    bool ok = true;
    auto sym = [&](auto &fn, const char *name) {
        fn = reinterpret_cast<std::remove_reference_t<decltype(fn)>>(dlsym(h, name));
        if (!fn) ok = false;
    };
    sym(g_nccl.GetUniqueId, "ncclGetUniqueId");
    sym(g_nccl.CommInitRankConfig, "ncclCommInitRankConfig");
    sym(g_nccl.CommGetAsyncError, "ncclCommGetAsyncError");
    sym(g_nccl.CommDestroy, "ncclCommDestroy");
    sym(g_nccl.CommAbort, "ncclCommAbort");
    sym(g_nccl.AllGather, "ncclAllGather");
    sym(g_nccl.AllReduce, "ncclAllReduce");
    sym(g_nccl.GroupStart, "ncclGroupStart");
    sym(g_nccl.GroupEnd, "ncclGroupEnd");
    sym(g_nccl.GetErrorString, "ncclGetErrorString");
    if (!ok) g_nccl.why = "libnccl.so.2 lacks an expected symbol";
    g_nccl.ok = ok;
    return ok;
}

// Ends the context's sharded state: the communicator destroyed (or aborted,
// which also ends its kernels still waiting on a peer), the exchange buffers
// freed once the context's own stream is idle.
static void shard_release(g4s_ctx *ctx, bool abort = false)
{
    if (ctx->nccl_comm && g_nccl.ok) {
        if (abort) g_nccl.CommAbort((ncclComm_t)ctx->nccl_comm);
        else g_nccl.CommDestroy((ncclComm_t)ctx->nccl_comm);
    }
    ctx->nccl_comm = nullptr;
    if (ctx->sh_send) cudaFree(ctx->sh_send);
    if (ctx->sh_recv) cudaFree(ctx->sh_recv);
    if (ctx->sh_off) cudaFree(ctx->sh_off);
    ctx->sh_send = ctx->sh_recv = nullptr;
    ctx->sh_off = nullptr;
    ctx->shard_world = 0;
}

// Polls a non-blocking communicator until its state leaves ncclInProgress, at
// most limit_ms of host time (*timed_out then set).  Returns the state, or the
// query's own error.
static ncclResult_t nccl_settle(ncclComm_t comm, int64_t limit_ms, bool *timed_out)
{
    const auto t0 = std::chrono::steady_clock::now();
    *timed_out = false;
    for (;;) {
        ncclResult_t st = ncclInProgress;
        const ncclResult_t r = g_nccl.CommGetAsyncError(comm, &st);
        if (r != ncclSuccess) return r;
        if (st != ncclInProgress) return st;
        const int64_t ms =
            std::chrono::duration_cast<std::chrono::milliseconds>(std::chrono::steady_clock::now() - t0).count();
        if (ms >= limit_ms) {
            *timed_out = true;
            return ncclInProgress;
        }
        std::this_thread::sleep_for(std::chrono::microseconds(100));
    }
}

// After a group of collectives on the context's communicator: a non-blocking
// communicator may still be enqueueing them (ncclInProgress); wait for that
// within the shard deadline, aborting the communicator when it passes.
static int32_t nccl_group_done(g4s_ctx *ctx, const char *who, const char *what, ncclResult_t r)
{
    if (r == ncclInProgress) {
        bool to = false;
        r = nccl_settle((ncclComm_t)ctx->nccl_comm, ctx->shard_timeout_ms, &to);
        if (to) {
            shard_release(ctx, true);
            return fail(ctx, G4S_ERR_TIMEOUT, "%s: %s not enqueued within %lld ms; communicator aborted", who, what,
                        (long long)ctx->shard_timeout_ms);
        }
    }
    if (r != ncclSuccess) {
        const char *why = g_nccl.GetErrorString(r);
        shard_release(ctx, true);
        return fail(ctx, G4S_ERR_NCCL, "%s: %s: %s; communicator aborted", who, what, why);
    }
    return G4S_OK;
}

// Per-row parameters into the launch arguments: a broadcast record travels in
// the kernel arguments; per-row records go through the pinned staging buffer
// (with fl32(1/T) computed here, the same IEEE division as on the device).
static int32_t stage_params(g4s_ctx *ctx, const char *who, const g4s_params *params, int32_t params_stride,
                            int rows, cudaStream_t s, RowParams &out)
{
    if (params_stride) {
        cudaStreamCaptureStatus cs = cudaStreamCaptureStatusNone;
        if (cudaStreamIsCapturing(s, &cs) != cudaSuccess || cs != cudaStreamCaptureStatusNone) {
            cudaGetLastError();
            return fail(ctx, G4S_ERR_STATE,
                        "%s: per-row params are staged through host memory, which a captured graph would read at "
                        "replay; capture calls with broadcast params (params_stride 0)", who);
        }
        // slot k's pinned copy may still feed the copy of the call PSLOTS calls ago
        const int k = ctx->params_slot;
        ctx->params_slot = (k + 1) % PSLOTS;
        if (ctx->params_ev_pending[k] && cudaEventSynchronize(ctx->params_ev[k]) != cudaSuccess)
            return fail(ctx, G4S_ERR_CUDA, "%s: waiting on an earlier params copy failed", who);
        const size_t slot_bytes = (size_t)ctx->max_rows * (sizeof(g4s_params) + sizeof(float) + sizeof(int32_t));
        g4s_params *hp = (g4s_params *)((char *)ctx->params_pinned + k * slot_bytes);
        g4s_params *dp = (g4s_params *)((char *)ctx->params_dev + k * slot_bytes);
        memcpy(hp, params, (size_t)rows * sizeof(g4s_params));
        float *inv_t = (float *)(hp + rows);
        for (int r = 0; r < rows; r++) {
            const float T = params[r].temperature;
            inv_t[r] = (T > 0.0f && T != 1.0f) ? 1.0f / T : 1.0f;
        }
        // launch order of the streaming top-K pass: its CTAs take longer the
        // larger the row's top_k, so the rows go by descending top_k (rows of
        // other paths last) and the short ones fill the last partial wave
        int32_t *ord = (int32_t *)(inv_t + rows);
        {
            int cnt[KMAX_ + 2] = {};
            auto bucket = [&](int r) {
                const int k = params[r].top_k;
                return (k > 0 && k <= KMAX_) ? KMAX_ - k : KMAX_ + 1;  // descending top_k
            };
            for (int r = 0; r < rows; r++) cnt[bucket(r)]++;
            int o = 0;
            for (int b = 0; b < KMAX_ + 2; b++) {
                const int c = cnt[b];
                cnt[b] = o;
                o += c;
            }
            for (int r = 0; r < rows; r++) ord[cnt[bucket(r)]++] = r;
        }
        if (cudaMemcpyAsync(dp, hp, (size_t)rows * (sizeof(g4s_params) + sizeof(float) + sizeof(int32_t)), cudaMemcpyHostToDevice, s) !=
                cudaSuccess ||
            cudaEventRecord(ctx->params_ev[k], s) != cudaSuccess) {
            cudaError_t e = cudaGetLastError();
            return fail(ctx, G4S_ERR_CUDA, "%s: params upload failed: %s", who, cudaGetErrorString(e));
        }
        ctx->params_ev_pending[k] = true;
        out.dev = dp;
        out.inv_t_dev = (const float *)(dp + rows);
        out.order_dev = (const int32_t *)(out.inv_t_dev + rows);
    } else {
        out.dev = nullptr;
        out.order_dev = nullptr;
        out.p0 = params[0];
        const float T = params[0].temperature;
        out.inv_t0 = (T > 0.0f && T != 1.0f) ? 1.0f / T : 1.0f;
    }
    return G4S_OK;
}

// Checks the rows of a sharded call: top-K rows need 0 < top_k <= 256 below
// both the slice and the vocabulary; rows with top_k <= 0 or >= the
// vocabulary take the full-vocabulary path.  Reports what the call holds.
struct ShardRows {
    bool any_draw = false, any_full = false, any_full_draw = false, any_topk = false;
};
static int32_t check_shard_rows(g4s_ctx *ctx, const char *who, const g4s_params *params, int32_t params_stride,
                                int rows, int slice_vocab, int vocab_total, ShardRows *sr)
{
    const int nparam = params_stride ? rows : 1;
    *sr = ShardRows();
    for (int r = 0; r < nparam; r++) {
        const g4s_params &p = params[r];
        if (p.temperature != p.temperature || p.top_p != p.top_p)
            return fail(ctx, G4S_ERR_ARG, "%s: NaN temperature/top_p in params[%d]", who, r);
        const bool draw = p.temperature > 0.0f;
        sr->any_draw |= draw;
        if (p.top_k <= 0 || p.top_k >= vocab_total) {
            sr->any_full = true;
            sr->any_full_draw |= draw;
            continue;
        }
        if (p.top_k > KMAX_ || (slice_vocab > 0 && p.top_k >= slice_vocab))
            return fail(ctx, G4S_ERR_ARG,
                        "%s: params[%d].top_k = %d; the sharded path takes top-K rows with top_k <= %d below the "
                        "slice (%d), or full-vocabulary rows (top_k <= 0 or >= %d)",
                        who, r, p.top_k, KMAX_, slice_vocab, vocab_total);
        sr->any_topk = true;
    }
    return G4S_OK;
}

// Set-up of a call's full-vocabulary rows: the softcap and weight tables the
// bf16 streaming kernels read (built once per softcap, resp. per (softcap,
// temperature)), the streaming grid and the item statistics.  Outside stream
// capture a table build is waited for, so calls on any stream may use it
// afterwards; a captured build is part of the graph and is not remembered
// (the next call outside the graph builds again).
static int32_t prepare_full_path(g4s_ctx *ctx, const char *who, SampleArgs &a, int dtype, bool vec, float softcap,
                                 const g4s_params *params, int32_t params_stride, cudaStream_t s)
{
    a.istat = ctx->istat;
    a.rowstat = ctx->rowstat;
    const bool use_tab = dtype == G4S_BF16 && vec && softcap > 0.0f && softcap <= SC_TABLE_MAX_CAP;
    cudaStreamCaptureStatus cs = cudaStreamCaptureStatusNone;
    if (use_tab && cudaStreamIsCapturing(s, &cs) != cudaSuccess) {
        cudaGetLastError();
        return fail(ctx, G4S_ERR_CUDA, "%s: cannot query the stream's capture state", who);
    }
    if (use_tab && ctx->sc_tab_cap != softcap) {
        cudaError_t te = launch_softcap_table(softcap, a.invcap, ctx->sc_tab, s);
        if (te == cudaSuccess && cs == cudaStreamCaptureStatusNone) te = cudaStreamSynchronize(s);
        if (te != cudaSuccess) return fail(ctx, G4S_ERR_CUDA, "%s: softcap table: %s", who, cudaGetErrorString(te));
        if (cs == cudaStreamCaptureStatusNone) ctx->sc_tab_cap = softcap;
    }
    a.sc_table = use_tab ? ctx->sc_tab : nullptr;
    // one temperature for every row that draws: the per-logit weight itself
    // comes from a table
    const float T0 = params[0].temperature;
    const float invt0 = (T0 > 0.0f && T0 != 1.0f) ? 1.0f / T0 : 1.0f;
    const bool use_etab = use_tab && params_stride == 0 && T0 > 0.0f && softcap * invt0 <= ETAB_MAX_CAP_OVER_T &&
                          (ctx->persist_etab > 0 || (ctx->persist_etab = full_etab_blocks_per_sm()) > 0);
    if (use_etab && (ctx->e_tab_cap != softcap || ctx->e_tab_invt != invt0)) {
        cudaError_t te = launch_etable(softcap, a.invcap, invt0, T0 != 1.0f, ctx->e_tab, nullptr, s);
        if (te == cudaSuccess && cs == cudaStreamCaptureStatusNone) te = cudaStreamSynchronize(s);
        if (te != cudaSuccess) return fail(ctx, G4S_ERR_CUDA, "%s: weight table: %s", who, cudaGetErrorString(te));
        if (cs == cudaStreamCaptureStatusNone) {
            ctx->e_tab_cap = softcap;
            ctx->e_tab_invt = invt0;
        }
    }
    a.e_table = use_etab ? ctx->e_tab : nullptr;
    int &bps = use_etab ? ctx->persist_etab : use_tab ? ctx->persist_tab : ctx->persist[dtype][vec ? 1 : 0];
    if (bps == 0) bps = full_stream_blocks_per_sm(dtype, vec, use_tab);
    a.persist_blocks = bps * ctx->sm_count;
    return G4S_OK;
}

extern "C" {

int32_t g4s_version(void) { return G4S_ABI_VERSION; }

void g4s_params_defaults(g4s_params *p)
{
    if (!p) return;
    p->temperature = 1.0f;
    p->top_k = 64;
    p->top_p = 0.95f;
    p->repetition_penalty = 1.0f;
}

const char *g4s_last_error(const g4s_ctx *ctx) { return ctx ? ctx->err.c_str() : g_create_err.c_str(); }

// error text of the context-free entry point (g4s_noalloc.cu), read with g4s_last_error(NULL)
int32_t g4s_noalloc_set_error(const char *msg)
{
    g_create_err = msg ? msg : "";
    return 0;
}

void *g4s_stream(g4s_ctx *ctx) { return ctx ? (void *)ctx->stream : nullptr; }

int64_t g4s_workspace_bytes(const g4s_ctx *ctx) { return ctx ? (int64_t)ctx->ws_bytes : 0; }

static int32_t alloc_host_staging(g4s_ctx *ctx)
{
    if (ctx->h_logits) return G4S_OK;
    const size_t lb = (size_t)ctx->max_rows * (size_t)ctx->max_vocab * 4u;
    if (cudaMalloc(&ctx->h_logits, lb) != cudaSuccess ||
        cudaMalloc((void **)&ctx->h_u, (size_t)ctx->max_rows * sizeof(double)) != cudaSuccess ||
        cudaMalloc((void **)&ctx->h_tok, (size_t)ctx->max_rows * sizeof(int32_t)) != cudaSuccess) {
        cudaGetLastError();
        return fail(ctx, G4S_ERR_NOMEM, "g4s: cannot allocate %zu bytes of host-form staging", lb);
    }
    return G4S_OK;
}

int32_t g4s_create(int32_t device, int32_t max_rows, int32_t max_vocab, uint32_t flags,
                   g4s_ctx **out_ctx)
{
    g_create_err.clear();
    if (!out_ctx) return fail(nullptr, G4S_ERR_ARG, "g4s_create: out_ctx is NULL");
    *out_ctx = nullptr;
    if (max_rows < 1 || max_vocab < 1)
        return fail(nullptr, G4S_ERR_ARG, "g4s_create: max_rows (%d) and max_vocab (%d) must be >= 1",
                    max_rows, max_vocab);
    if (ceil_div(max_vocab, 8192) > NCH_MAX_)
        return fail(nullptr, G4S_ERR_CAPACITY, "g4s_create: max_vocab %d above the supported %d",
                    max_vocab, 8192 * NCH_MAX_);
    int ndev = 0;
    cudaError_t ce = cudaGetDeviceCount(&ndev);
    if (ce != cudaSuccess || ndev == 0) {
        cudaGetLastError();
        return fail(nullptr, G4S_ERR_UNAVAILABLE, "g4s_create: no CUDA device (%s)",
                    ce != cudaSuccess ? cudaGetErrorString(ce) : "device count 0");
    }
    if (device < 0 || device >= ndev)
        return fail(nullptr, G4S_ERR_ARG, "g4s_create: device %d out of range [0, %d)", device, ndev);
    DeviceGuard guard(device);
    if (!guard.ok) return fail(nullptr, G4S_ERR_CUDA, "g4s_create: cudaSetDevice(%d) failed", device);
    int major = 0, minor = 0;
    cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, device);
    cudaDeviceGetAttribute(&minor, cudaDevAttrComputeCapabilityMinor, device);
    if (major != 10 || minor != 0)
        return fail(nullptr, G4S_ERR_UNAVAILABLE,
                    "g4s_create: device %d is sm_%d%d; this library is built for sm_100a (B200)", device,
                    major, minor);

    g4s_ctx *ctx = new g4s_ctx();
    ctx->device = device;
    ctx->max_rows = max_rows;
    ctx->max_vocab = max_vocab;
    ctx->flags = flags;
    cudaDeviceGetAttribute(&ctx->sm_count, cudaDevAttrMultiProcessorCount, device);
    ctx->cluster_ok = topk_cluster_available();

    // per-chunk lists: big chunks for every row, or small chunks for the few rows
    // that choose them
    const int64_t nch_big = ceil_div(max_vocab, 8192), nch_small = ceil_div(max_vocab, 2048);
    int64_t small_rows = ceil_div(2LL * ctx->sm_count, nch_big);
    if (small_rows > max_rows) small_rows = max_rows;
    int64_t lists = (int64_t)max_rows * nch_big;
    if (nch_small <= NCH_MAX_ && small_rows * nch_small > lists) lists = small_rows * nch_small;
    ctx->lists_cap = lists;

    auto align = [](size_t x) { return (x + 255u) & ~(size_t)255u; };
    size_t off = 0;
    const size_t o_cand = off; off = align(off + (size_t)lists * KMAX_ * sizeof(uint64_t));
    const size_t o_cnt = off; off = align(off + (size_t)lists * sizeof(int32_t));
    const size_t o_ct = off; off = align(off + (size_t)max_rows * sizeof(uint32_t));
    const int64_t item_min = std::min(full_item_logits(G4S_F32), full_item_logits(G4S_BF16));
    const int64_t items = (int64_t)max_rows * ceil_div(max_vocab, item_min);
    const size_t o_st = off; off = align(off + (size_t)items * sizeof(float4));
    const size_t o_rs = off; off = align(off + (size_t)max_rows * sizeof(RowStat));
    const size_t o_li = off; off = align(off + (size_t)LK_SLOTS * max_vocab * sizeof(int32_t));
    const size_t o_lv = off; off = align(off + (size_t)LK_SLOTS * max_vocab * sizeof(float));
    const size_t o_pd = off; off = align(off + (size_t)PSLOTS * max_rows * (sizeof(g4s_params) + sizeof(float) + sizeof(int32_t)));
    const size_t o_err = off; off = align(off + sizeof(int));
    const size_t o_tab = off; off = align(off + (size_t)SC_TABLE_BYTES);
    const size_t o_etab = off; off = align(off + (size_t)ETAB_TABLE_BYTES);
    const size_t o_stg = off; off = align(off + (size_t)max_rows * sizeof(ShardTarget));
    const size_t o_bst = off; off = align(off + (size_t)max_rows * beam_items(max_vocab) * sizeof(float4));
    const size_t o_pgc = off; off = align(off + (size_t)max_rows * sizeof(int4));
    const size_t o_pgn = off; off = align(off + sizeof(int));
    ctx->ws_bytes = off;
    if (cudaMalloc(&ctx->ws, off) != cudaSuccess) {
        cudaGetLastError();
        delete ctx;
        return fail(nullptr, G4S_ERR_NOMEM, "g4s_create: cannot allocate %zu bytes of workspace", off);
    }
    char *base = (char *)ctx->ws;
    ctx->cand = (uint64_t *)(base + o_cand);
    ctx->cand_cnt = (int32_t *)(base + o_cnt);
    ctx->counters_topk = (uint32_t *)(base + o_ct);
    ctx->istat = (float4 *)(base + o_st);
    ctx->rowstat = (RowStat *)(base + o_rs);
    ctx->lk_idx = (int32_t *)(base + o_li);
    ctx->lk_val = (float *)(base + o_lv);
    ctx->params_dev = (g4s_params *)(base + o_pd);
    ctx->dev_err = (int *)(base + o_err);
    ctx->sc_tab = (float *)(base + o_tab);
    ctx->e_tab = (float *)(base + o_etab);
    ctx->shard_tgt = (ShardTarget *)(base + o_stg);
    ctx->beam_stat = (float4 *)(base + o_bst);
    ctx->pg_copies = (int4 *)(base + o_pgc);
    ctx->pg_n_copies = (int *)(base + o_pgn);
    if (cudaMemset(ctx->ws, 0, off) != cudaSuccess ||
        cudaStreamCreateWithFlags(&ctx->stream, cudaStreamNonBlocking) != cudaSuccess ||
        cudaHostAlloc((void **)&ctx->params_pinned, (size_t)PSLOTS * max_rows * (sizeof(g4s_params) + sizeof(float) + sizeof(int32_t)),
                      cudaHostAllocDefault) != cudaSuccess ||
        !create_param_events(ctx)) {
        cudaGetLastError();
        g4s_destroy(ctx);
        return fail(nullptr, G4S_ERR_CUDA, "g4s_create: stream/event/pinned setup failed");
    }
    if (flags & G4S_FLAG_HOST_STAGING) {
        int32_t rc = alloc_host_staging(ctx);
        if (rc != G4S_OK) {
            std::string e = ctx->err;
            g4s_destroy(ctx);
            return fail(nullptr, rc, "%s", e.c_str());
        }
    }
    *out_ctx = ctx;
    return G4S_OK;
}

int32_t g4s_destroy(g4s_ctx *ctx)
{
    if (!ctx) return G4S_OK;
    DeviceGuard guard(ctx->device);
    if (ctx->nccl_comm && g_nccl.ok && ctx->stream && ctx->shard_ev &&
        cudaEventRecord(ctx->shard_ev, ctx->stream) == cudaSuccess) {
        // a sharded step still waiting on a peer ends by an abort after the
        // shard deadline, so that the synchronisation below returns
        const auto t0 = std::chrono::steady_clock::now();
        while (cudaEventQuery(ctx->shard_ev) == cudaErrorNotReady &&
               std::chrono::steady_clock::now() - t0 < std::chrono::milliseconds(ctx->shard_timeout_ms))
            std::this_thread::sleep_for(std::chrono::microseconds(200));
        if (cudaEventQuery(ctx->shard_ev) == cudaErrorNotReady) {
            g_nccl.CommAbort((ncclComm_t)ctx->nccl_comm);
            ctx->nccl_comm = nullptr;
        }
    }
    if (ctx->stream) cudaStreamSynchronize(ctx->stream);
    for (int k = 0; k < PSLOTS; k++)
        if (ctx->params_ev[k]) cudaEventDestroy(ctx->params_ev[k]);
    if (ctx->stream) cudaStreamDestroy(ctx->stream);
    if (ctx->params_pinned) cudaFreeHost(ctx->params_pinned);
    if (ctx->ws) cudaFree(ctx->ws);
    if (ctx->h_logits) cudaFree(ctx->h_logits);
    if (ctx->h_u) cudaFree(ctx->h_u);
    if (ctx->h_tok) cudaFree(ctx->h_tok);
    shard_release(ctx);
    if (ctx->shard_ev) cudaEventDestroy(ctx->shard_ev);
    if (ctx->lm_logits) cudaFree(ctx->lm_logits);
    if (ctx->lm_xh) cudaFree(ctx->lm_xh);
    if (ctx->lm_fused) cudaFree(ctx->lm_fused);
    delete ctx;
    return G4S_OK;
}

int32_t g4s_sample_ex(g4s_ctx *ctx, const void *logits, int32_t dtype, int32_t rows, int32_t vocab,
                      int64_t row_stride, const g4s_params *params, int32_t params_stride,
                      float softcap, const double *u, int32_t *out_tokens, const g4s_outputs *extra,
                      void *stream)
{
    if (!ctx) return fail(nullptr, G4S_ERR_ARG, "g4s_sample: ctx is NULL");
    if (!logits || !params || !out_tokens)
        return fail(ctx, G4S_ERR_ARG, "g4s_sample: logits, params and out_tokens must be non-NULL");
    if (dtype != G4S_F32 && dtype != G4S_BF16) return fail(ctx, G4S_ERR_ARG, "g4s_sample: bad dtype %d", dtype);
    if (rows < 1 || vocab < 1) return fail(ctx, G4S_ERR_ARG, "g4s_sample: rows (%d) and vocab (%d) must be >= 1", rows, vocab);
    if (rows > ctx->max_rows || vocab > ctx->max_vocab)
        return fail(ctx, G4S_ERR_CAPACITY, "g4s_sample: rows %d / vocab %d exceed the context (%d / %d)",
                    rows, vocab, ctx->max_rows, ctx->max_vocab);
    if (row_stride < vocab) return fail(ctx, G4S_ERR_ARG, "g4s_sample: row_stride %lld < vocab %d", (long long)row_stride, vocab);
    if (params_stride != 0 && params_stride != 1)
        return fail(ctx, G4S_ERR_ARG, "g4s_sample: params_stride must be 0 (broadcast) or 1 (per row)");

    // route rows by kind (host side: params are host memory)
    const int nparam = params_stride ? rows : 1;
    bool any_topk = false, any_full = false, any_large = false, any_draw = false;
    int max_k_small = 0;
    for (int r = 0; r < nparam; r++) {
        const g4s_params &p = params[r];
        if (p.temperature != p.temperature || p.top_p != p.top_p)
            return fail(ctx, G4S_ERR_ARG, "g4s_sample: NaN temperature/top_p in params[%d]", r);
        if (p.temperature > 0.0f) any_draw = true;
        if (p.top_k <= 0 || p.top_k >= vocab) any_full = true;
        else if (p.top_k <= KMAX_) { any_topk = true; max_k_small = p.top_k > max_k_small ? p.top_k : max_k_small; }
        else any_large = true;
    }
    if (any_draw && !u) return fail(ctx, G4S_ERR_ARG, "g4s_sample: u is NULL but a row has temperature > 0");
    g4s_outputs ex;
    memset(&ex, 0, sizeof(ex));
    if (extra) ex = *extra;
    if ((ex.cand_ids || ex.cand_probs) && ex.cand_stride < 1)
        return fail(ctx, G4S_ERR_ARG, "g4s_sample: cand_stride must be >= 1 when cand_ids/cand_probs are set");
    if ((ex.cand_ids || ex.cand_probs) && any_topk && ex.cand_stride < max_k_small)
        return fail(ctx, G4S_ERR_ARG, "g4s_sample: cand_stride %d < largest top_k %d", ex.cand_stride, max_k_small);

    // the context's device is current before the chunk choice: its occupancy
    // query and launch attributes are per device
    DeviceGuard guard(ctx->device);
    if (!guard.ok) return fail(ctx, G4S_ERR_CUDA, "g4s_sample: cannot select device %d", ctx->device);
    const int esize = dtype == G4S_F32 ? 4 : 2;
    const bool vec = ((uintptr_t)logits % 16u == 0) && (((int64_t)row_stride * esize) % 16 == 0);
    const int ept = choose_ept(ctx, rows, vocab);
    const TopkChunks tc = choose_topk_chunks(ctx, rows, vocab, vec);
    const int chunk = tc.chunk;
    const int nch = tc.nch;
    if (nch > NCH_MAX_ || (int64_t)rows * nch > ctx->lists_cap)
        return fail(ctx, G4S_ERR_CAPACITY, "g4s_sample: %d rows x %d chunks exceed the workspace", rows, nch);
    cudaStream_t s = stream ? (cudaStream_t)stream : ctx->stream;

    SampleArgs a;
    memset(&a, 0, sizeof(a));
    a.logits = logits;
    a.row_stride = row_stride;
    a.rows = rows;
    a.vocab = vocab;
    a.dtype = dtype;
    a.chunk = chunk;
    a.nch = nch;
    a.lk_slots = LK_SLOTS;
    a.softcap = softcap;
    a.invcap = softcap > 0.0f ? 1.0f / softcap : 0.0f;
    a.u = u;
    a.out_tokens = out_tokens;
    a.token_prob = ex.token_prob;
    a.row_flags = ex.row_flags;
    a.cand_ids = ex.cand_ids;
    a.cand_probs = ex.cand_probs;
    a.cand_stride = ex.cand_stride;
    a.full_probs = ex.full_probs;
    a.stream_only = (ex.phase_mask & G4S_PHASE_FULL_STREAM_ONLY) ? 1 : 0;
    a.cand = ctx->cand;
    a.cand_cnt = ctx->cand_cnt;
    a.counters_topk = ctx->counters_topk;
    a.err = ctx->dev_err;
    a.wait_limit = ctx->wait_limit;
    a.istat = ctx->istat;
    if (any_full) {
        const int32_t rc = prepare_full_path(ctx, "g4s_sample", a, dtype, vec, softcap, params, params_stride, s);
        if (rc != G4S_OK) return rc;
    }
    a.rowstat = ctx->rowstat;
    a.lk_idx = ctx->lk_idx;
    a.lk_val = ctx->lk_val;
    {
        const int32_t rc = stage_params(ctx, "g4s_sample", params, params_stride, rows, s, a.params);
        if (rc != G4S_OK) return rc;
    }

    cudaError_t e = cudaSuccess;
    // a few rows: one thread-block cluster per row (latency); else the chunked grid
    const bool use_cluster = ctx->cluster_ok && rows <= TOPK_CLUSTER_MAX_ROWS && vocab <= TOPK_CLUSTER_MAX_VOCAB &&
                             max_k_small <= TOPK_CLUSTER_KMAX;
    if (any_topk && e == cudaSuccess)
        e = use_cluster ? launch_topk_cluster(a, vec, s) : tc.stream ? launch_topk_stream(a, s) : launch_topk(a, ept, vec, s);
    if (any_full && e == cudaSuccess) e = launch_full(a, ept, vec, s);
    if (any_full && ex.full_probs && e == cudaSuccess) e = launch_full_probs(a, ept, vec, s);
    if (any_large && e == cudaSuccess) e = launch_largek(a, s);
    if (e != cudaSuccess) return fail(ctx, G4S_ERR_CUDA, "g4s_sample: launch failed: %s", cudaGetErrorString(e));
    return G4S_OK;
}

int32_t g4s_sample(g4s_ctx *ctx, const void *logits, int32_t dtype, int32_t rows, int32_t vocab,
                   int64_t row_stride, const g4s_params *params, int32_t params_stride, float softcap,
                   const double *u, int32_t *out_tokens, void *stream)
{
    return g4s_sample_ex(ctx, logits, dtype, rows, vocab, row_stride, params, params_stride, softcap,
                         u, out_tokens, nullptr, stream);
}

int32_t g4s_sample_host(g4s_ctx *ctx, const void *host_logits, int32_t dtype, int32_t rows,
                        int32_t vocab, int64_t row_stride, const g4s_params *params,
                        int32_t params_stride, float softcap, const double *host_u,
                        int32_t *host_tokens)
{
    if (!ctx) return fail(nullptr, G4S_ERR_ARG, "g4s_sample_host: ctx is NULL");
    if (!host_logits || !host_tokens || !params)
        return fail(ctx, G4S_ERR_ARG, "g4s_sample_host: host_logits, params and host_tokens must be non-NULL");
    if (dtype != G4S_F32 && dtype != G4S_BF16) return fail(ctx, G4S_ERR_ARG, "g4s_sample_host: bad dtype %d", dtype);
    if (rows < 1 || vocab < 1 || rows > ctx->max_rows || vocab > ctx->max_vocab || row_stride < vocab)
        return fail(ctx, G4S_ERR_ARG, "g4s_sample_host: bad shape rows=%d vocab=%d stride=%lld", rows,
                    vocab, (long long)row_stride);
    DeviceGuard guard(ctx->device);
    int32_t rc = alloc_host_staging(ctx);
    if (rc != G4S_OK) return rc;
    const size_t esize = dtype == G4S_F32 ? 4u : 2u;
    cudaStream_t s = ctx->stream;
    cudaError_t e = cudaMemcpy2DAsync(ctx->h_logits, (size_t)vocab * esize, host_logits,
                                      (size_t)row_stride * esize, (size_t)vocab * esize, (size_t)rows,
                                      cudaMemcpyHostToDevice, s);
    if (e == cudaSuccess && host_u)
        e = cudaMemcpyAsync(ctx->h_u, host_u, (size_t)rows * sizeof(double), cudaMemcpyHostToDevice, s);
    if (e != cudaSuccess) return fail(ctx, G4S_ERR_CUDA, "g4s_sample_host: upload failed: %s", cudaGetErrorString(e));
    rc = g4s_sample_ex(ctx, ctx->h_logits, dtype, rows, vocab, vocab, params, params_stride, softcap,
                       host_u ? ctx->h_u : nullptr, ctx->h_tok, nullptr, s);
    if (rc != G4S_OK) return rc;
    e = cudaMemcpyAsync(host_tokens, ctx->h_tok, (size_t)rows * sizeof(int32_t), cudaMemcpyDeviceToHost, s);
    if (e == cudaSuccess) e = cudaStreamSynchronize(s);
    if (e != cudaSuccess) return fail(ctx, G4S_ERR_CUDA, "g4s_sample_host: %s", cudaGetErrorString(e));
    return G4S_OK;
}

// ---------------------------------------------------------------------------
// LM head + sampling (config C4)
// ---------------------------------------------------------------------------
int32_t g4s_q4_repack(const uint8_t *blocks, int32_t vocab, int32_t hidden, uint8_t *nibbles, uint16_t *scales,
                      void *stream)
{
    if (!blocks || !nibbles || !scales) return fail(nullptr, G4S_ERR_ARG, "g4s_q4_repack: NULL buffer");
    if (vocab < 1 || hidden < 32 || hidden % 32)
        return fail(nullptr, G4S_ERR_ARG, "g4s_q4_repack: vocab %d / hidden %d (a multiple of 32)", vocab, hidden);
    const cudaError_t e = launch_q4_repack(blocks, vocab, hidden, nibbles, scales, (cudaStream_t)stream);
    if (e != cudaSuccess) return fail(nullptr, G4S_ERR_CUDA, "g4s_q4_repack: %s", cudaGetErrorString(e));
    return G4S_OK;
}

// The LM head with top-K selection in its epilogue: taken when the caller
// wants no logits and every row is a top-K row (0 < top_k <= KMAX, below the
// vocabulary) of a vocabulary of at least two waves of tiles; returns
// G4S_ERR_UNAVAILABLE (nothing launched, no error recorded) for other calls.
// Launches: activations to fp16 tiles; the LM head over the sample tiles (one
// per SM) into the sample buffer and its group maxima; per row the threshold
// and the sample's candidates; the LM head over the other tiles with the
// candidate epilogue; per row the exact top K and the sampling tail.  The
// middle three are a chain of programmatic dependents: the last one's CTAs
// take the SMs' free slots during the sample pass and wait for the
// thresholds only in their epilogue.
static int32_t lmhead_sample_fused(g4s_ctx *ctx, const char *who, const float *hidden, int rows, int H,
                                   const float *norm_weight, float norm_eps, const uint8_t *nibbles,
                                   const uint16_t *scales, int vocab, const g4s_params *params, int params_stride,
                                   float softcap, const double *u, int32_t *out_tokens, const g4s_outputs *extra,
                                   cudaStream_t s)
{
    g4s_outputs ex;
    memset(&ex, 0, sizeof(ex));
    if (extra) ex = *extra;
    const int ntiles = (vocab + LMHEAD_TILE - 1) / LMHEAD_TILE;
    const int nA = ctx->sm_count;
    if (ex.full_probs || (ex.phase_mask & G4S_PHASE_LMHEAD_UNFUSED) || ntiles < 2 * nA || nA * LMHEAD_TILE / 32 > 2048)
        return G4S_ERR_UNAVAILABLE;
    bool any_draw = false;
    int max_k = 0;
    for (int r = 0; r < (params_stride ? rows : 1); r++) {
        const g4s_params &p = params[r];
        if (p.temperature != p.temperature || p.top_p != p.top_p)
            return fail(ctx, G4S_ERR_ARG, "%s: NaN temperature/top_p in params[%d]", who, r);
        if (p.top_k <= 0 || p.top_k > KMAX_ || p.top_k >= vocab) return G4S_ERR_UNAVAILABLE;
        any_draw |= p.temperature > 0.0f;
        max_k = std::max(max_k, (int)p.top_k);
    }
    if (any_draw && !u) return fail(ctx, G4S_ERR_ARG, "%s: u is NULL but a row has temperature > 0", who);
    if ((ex.cand_ids || ex.cand_probs) && ex.cand_stride < max_k)
        return fail(ctx, G4S_ERR_ARG, "%s: cand_stride %d < largest top_k %d", who, ex.cand_stride, max_k);
    // workspace: candidates [rows][vocab] (a row can never hold more), counts,
    // thresholds, sample logits [rows][ns]
    const int ns = nA * LMHEAD_TILE;
    auto al = [](size_t x) { return (x + 255u) & ~(size_t)255u; };
    const size_t o_cnt = al((size_t)rows * vocab * sizeof(uint64_t));
    const size_t o_thr = o_cnt + al((size_t)rows * sizeof(int32_t));
    const size_t o_smp = o_thr + al((size_t)rows * sizeof(uint64_t));
    const size_t o_gmx = o_smp + al((size_t)rows * ns * sizeof(float));
    const size_t need = o_gmx + al((size_t)rows * (ns / 32) * sizeof(uint32_t));
    if (ctx->lm_fused_n < need) {
        if (ctx->lm_fused) cudaFree(ctx->lm_fused);
        ctx->lm_fused = nullptr;
        ctx->lm_fused_n = 0;
        if (cudaMalloc(&ctx->lm_fused, need) != cudaSuccess) {
            cudaGetLastError();
            return fail(ctx, G4S_ERR_NOMEM, "%s: cannot allocate %zu bytes of candidate lists", who, need);
        }
        ctx->lm_fused_n = need;
    }
    char *base = (char *)ctx->lm_fused;
    LmCand c;
    c.cand = (uint64_t *)base;
    c.cnt = (int32_t *)(base + o_cnt);
    c.thr = (uint64_t *)(base + o_thr);
    c.cap = vocab;
    c.sample = (float *)(base + o_smp);
    c.gmax = (uint32_t *)(base + o_gmx);
    c.ns = ns;
    SampleArgs a;
    memset(&a, 0, sizeof(a));
    a.rows = rows;
    a.vocab = vocab;
    a.dtype = G4S_F32;
    a.softcap = softcap;
    a.invcap = softcap > 0.0f ? 1.0f / softcap : 0.0f;
    a.u = u;
    a.out_tokens = out_tokens;
    a.token_prob = ex.token_prob;
    a.row_flags = ex.row_flags;
    a.cand_ids = ex.cand_ids;
    a.cand_probs = ex.cand_probs;
    a.cand_stride = ex.cand_stride;
    a.err = ctx->dev_err;
    int32_t rc = stage_params(ctx, who, params, params_stride, rows, s, a.params);
    if (rc != G4S_OK) return rc;
    __half *xh = (__half *)ctx->lm_xh;
    cudaError_t e = launch_lmhead_prep(hidden, rows, H, norm_weight, norm_eps, xh, s);
    if (e == cudaSuccess)
        e = launch_lmhead_part(xh, rows, H, nibbles, scales, vocab, 0, nA, nullptr, 0, 1, &c, ctx->dev_err, s);
    if (e == cudaSuccess) e = launch_lm_threshold(a, c, s);
    if (e == cudaSuccess)
        e = launch_lmhead_part(xh, rows, H, nibbles, scales, vocab, nA, ntiles - nA, nullptr, 0, 2, &c, ctx->dev_err,
                               s);
    if (e == cudaSuccess) e = launch_lm_finish(a, c, s);
    if (e != cudaSuccess) return fail(ctx, G4S_ERR_CUDA, "%s: launch failed: %s", who, cudaGetErrorString(e));
    return G4S_OK;
}

int32_t g4s_lmhead_sample(g4s_ctx *ctx, const float *hidden, int32_t rows, int32_t hidden_size,
                          const float *norm_weight, float norm_eps, const uint8_t *nibbles, const uint16_t *scales,
                          int32_t vocab, const g4s_params *params, int32_t params_stride, float softcap,
                          const double *u, int32_t *out_tokens, const g4s_outputs *extra, float *out_logits,
                          void *stream)
{
    static const char *who = "g4s_lmhead_sample";
    if (!ctx) return fail(nullptr, G4S_ERR_ARG, "%s: ctx is NULL", who);
    if (!hidden || !nibbles || !scales || !params || !out_tokens)
        return fail(ctx, G4S_ERR_ARG, "%s: hidden, nibbles, scales, params and out_tokens must be non-NULL", who);
    if (rows < 1 || rows > LMHEAD_MAX_ROWS || rows > ctx->max_rows)
        return fail(ctx, G4S_ERR_CAPACITY, "%s: rows %d outside [1, %d]", who, rows,
                    std::min(LMHEAD_MAX_ROWS, ctx->max_rows));
    if (hidden_size < 128 || hidden_size % 128)
        return fail(ctx, G4S_ERR_ARG, "%s: hidden %d must be a positive multiple of 128", who, hidden_size);
    if (vocab < 8 || vocab % 8 || vocab > ctx->max_vocab)
        return fail(ctx, G4S_ERR_ARG, "%s: vocab %d must be a multiple of 8 within max_vocab %d", who, vocab,
                    ctx->max_vocab);
    DeviceGuard guard(ctx->device);
    if (!guard.ok) return fail(ctx, G4S_ERR_CUDA, "%s: cannot select device %d", who, ctx->device);
    cudaStream_t s = stream ? (cudaStream_t)stream : ctx->stream;
    float *logits = out_logits;
    const size_t need_x = (size_t)LMHEAD_MAX_ROWS * hidden_size;
    if (ctx->lm_xh_n < need_x) {
        if (ctx->lm_xh) cudaFree(ctx->lm_xh);
        ctx->lm_xh = nullptr;
        ctx->lm_xh_n = 0;
        if (cudaMalloc(&ctx->lm_xh, need_x * sizeof(uint16_t)) != cudaSuccess) {
            cudaGetLastError();
            return fail(ctx, G4S_ERR_NOMEM, "%s: cannot allocate the fp16 hidden buffer", who);
        }
        ctx->lm_xh_n = need_x;
    }
    if (!logits) {
        int32_t rc = lmhead_sample_fused(ctx, who, hidden, rows, hidden_size, norm_weight, norm_eps, nibbles, scales,
                                         vocab, params, params_stride, softcap, u, out_tokens, extra, s);
        if (rc != G4S_ERR_UNAVAILABLE) return rc;  // else: a call the fused path does not take
        const size_t need_l = (size_t)rows * vocab;
        if (ctx->lm_logits_n < need_l) {
            if (ctx->lm_logits) cudaFree(ctx->lm_logits);
            ctx->lm_logits = nullptr;
            ctx->lm_logits_n = 0;
            if (cudaMalloc(&ctx->lm_logits, need_l * sizeof(float)) != cudaSuccess) {
                cudaGetLastError();
                return fail(ctx, G4S_ERR_NOMEM, "%s: cannot allocate %zu bytes of logits", who, need_l * sizeof(float));
            }
            ctx->lm_logits_n = need_l;
        }
        logits = ctx->lm_logits;
    }
    const cudaError_t e = launch_lmhead(hidden, rows, hidden_size, norm_weight, norm_eps, nibbles, scales, vocab,
                                        (__half *)ctx->lm_xh, logits, ctx->dev_err, s);
    if (e != cudaSuccess) return fail(ctx, G4S_ERR_CUDA, "%s: launch failed: %s", who, cudaGetErrorString(e));
    return g4s_sample_ex(ctx, logits, G4S_F32, rows, vocab, vocab, params, params_stride, softcap, u, out_tokens,
                         extra, s);
}

int32_t g4s_set_wait_limit(g4s_ctx *ctx, int64_t polls)
{
    if (!ctx) return fail(nullptr, G4S_ERR_ARG, "g4s_set_wait_limit: ctx is NULL");
    if (polls < 0) return fail(ctx, G4S_ERR_ARG, "g4s_set_wait_limit: polls %lld < 0", (long long)polls);
    ctx->wait_limit = polls;
    return G4S_OK;
}

int32_t g4s_device_status(g4s_ctx *ctx)
{
    if (!ctx) return fail(nullptr, G4S_ERR_ARG, "g4s_device_status: ctx is NULL");
    if (!ctx->dev_err) return G4S_OK;
    DeviceGuard guard(ctx->device);
    int v = 0;
    if (cudaDeviceSynchronize() != cudaSuccess ||
        cudaMemcpy(&v, ctx->dev_err, sizeof(int), cudaMemcpyDeviceToHost) != cudaSuccess) {
        cudaError_t e = cudaGetLastError();
        return fail(ctx, G4S_ERR_CUDA, "g4s_device_status: %s", cudaGetErrorString(e));
    }
    if (v) {
        cudaMemset(ctx->dev_err, 0, sizeof(int));
        return fail(ctx, G4S_ERR_TIMEOUT, "g4s_device_status: a kernel's bounded wait ran out (its results are invalid)");
    }
    return G4S_OK;
}

// ---------------------------------------------------------------------------
// vocabulary-sharded mode
// ---------------------------------------------------------------------------
// The two phases of the sharded mode; `staged` (nullable) is the call's per-row
// params already on the device (g4s_shard_sample stages them once for both).
static int32_t shard_lists_core(g4s_ctx *ctx, const void *logits, int32_t dtype, int32_t rows, int32_t slice_vocab,
                                int64_t row_stride, int32_t id_offset, int32_t vocab_total, const g4s_params *params,
                                int32_t params_stride, float softcap, uint64_t *out_lists, int32_t *out_counts,
                                void *stream, const RowParams *staged, const int32_t *list_off = nullptr)
{
    static const char *who = "g4s_shard_lists";
    if (!ctx) return fail(nullptr, G4S_ERR_ARG, "%s: ctx is NULL", who);
    if (!logits || !params || !out_lists || !out_counts)
        return fail(ctx, G4S_ERR_ARG, "%s: logits, params, out_lists and out_counts must be non-NULL", who);
    if (dtype != G4S_F32 && dtype != G4S_BF16) return fail(ctx, G4S_ERR_ARG, "%s: bad dtype %d", who, dtype);
    if (rows < 1 || slice_vocab < 1 || rows > ctx->max_rows || slice_vocab > ctx->max_vocab)
        return fail(ctx, G4S_ERR_CAPACITY, "%s: rows %d / slice %d outside the context (%d / %d)", who, rows,
                    slice_vocab, ctx->max_rows, ctx->max_vocab);
    if (row_stride < slice_vocab) return fail(ctx, G4S_ERR_ARG, "%s: row_stride < slice_vocab", who);
    if (id_offset < 0 || vocab_total < 1 || (int64_t)id_offset + slice_vocab > vocab_total)
        return fail(ctx, G4S_ERR_ARG, "%s: slice [%d, %lld) outside the vocabulary %d", who, id_offset,
                    (long long)id_offset + slice_vocab, vocab_total);
    if (params_stride != 0 && params_stride != 1)
        return fail(ctx, G4S_ERR_ARG, "%s: params_stride must be 0 or 1", who);
    ShardRows sr;
    int32_t rc = check_shard_rows(ctx, who, params, params_stride, rows, slice_vocab, vocab_total, &sr);
    if (rc != G4S_OK) return rc;
    DeviceGuard guard(ctx->device);
    if (!guard.ok) return fail(ctx, G4S_ERR_CUDA, "%s: cannot select device %d", who, ctx->device);
    const int esize = dtype == G4S_F32 ? 4 : 2;
    const bool vec = ((uintptr_t)logits % 16u == 0) && (((int64_t)row_stride * esize) % 16 == 0);
    const int ept = choose_ept(ctx, rows, slice_vocab);
    const TopkChunks tc = choose_topk_chunks(ctx, rows, slice_vocab, vec);
    const int nch = tc.nch;
    if (nch > NCH_MAX_ || (int64_t)rows * nch > ctx->lists_cap)
        return fail(ctx, G4S_ERR_CAPACITY, "%s: %d rows x %d chunks exceed the workspace", who, rows, nch);
    cudaStream_t s = stream ? (cudaStream_t)stream : ctx->stream;
    SampleArgs a;
    memset(&a, 0, sizeof(a));
    a.logits = logits;
    a.row_stride = row_stride;
    a.rows = rows;
    a.vocab = slice_vocab;
    a.dtype = dtype;
    a.chunk = tc.chunk;
    a.nch = nch;
    a.cand = ctx->cand;
    a.cand_cnt = ctx->cand_cnt;
    a.counters_topk = ctx->counters_topk;
    a.err = ctx->dev_err;
    a.wait_limit = ctx->wait_limit;
    a.id_offset = id_offset;
    a.list_out = out_lists;
    a.list_cnt = out_counts;
    a.list_off = list_off;
    a.softcap = softcap;
    a.invcap = softcap > 0.0f ? 1.0f / softcap : 0.0f;
    if (staged) a.params = *staged;
    else if ((rc = stage_params(ctx, who, params, params_stride, rows, s, a.params)) != G4S_OK) return rc;
    cudaError_t e = cudaSuccess;
    if (sr.any_full) {
        // full-vocabulary rows: the streaming pass over the slice, then each
        // row's slice summary into its list slot (the item statistics stay in
        // the context for g4s_shard_resolve)
        if ((rc = prepare_full_path(ctx, who, a, dtype, vec, softcap, params, params_stride, s)) != G4S_OK) return rc;
        SampleArgs af = a;
        af.stream_only = 1;
        e = launch_full(af, ept, vec, s);
        af.shard_mode = 1;
        if (e == cudaSuccess) e = launch_full_combine(af, vec, s);
    }
    if (sr.any_topk && e == cudaSuccess) e = tc.stream ? launch_topk_stream(a, s) : launch_topk(a, ept, vec, s);
    if (e != cudaSuccess) return fail(ctx, G4S_ERR_CUDA, "%s: launch failed: %s", who, cudaGetErrorString(e));
    return G4S_OK;
}

static int32_t shard_merge_core(g4s_ctx *ctx, const uint64_t *lists, const int32_t *counts, int32_t world,
                                int32_t rows, int32_t vocab_total, const g4s_params *params, int32_t params_stride,
                                float softcap, const double *u, int32_t *out_tokens, const g4s_outputs *extra,
                                void *stream, const RowParams *staged, const int32_t *list_off = nullptr,
                                int64_t list_total = 0)
{
    static const char *who = "g4s_shard_merge";
    if (!ctx) return fail(nullptr, G4S_ERR_ARG, "%s: ctx is NULL", who);
    if (!lists || !counts || !params || !out_tokens)
        return fail(ctx, G4S_ERR_ARG, "%s: lists, counts, params and out_tokens must be non-NULL", who);
    if (world < 1 || world > NCH_MAX_) return fail(ctx, G4S_ERR_ARG, "%s: world %d outside [1, %d]", who, world, NCH_MAX_);
    if (rows < 1 || rows > ctx->max_rows) return fail(ctx, G4S_ERR_CAPACITY, "%s: rows %d outside [1, %d]", who, rows, ctx->max_rows);
    if (params_stride != 0 && params_stride != 1)
        return fail(ctx, G4S_ERR_ARG, "%s: params_stride must be 0 or 1", who);
    ShardRows sr;
    int32_t rc = check_shard_rows(ctx, who, params, params_stride, rows, 0, vocab_total, &sr);
    if (rc != G4S_OK) return rc;
    if (sr.any_draw && !u) return fail(ctx, G4S_ERR_ARG, "%s: u is NULL but a row has temperature > 0", who);
    g4s_outputs ex;
    memset(&ex, 0, sizeof(ex));
    if (extra) ex = *extra;
    int max_k = 0;
    for (int r = 0; r < (params_stride ? rows : 1); r++) max_k = params[r].top_k > max_k ? params[r].top_k : max_k;
    if ((ex.cand_ids || ex.cand_probs) && ex.cand_stride < max_k)
        return fail(ctx, G4S_ERR_ARG, "%s: cand_stride %d < largest top_k %d", who, ex.cand_stride, max_k);
    DeviceGuard guard(ctx->device);
    if (!guard.ok) return fail(ctx, G4S_ERR_CUDA, "%s: cannot select device %d", who, ctx->device);
    cudaStream_t s = stream ? (cudaStream_t)stream : ctx->stream;
    SampleArgs a;
    memset(&a, 0, sizeof(a));
    a.rows = rows;
    a.vocab = vocab_total;
    a.softcap = softcap;
    a.invcap = softcap > 0.0f ? 1.0f / softcap : 0.0f;
    a.u = u;
    a.out_tokens = out_tokens;
    a.token_prob = ex.token_prob;
    a.row_flags = ex.row_flags;
    a.cand_ids = ex.cand_ids;
    a.cand_probs = ex.cand_probs;
    a.cand_stride = ex.cand_stride;
    a.glists = lists;
    a.gcnts = counts;
    a.gworld = world;
    a.list_off = list_off;
    a.list_total = list_total;
    a.shard_tgt = ctx->shard_tgt;
    if (staged) a.params = *staged;
    else if ((rc = stage_params(ctx, who, params, params_stride, rows, s, a.params)) != G4S_OK) return rc;
    cudaError_t e = launch_shard_merge(a, s);
    if (e != cudaSuccess) return fail(ctx, G4S_ERR_CUDA, "%s: launch failed: %s", who, cudaGetErrorString(e));
    return G4S_OK;
}

int32_t g4s_shard_lists(g4s_ctx *ctx, const void *logits, int32_t dtype, int32_t rows, int32_t slice_vocab,
                        int64_t row_stride, int32_t id_offset, int32_t vocab_total, const g4s_params *params,
                        int32_t params_stride, float softcap, uint64_t *out_lists, int32_t *out_counts, void *stream)
{
    return shard_lists_core(ctx, logits, dtype, rows, slice_vocab, row_stride, id_offset, vocab_total, params,
                            params_stride, softcap, out_lists, out_counts, stream, nullptr);
}

// The full-vocabulary draws shard_tgt assigns to this rank (after
// g4s_shard_merge on the same context): the crossing item among this slice's
// item statistics (from g4s_shard_lists on the same context), rescanned from
// the slice's logits.
static int32_t shard_resolve_core(g4s_ctx *ctx, const void *logits, int32_t dtype, int32_t rows, int32_t slice_vocab,
                                  int64_t row_stride, int32_t id_offset, int32_t rank, const g4s_params *params,
                                  int32_t params_stride, float softcap, const double *u, int32_t *out_tokens,
                                  const g4s_outputs *extra, void *stream, const RowParams *staged)
{
    static const char *who = "g4s_shard_resolve";
    if (!ctx) return fail(nullptr, G4S_ERR_ARG, "%s: ctx is NULL", who);
    if (!logits || !params || !out_tokens || !u)
        return fail(ctx, G4S_ERR_ARG, "%s: logits, params, u and out_tokens must be non-NULL", who);
    if (dtype != G4S_F32 && dtype != G4S_BF16) return fail(ctx, G4S_ERR_ARG, "%s: bad dtype %d", who, dtype);
    if (rows < 1 || slice_vocab < 1 || rows > ctx->max_rows || slice_vocab > ctx->max_vocab || row_stride < slice_vocab)
        return fail(ctx, G4S_ERR_CAPACITY, "%s: rows %d / slice %d outside the context (%d / %d)", who, rows,
                    slice_vocab, ctx->max_rows, ctx->max_vocab);
    if (params_stride != 0 && params_stride != 1)
        return fail(ctx, G4S_ERR_ARG, "%s: params_stride must be 0 or 1", who);
    DeviceGuard guard(ctx->device);
    if (!guard.ok) return fail(ctx, G4S_ERR_CUDA, "%s: cannot select device %d", who, ctx->device);
    cudaStream_t s = stream ? (cudaStream_t)stream : ctx->stream;
    const int esize = dtype == G4S_F32 ? 4 : 2;
    const bool vec = ((uintptr_t)logits % 16u == 0) && (((int64_t)row_stride * esize) % 16 == 0);
    g4s_outputs ex;
    memset(&ex, 0, sizeof(ex));
    if (extra) ex = *extra;
    SampleArgs a;
    memset(&a, 0, sizeof(a));
    a.logits = logits;
    a.row_stride = row_stride;
    a.rows = rows;
    a.vocab = slice_vocab;
    a.dtype = dtype;
    a.softcap = softcap;
    a.invcap = softcap > 0.0f ? 1.0f / softcap : 0.0f;
    a.u = u;
    a.out_tokens = out_tokens;
    a.token_prob = ex.token_prob;
    a.row_flags = ex.row_flags;
    a.id_offset = id_offset;
    a.istat = ctx->istat;
    a.rowstat = ctx->rowstat;
    a.shard_tgt = ctx->shard_tgt;
    a.shard_mode = 2;
    a.shard_rank = rank;
    int32_t rc;
    if (staged) a.params = *staged;
    else if ((rc = stage_params(ctx, who, params, params_stride, rows, s, a.params)) != G4S_OK) return rc;
    const cudaError_t e = launch_full_combine(a, vec, s);
    if (e != cudaSuccess) return fail(ctx, G4S_ERR_CUDA, "%s: launch failed: %s", who, cudaGetErrorString(e));
    return G4S_OK;
}

int32_t g4s_shard_resolve(g4s_ctx *ctx, const void *logits_slice, int32_t dtype, int32_t rows, int32_t slice_vocab,
                          int64_t row_stride, int32_t id_offset, int32_t rank, const g4s_params *params,
                          int32_t params_stride, float softcap, const double *u, int32_t *out_tokens,
                          const g4s_outputs *extra, void *stream)
{
    return shard_resolve_core(ctx, logits_slice, dtype, rows, slice_vocab, row_stride, id_offset, rank, params,
                              params_stride, softcap, u, out_tokens, extra, stream, nullptr);
}

int32_t g4s_shard_merge(g4s_ctx *ctx, const uint64_t *lists, const int32_t *counts, int32_t world, int32_t rows,
                        int32_t vocab_total, const g4s_params *params, int32_t params_stride, float softcap,
                        const double *u, int32_t *out_tokens, const g4s_outputs *extra, void *stream)
{
    return shard_merge_core(ctx, lists, counts, world, rows, vocab_total, params, params_stride, softcap, u, out_tokens,
                            extra, stream, nullptr);
}

int32_t g4s_shard_unique_id(uint8_t *uid)
{
    if (!uid) return fail(nullptr, G4S_ERR_ARG, "g4s_shard_unique_id: uid is NULL");
    if (!nccl_load()) return fail(nullptr, G4S_ERR_UNAVAILABLE, "g4s_shard_unique_id: %s", g_nccl.why.c_str());
    static_assert(sizeof(ncclUniqueId) == G4S_SHARD_UID_BYTES, "NCCL unique id size");
    ncclUniqueId id;
    const ncclResult_t r = g_nccl.GetUniqueId(&id);
    if (r != ncclSuccess) return fail(nullptr, G4S_ERR_NCCL, "ncclGetUniqueId: %s", g_nccl.GetErrorString(r));
    memcpy(uid, &id, sizeof(id));
    return G4S_OK;
}

int32_t g4s_shard_init(g4s_ctx *ctx, int32_t world, int32_t rank, int32_t vocab_total, const uint8_t *uid)
{
    static const char *who = "g4s_shard_init";
    if (!ctx) return fail(nullptr, G4S_ERR_ARG, "%s: ctx is NULL", who);
    if (!uid || world < 1 || world > 64 || rank < 0 || rank >= world || vocab_total < world)
        return fail(ctx, G4S_ERR_ARG, "%s: bad world %d / rank %d / vocab %d", who, world, rank, vocab_total);
    const int slice = (int)ceil_div(vocab_total, world);
    if (slice > ctx->max_vocab)
        return fail(ctx, G4S_ERR_CAPACITY, "%s: slice %d exceeds the context's max_vocab %d", who, slice, ctx->max_vocab);
    if (ctx->nccl_comm) return fail(ctx, G4S_ERR_STATE, "%s: the context is already sharded", who);
    if (ctx->sh_send || ctx->sh_recv) shard_release(ctx);  // buffers kept by an abort whose stream was busy
    if (!nccl_load()) return fail(ctx, G4S_ERR_UNAVAILABLE, "%s: %s", who, g_nccl.why.c_str());
    DeviceGuard guard(ctx->device);
    if (!guard.ok) return fail(ctx, G4S_ERR_CUDA, "%s: cannot select device %d", who, ctx->device);
    const size_t per_rank = (size_t)ctx->max_rows * (KMAX_ + 1) * sizeof(uint64_t);
    if (cudaMalloc(&ctx->sh_send, per_rank) != cudaSuccess ||
        cudaMalloc(&ctx->sh_recv, per_rank * (size_t)world) != cudaSuccess ||
        cudaMalloc(&ctx->sh_off, (size_t)ctx->max_rows * sizeof(int32_t)) != cudaSuccess) {
        cudaGetLastError();
        shard_release(ctx);
        return fail(ctx, G4S_ERR_NOMEM, "%s: cannot allocate the exchange buffers", who);
    }
    if (!ctx->shard_ev && cudaEventCreateWithFlags(&ctx->shard_ev, cudaEventDisableTiming) != cudaSuccess) {
        cudaGetLastError();
        shard_release(ctx);
        return fail(ctx, G4S_ERR_CUDA, "%s: cannot create the wait event", who);
    }
    ncclUniqueId id;
    memcpy(&id, uid, sizeof(id));
    // non-blocking communicator: the rendezvous runs in NCCL's threads while
    // this thread polls it against the deadline, so a rank that never joins
    // ends the call with G4S_ERR_TIMEOUT instead of blocking it for good
    ncclConfig_t cfg = NCCL_CONFIG_INITIALIZER;
    cfg.blocking = 0;
    ncclComm_t comm = nullptr;
    ncclResult_t r = g_nccl.CommInitRankConfig(&comm, world, id, rank, &cfg);
    if (r != ncclSuccess && r != ncclInProgress) {
        if (comm) g_nccl.CommAbort(comm);
        shard_release(ctx);
        return fail(ctx, G4S_ERR_NCCL, "%s: ncclCommInitRankConfig: %s", who, g_nccl.GetErrorString(r));
    }
    bool to = false;
    r = nccl_settle(comm, ctx->shard_timeout_ms, &to);
    if (to || r != ncclSuccess) {
        g_nccl.CommAbort(comm);
        shard_release(ctx);
        if (to)
            return fail(ctx, G4S_ERR_TIMEOUT, "%s: the %d ranks did not meet within %lld ms (a rank did not join)", who,
                        world, (long long)ctx->shard_timeout_ms);
        return fail(ctx, G4S_ERR_NCCL, "%s: communicator set-up: %s", who, g_nccl.GetErrorString(r));
    }
    ctx->nccl_comm = comm;
    ctx->shard_world = world;
    ctx->shard_rank = rank;
    ctx->shard_vocab = vocab_total;
    ctx->shard_slice = slice;
    return G4S_OK;
}

int32_t g4s_shard_sample(g4s_ctx *ctx, const void *logits_slice, int32_t dtype, int32_t rows, int64_t row_stride,
                         const g4s_params *params, int32_t params_stride, float softcap, const double *u,
                         int32_t *out_tokens, const g4s_outputs *extra, void *stream)
{
    static const char *who = "g4s_shard_sample";
    if (!ctx) return fail(nullptr, G4S_ERR_ARG, "%s: ctx is NULL", who);
    if (!ctx->nccl_comm) return fail(ctx, G4S_ERR_STATE, "%s: call g4s_shard_init first", who);
    const int W = ctx->shard_world, Vs = ctx->shard_slice;
    const int off = ctx->shard_rank * Vs;
    const int n = std::min(Vs, ctx->shard_vocab - off);
    if (rows < 1 || rows > ctx->max_rows) return fail(ctx, G4S_ERR_CAPACITY, "%s: rows %d outside [1, %d]", who, rows, ctx->max_rows);
    cudaStream_t s = stream ? (cudaStream_t)stream : ctx->stream;
    uint64_t *send = ctx->sh_send;
    int32_t *send_cnt = (int32_t *)(ctx->sh_send + (size_t)ctx->max_rows * KMAX_);
    uint64_t *recv = ctx->sh_recv;
    int32_t *recv_cnt = (int32_t *)(ctx->sh_recv + (size_t)W * ctx->max_rows * KMAX_);
    if (!params || (params_stride != 0 && params_stride != 1))
        return fail(ctx, G4S_ERR_ARG, "%s: params must be non-NULL, params_stride 0 or 1", who);
    ShardRows sr;
    int32_t rc = check_shard_rows(ctx, who, params, params_stride, rows, n, ctx->shard_vocab, &sr);
    if (rc != G4S_OK) return rc;
    DeviceGuard guard(ctx->device);
    if (!guard.ok) return fail(ctx, G4S_ERR_CUDA, "%s: cannot select device %d", who, ctx->device);
    // per-row params go to the device once for both phases
    RowParams rp;
    memset(&rp, 0, sizeof(rp));
    if ((rc = stage_params(ctx, who, params, params_stride, rows, s, rp)) != G4S_OK) return rc;
    // the exchange carries each row's own slots (its top_k; 2 for a
    // full-vocabulary row's summary) packed back to back: every rank computes
    // the same offsets from the same params
    int64_t P = 0;
    for (int r = 0; r < rows; r++) P += shard_slots(params[params_stride ? r : 0].top_k, ctx->shard_vocab);
    {
        SampleArgs ao;
        memset(&ao, 0, sizeof(ao));
        ao.rows = rows;
        ao.vocab = ctx->shard_vocab;
        ao.params = rp;
        const cudaError_t e = launch_shard_offsets(ao, ctx->sh_off, s);
        if (e != cudaSuccess) return fail(ctx, G4S_ERR_CUDA, "%s: launch failed: %s", who, cudaGetErrorString(e));
    }
    rc = shard_lists_core(ctx, logits_slice, dtype, rows, n, row_stride, off, ctx->shard_vocab, params, params_stride,
                          softcap, send, send_cnt, s, &rp, ctx->sh_off);
    if (rc != G4S_OK) return rc;
    ncclComm_t comm = (ncclComm_t)ctx->nccl_comm;
    {
        // an error the communicator raised since the last step (a peer that
        // failed) ends the sharded state before anything more is queued
        ncclResult_t st = ncclSuccess;
        if (g_nccl.CommGetAsyncError(comm, &st) == ncclSuccess && st != ncclSuccess && st != ncclInProgress) {
            shard_release(ctx, true);
            return fail(ctx, G4S_ERR_NCCL, "%s: communicator error: %s; communicator aborted", who,
                        g_nccl.GetErrorString(st));
        }
    }
    // a call of a non-blocking communicator succeeds or is still in progress
    auto ok = [](ncclResult_t x) { return x == ncclSuccess || x == ncclInProgress; };
    ncclResult_t r = g_nccl.GroupStart();
    if (ok(r)) r = g_nccl.AllGather(send, recv, (size_t)P, ncclUint64, comm, s);
    if (ok(r)) r = g_nccl.AllGather(send_cnt, recv_cnt, (size_t)rows, ncclInt32, comm, s);
    const ncclResult_t r2 = g_nccl.GroupEnd();
    if (ok(r)) r = r2;
    if ((rc = nccl_group_done(ctx, who, "all-gather", r)) != G4S_OK) return rc;
    // the merge reads list w of row i at recv + w * P + offset[i]
    rc = shard_merge_core(ctx, recv, recv_cnt, W, rows, ctx->shard_vocab, params, params_stride, softcap, u, out_tokens,
                          extra, s, &rp, ctx->sh_off, P);
    if (rc != G4S_OK || !sr.any_full_draw) return rc;
    // full-vocabulary draws: the rank whose slice holds the crossing writes the
    // token, the others keep -1; a max over the ranks gives every rank the token
    rc = shard_resolve_core(ctx, logits_slice, dtype, rows, n, row_stride, off, ctx->shard_rank, params,
                            params_stride, softcap, u, out_tokens, extra, s, &rp);
    if (rc != G4S_OK) return rc;
    r = g_nccl.GroupStart();
    if (ok(r)) r = g_nccl.AllReduce(out_tokens, out_tokens, (size_t)rows, ncclInt32, ncclMax, comm, s);
    if (ok(r) && extra && extra->token_prob)
        r = g_nccl.AllReduce(extra->token_prob, extra->token_prob, (size_t)rows, ncclFloat32, ncclMax, comm, s);
    const ncclResult_t r3 = g_nccl.GroupEnd();
    if (ok(r)) r = r3;
    return nccl_group_done(ctx, who, "all-reduce", r);
}

int32_t g4s_shard_set_timeout(g4s_ctx *ctx, int64_t ms)
{
    if (!ctx) return fail(nullptr, G4S_ERR_ARG, "g4s_shard_set_timeout: ctx is NULL");
    if (ms < 0) return fail(ctx, G4S_ERR_ARG, "g4s_shard_set_timeout: negative deadline %lld", (long long)ms);
    ctx->shard_timeout_ms = ms ? ms : G4S_SHARD_TIMEOUT_MS_DEFAULT;
    return G4S_OK;
}

int32_t g4s_shard_wait(g4s_ctx *ctx, void *stream, int64_t timeout_ms)
{
    static const char *who = "g4s_shard_wait";
    if (!ctx) return fail(nullptr, G4S_ERR_ARG, "%s: ctx is NULL", who);
    if (!ctx->nccl_comm) return fail(ctx, G4S_ERR_STATE, "%s: the context is not sharded", who);
    DeviceGuard guard(ctx->device);
    if (!guard.ok) return fail(ctx, G4S_ERR_CUDA, "%s: cannot select device %d", who, ctx->device);
    cudaStream_t s = stream ? (cudaStream_t)stream : ctx->stream;
    if (cudaEventRecord(ctx->shard_ev, s) != cudaSuccess) {
        const cudaError_t e = cudaGetLastError();
        return fail(ctx, G4S_ERR_CUDA, "%s: event record: %s", who, cudaGetErrorString(e));
    }
    const int64_t limit = timeout_ms > 0 ? timeout_ms : ctx->shard_timeout_ms;
    const auto t0 = std::chrono::steady_clock::now();
    auto elapsed_ms = [&]() {
        return (int64_t)std::chrono::duration_cast<std::chrono::milliseconds>(std::chrono::steady_clock::now() - t0)
            .count();
    };
    ncclComm_t comm = (ncclComm_t)ctx->nccl_comm;
    for (;;) {
        const cudaError_t q = cudaEventQuery(ctx->shard_ev);
        if (q == cudaSuccess) return G4S_OK;
        if (q != cudaErrorNotReady) return fail(ctx, G4S_ERR_CUDA, "%s: %s", who, cudaGetErrorString(q));
        ncclResult_t st = ncclSuccess;
        const ncclResult_t r = g_nccl.CommGetAsyncError(comm, &st);
        const bool failed = r != ncclSuccess || (st != ncclSuccess && st != ncclInProgress);
        const bool late = elapsed_ms() >= limit;
        if (failed || late) {
            // the abort ends the communicator's kernels that still wait on a
            // peer; the stream then drains (bounded), and the exchange buffers go
            const char *why = g_nccl.GetErrorString(r != ncclSuccess ? r : st);
            g_nccl.CommAbort(comm);
            ctx->nccl_comm = nullptr;
            const auto t1 = std::chrono::steady_clock::now();
            while (cudaEventQuery(ctx->shard_ev) == cudaErrorNotReady &&
                   std::chrono::steady_clock::now() - t1 < std::chrono::milliseconds(limit))
                std::this_thread::sleep_for(std::chrono::microseconds(200));
            const bool drained = cudaEventQuery(ctx->shard_ev) == cudaSuccess;
            if (drained) shard_release(ctx);
            if (late)
                return fail(ctx, G4S_ERR_TIMEOUT,
                            "%s: the step did not finish within %lld ms (a rank stalled or left); communicator "
                            "aborted%s",
                            who, (long long)limit, drained ? "" : ", stream still busy");
            return fail(ctx, G4S_ERR_NCCL, "%s: communicator error: %s; communicator aborted", who, why);
        }
        std::this_thread::sleep_for(std::chrono::microseconds(50));
    }
}

int32_t g4s_shard_abort(g4s_ctx *ctx)
{
    if (!ctx) return fail(nullptr, G4S_ERR_ARG, "g4s_shard_abort: ctx is NULL");
    if (!ctx->nccl_comm) return G4S_OK;
    DeviceGuard guard(ctx->device);
    if (!guard.ok) return fail(ctx, G4S_ERR_CUDA, "g4s_shard_abort: cannot select device %d", ctx->device);
    shard_release(ctx, true);
    return G4S_OK;
}

// ---------------------------------------------------------------------------
// beam search
// ---------------------------------------------------------------------------
void g4s_beam_params_defaults(g4s_beam_params *p)
{
    if (!p) return;
    memset(p, 0, sizeof(*p));
    p->beams = p->n_out = 4;
    p->temperature = 1.0;
    p->n_eos = 3;
    p->eos[0] = 1;
    p->eos[1] = 106;
    p->eos[2] = 50;
}

// Whether out may be written while in is read: other memory, or (same) the very same array.
static bool aliasing_ok(const void *in, const void *out, size_t in_bytes, size_t out_bytes, bool same)
{
    if (!in || !out) return true;
    if (in == out) return same;
    const char *a = (const char *)in, *b = (const char *)out;
    return a + in_bytes <= b || b + out_bytes <= a;
}

// Whether each output is memory of its own: it shares no byte with another output nor with an
// input, except that output i may be input i itself where bit i of `same` is set.
struct Span {
    const void *p;  // NULL: not given
    size_t bytes;
};
static bool spans_apart(std::initializer_list<Span> outs, std::initializer_list<Span> ins, unsigned same)
{
    int i = 0;
    for (const Span *o = outs.begin(); o != outs.end(); o++, i++) {
        for (const Span *q = o + 1; q != outs.end(); q++)
            if (!aliasing_ok(o->p, q->p, o->bytes, q->bytes, false)) return false;
        int j = 0;
        for (const Span *q = ins.begin(); q != ins.end(); q++, j++)
            if (!aliasing_ok(q->p, o->p, q->bytes, o->bytes, i == j && (same >> i & 1))) return false;
    }
    return true;
}

// Whether an array lies apart from rows of row_bytes, `stride` bytes from one to the next
// (between two rows, for one).
static bool apart_from_rows(Span s, const void *base, int64_t rows, int64_t row_bytes, int64_t stride)
{
    if (!s.p) return true;
    const int64_t lo = (int64_t)((intptr_t)s.p - (intptr_t)base), hi = lo + (int64_t)s.bytes;
    const int64_t first = lo < row_bytes ? 0 : (lo - row_bytes) / stride + 1;  // the first row that ends behind lo
    return first >= rows || first * stride >= hi;
}

// Whether all arrays of 4-byte elements stand on their alignment.
static bool aligned4(std::initializer_list<const void *> arrays)
{
    uintptr_t bits = 0;
    for (const void *p : arrays) bits |= (uintptr_t)p;
    return bits % 4 == 0;
}

static int pow2_at_least(int n)
{
    int p = 4;
    while (p < n) p <<= 1;
    return p;
}

static int32_t beam_select_args(g4s_ctx *ctx, const char *who, const void *logits, int32_t dtype, int32_t groups,
                                int32_t vocab, int64_t row_stride, float softcap, const g4s_beam_params *p,
                                const g4s_beam_state *in, const g4s_beam_state *out, int32_t *out_parents,
                                int32_t *out_tokens, BeamArgs &a, bool &vec)
{
    if (!logits || !p || !in || !out || !out_parents || !out_tokens || !in->scores || !out->scores)
        return fail(ctx, G4S_ERR_ARG,
                    "%s: logits, params, in, out, their scores, out_parents and out_tokens must be non-NULL", who);
    if (dtype != G4S_F32 && dtype != G4S_BF16) return fail(ctx, G4S_ERR_ARG, "%s: bad dtype %d", who, dtype);
    if (p->beams < 1 || p->beams > G4S_BEAM_MAX || p->n_out < 1 || p->n_out > G4S_BEAM_MAX_OUT)
        return fail(ctx, G4S_ERR_ARG, "%s: beams %d outside [1, %d] or n_out %d outside [1, %d]", who, p->beams,
                    G4S_BEAM_MAX, p->n_out, G4S_BEAM_MAX_OUT);
    if (groups < 1 || vocab < 1)
        return fail(ctx, G4S_ERR_ARG, "%s: groups (%d) and vocab (%d) must be >= 1", who, groups, vocab);
    if ((int64_t)groups * p->beams > ctx->max_rows || vocab > ctx->max_vocab)
        return fail(ctx, G4S_ERR_CAPACITY, "%s: %d groups of %d beams / vocab %d exceed the context (%d / %d)", who,
                    groups, p->beams, vocab, ctx->max_rows, ctx->max_vocab);
    if (row_stride < vocab)
        return fail(ctx, G4S_ERR_ARG, "%s: row_stride %lld < vocab %d", who, (long long)row_stride, vocab);
    const size_t esize = dtype == G4S_F32 ? 4u : 2u;
    if ((uintptr_t)logits % esize) return fail(ctx, G4S_ERR_ARG, "%s: logits are not aligned to their type", who);
    if (!aligned4({in->scores, in->lens, out->scores, out->lens, out_parents, out_tokens}))
        return fail(ctx, G4S_ERR_ARG, "%s: scores, lens, out_parents or out_tokens are not aligned to their type", who);
    if (!(p->temperature >= 1e-6 && p->temperature <= 1e6))
        return fail(ctx, G4S_ERR_ARG, "%s: temperature %g outside [1e-6, 1e6]", who, p->temperature);
    if (!(p->length_alpha >= 0.0 && p->length_alpha <= 8.0))
        return fail(ctx, G4S_ERR_ARG, "%s: length_alpha %g outside [0, 8]", who, p->length_alpha);
    if (!(softcap <= 0.0f || (softcap >= 1e-6f && softcap <= 1e6f)))
        return fail(ctx, G4S_ERR_ARG, "%s: softcap %g is neither <= 0 nor within [1e-6, 1e6]", who, softcap);
    if (softcap > 1e8 * p->temperature)
        return fail(ctx, G4S_ERR_ARG, "%s: softcap %g is over 1e8 times temperature %g", who, softcap, p->temperature);
    if (p->n_eos < 0 || p->n_eos > G4S_BEAM_MAX_EOS)
        return fail(ctx, G4S_ERR_ARG, "%s: n_eos %d outside [0, %d]", who, p->n_eos, G4S_BEAM_MAX_EOS);
    if (!in->lens && (p->length_alpha != 0.0 || out->lens))
        return fail(ctx, G4S_ERR_ARG, "%s: in->lens is NULL with a length_alpha or out->lens", who);
    const size_t ni = (size_t)groups * p->beams, no = (size_t)groups * p->n_out;
    const bool same = p->n_out == p->beams;
    if (row_stride > ((int64_t)1 << 60) / (int64_t)ni)
        return fail(ctx, G4S_ERR_ARG, "%s: row_stride %lld beyond 2^60 elements in all", who, (long long)row_stride);
    const Span outs[5] = {{out->scores, no * 4}, {out->lens, no * 4}, {out->done, no}, {out_parents, no * 4}, {out_tokens, no * 4}};
    bool ok = spans_apart({outs[0], outs[1], outs[2], outs[3], outs[4]},
                          {{in->scores, ni * 4}, {in->lens, ni * 4}, {in->done, ni}}, same ? 7 : 0);
    for (const Span &o : outs) ok = ok && apart_from_rows(o, logits, (int64_t)ni, vocab * (int64_t)esize, row_stride * (int64_t)esize);
    if (!ok)
        return fail(ctx, G4S_ERR_ARG,
                    "%s: an output overlaps another, the logits or in (allowed: in's own arrays, with n_out == beams)", who);

    memset(&a, 0, sizeof(a));
    a.logits = logits;
    a.row_stride = row_stride;
    a.rows = groups * p->beams;
    a.beams = p->beams;
    a.vocab = vocab;
    a.n_out = p->n_out;
    a.pe = pow2_at_least(p->beams * p->n_out);
    a.pc = std::max(512, pow2_at_least(p->n_out * (p->n_out + 1) / 2));
    a.softcap = softcap > 0.0f ? softcap : 0.0f;
    a.k64 = 1.4426950408889634074 / p->temperature;
    a.alpha = p->length_alpha;
    a.pad_token = p->pad_token;
    a.n_eos = p->n_eos;
    memcpy(a.eos, p->eos, sizeof(a.eos));
    a.scores = in->scores;
    a.lens = in->lens;
    a.done = in->done;
    a.out_scores = out->scores;
    a.out_lens = out->lens;
    a.out_done = out->done;
    a.out_parents = out_parents;
    a.out_tokens = out_tokens;
    a.istat = ctx->beam_stat;
    vec = ((uintptr_t)logits % 16u == 0) && ((row_stride * (int64_t)esize) % 16 == 0);
    return G4S_OK;
}

// Strided memory: count[0] x count[1] x count[2] segments of `bytes`; `extent` bytes from its
// first to behind its last, -1 for 2^60 or more.
struct Strided {
    const char *p = nullptr;
    int64_t count[3], stride[3], bytes = 0, extent = 0;
    Strided() {}
    Strided(const g4s_beam_tensor &t, const void *at, int64_t rows)  // a tensor's src or dst
        : p((const char *)at), count{rows, t.segs0, t.segs1}, stride{t.row_stride, t.stride0, t.stride1}, bytes(t.seg_bytes)
    {
        __int128 e = bytes;
        for (int i = 0; i < 3; i++) e += (__int128)(count[i] - 1) * stride[i];
        extent = e < ((__int128)1 << 60) ? (int64_t)e : -1;
    }
};

// Whether a segment of x shares a byte with one of y (of x itself: two of its segments): whether
// whole numbers q_i, a segment's place along an axis less the other's, bring the distance
// d + sum q_i stride_i between two segments into (-x.bytes, y.bytes).  The axes go from the
// longest stride on, and of each only the q_i from which the shorter ones can still get there:
// one or two, where an axis' whole extent lies within the next one's stride.  A layout that
// takes over STEPS of them counts as overlapping.
struct Meeting {
    static constexpr int STEPS = 1 << 14;
    int n = 0, steps = 0;
    int64_t stride[6], least[6], most[6];  // axes, and the range of their q
    int64_t low[7], high[7];               // what the axes from i on can add
    int64_t before, behind;
    bool self;

    void add(int64_t s, int64_t from, int64_t to)
    {
        if (from == to) return;
        for (int i = 0; i < n && !self; i++) {
            if (stride[i] != s) continue;
            least[i] += from;
            most[i] += to;
            return;
        }
        int i = n++;
        for (; i > 0 && stride[i - 1] < s; i--) {
            stride[i] = stride[i - 1];
            least[i] = least[i - 1];
            most[i] = most[i - 1];
        }
        stride[i] = s;
        least[i] = from;
        most[i] = to;
    }
    static int64_t floor_of(int64_t a, int64_t s) { return a / s - (a % s < 0); }
    bool from(int i, int64_t d, bool same)
    {
        if (++steps > STEPS) return true;
        if (i == n) return d > -before && d < behind && !(self && same);
        const int64_t s = stride[i];
        const int64_t last = std::min(most[i], -floor_of(d + low[i + 1] - behind, s) - 1);
        for (int64_t q = std::max(least[i], floor_of(-before - high[i + 1] - d, s) + 1); q <= last; q++)
            if (from(i + 1, d + q * s, same && q == 0)) return true;
        return false;
    }
    static bool of(const Strided &x, const Strided &y)
    {
        const int64_t d = (int64_t)((intptr_t)x.p - (intptr_t)y.p);
        if (d >= y.extent || -d >= x.extent) return false;
        Meeting m;
        m.self = &x == &y;
        m.before = x.bytes;
        m.behind = y.bytes;
        for (int i = 0; i < 3; i++) m.add(x.stride[i], m.self ? 1 - x.count[i] : 0, x.count[i] - 1);
        for (int i = 0; i < 3 && !m.self; i++) m.add(y.stride[i], 1 - y.count[i], 0);
        m.low[m.n] = m.high[m.n] = 0;
        bool nested = true;  // (the usual layout, without a search)
        for (int i = m.n - 1; i >= 0; i--) {
            nested = nested && m.stride[i] >= m.high[i + 1] + m.behind;
            m.low[i] = m.low[i + 1] + m.least[i] * m.stride[i];
            m.high[i] = m.high[i + 1] + m.most[i] * m.stride[i];
        }
        return !(m.self && nested) && m.from(0, d, true);
    }
};

// Largest of 16, 4 and 1 that divides every value of `bits` (addresses and sizes or-ed together).
static int copy_width(uint64_t bits) { return bits % 16 == 0 ? 16 : bits % 4 == 0 ? 4 : 1; }

static int32_t beam_reorder_args(g4s_ctx *ctx, const char *who, const int32_t *parents, int32_t groups, int32_t beams,
                                 const g4s_beam_tensor *tensors, int32_t n_tensors, ReorderArgs &a, int64_t &blocks)
{
    if (n_tensors < 0 || n_tensors > G4S_BEAM_MAX_TENSORS)
        return fail(ctx, G4S_ERR_ARG, "%s: n_tensors %d outside [0, %d]", who, n_tensors, G4S_BEAM_MAX_TENSORS);
    if (!parents || (n_tensors && !tensors)) return fail(ctx, G4S_ERR_ARG, "%s: parents or tensors is NULL", who);
    if (!aligned4({parents})) return fail(ctx, G4S_ERR_ARG, "%s: parents are not aligned to their type", who);
    if (beams < 1 || beams > G4S_BEAM_MAX || groups < 1 || (int64_t)groups * beams > 0x7fffffff - G4S_BEAM_MAX)
        return fail(ctx, G4S_ERR_ARG, "%s: beams %d outside [1, %d], or %d groups", who, beams, G4S_BEAM_MAX, groups);
    a.parents = parents;
    a.beams = beams;
    a.n = 0;
    blocks = 0;
    for (int i = 0; i < n_tensors; i++) {
        const g4s_beam_tensor &t = tensors[i];
        if (t.segs0 < 1 || t.segs1 < 1 || t.seg_bytes < 0 || t.row_stride < 0 || t.stride0 < 0 || t.stride1 < 0)
            return fail(ctx, G4S_ERR_ARG, "%s: tensors[%d]: a negative stride or size, or no segment", who, i);
        if (t.seg_bytes == 0) continue;
        if (!t.src || !t.dst) return fail(ctx, G4S_ERR_ARG, "%s: tensors[%d]: NULL src or dst", who, i);
        if (groups * (int64_t)beams > 1 && t.row_stride < t.seg_bytes)
            return fail(ctx, G4S_ERR_ARG, "%s: tensors[%d]: row_stride %lld < seg_bytes %lld", who, i,
                        (long long)t.row_stride, (long long)t.seg_bytes);
        if ((t.segs0 > 1 && t.stride0 < t.seg_bytes) || (t.segs1 > 1 && t.stride1 < t.seg_bytes))
            return fail(ctx, G4S_ERR_ARG, "%s: tensors[%d]: segments overlap", who, i);
        ReorderTensor &q = a.t[a.n];
        q.width = copy_width((uint64_t)(uintptr_t)t.src | (uint64_t)(uintptr_t)t.dst | (uint64_t)t.seg_bytes |
                             (uint64_t)t.row_stride | (t.segs0 > 1 ? (uint64_t)t.stride0 : 0) |
                             (t.segs1 > 1 ? (uint64_t)t.stride1 : 0));
        const int64_t seg_cols = t.seg_bytes / q.width, segs = (int64_t)t.segs0 * t.segs1;
        if (seg_cols > 0x7fffffff || segs > 0x7fffffff || segs * seg_cols > 0x7fffffff)
            return fail(ctx, G4S_ERR_CAPACITY, "%s: tensors[%d]: over 2^31 columns of %d bytes a row", who, i, q.width);
        q.src = (const char *)t.src;
        q.dst = (char *)t.dst;
        q.row_stride = t.row_stride;
        q.stride0 = t.stride0;
        q.stride1 = t.stride1;
        q.segs1 = (uint32_t)t.segs1;
        q.seg_cols = (uint32_t)seg_cols;
        q.cols = (uint32_t)(segs * seg_cols);
        q.blocks = (uint32_t)ceil_div(q.cols, REORDER_THREADS);
        a.first[a.n++] = blocks;
        blocks += (int64_t)groups * q.blocks;
        if (blocks > 0x7fffffff) return fail(ctx, G4S_ERR_CAPACITY, "%s: over 2^31 blocks of work", who);
    }
    Strided dst[G4S_BEAM_MAX_TENSORS], src[G4S_BEAM_MAX_TENSORS];
    const Strided read(g4s_beam_tensor{nullptr, nullptr, 4, 1, 0, 1, 0, 4}, parents, (int64_t)groups * beams);
    for (int i = 0; i < n_tensors; i++) {
        const g4s_beam_tensor &t = tensors[i];
        if (t.seg_bytes == 0) continue;
        const bool in_place = t.src == t.dst;
        dst[i] = Strided(t, t.dst, (int64_t)groups * beams);
        src[i] = Strided(t, t.src, (int64_t)groups * beams);
        if (dst[i].extent < 0) return fail(ctx, G4S_ERR_ARG, "%s: tensors[%d]: strides beyond 2^60 bytes in all", who, i);
        if (Meeting::of(dst[i], dst[i])) return fail(ctx, G4S_ERR_ARG, "%s: tensors[%d]: segments or rows overlap", who, i);
        if (!in_place && Meeting::of(dst[i], src[i]))
            return fail(ctx, G4S_ERR_ARG, "%s: tensors[%d]: dst overlaps src (allowed: src itself)", who, i);
        if (Meeting::of(dst[i], read)) return fail(ctx, G4S_ERR_ARG, "%s: tensors[%d]: dst overlaps the parents", who, i);
        for (int j = 0; j < i; j++) {  // (an empty tensor's extent is 0)
            if (Meeting::of(dst[i], dst[j]) || (src[j].p != dst[j].p && Meeting::of(dst[i], src[j])) ||
                (!in_place && Meeting::of(src[i], dst[j])))
                return fail(ctx, G4S_ERR_ARG, "%s: tensors[%d] and tensors[%d] overlap where one is written", who, j, i);
        }
    }
    return G4S_OK;
}

static int32_t pages_cache_args(g4s_ctx *ctx, const char *who, const g4s_page_cache *c, PagesArgs &a, PoolArgs &pools)
{
    if (!c) return fail(ctx, G4S_ERR_ARG, "%s: cache is NULL", who);
    if (c->page_tokens < 1 || c->n_pages < 1 || c->max_seq_pages < 1 ||
        (int64_t)c->max_seq_pages * c->page_tokens > 0x3fffffff || c->n_pages > 0x3fffffff)
        return fail(ctx, G4S_ERR_ARG,
                    "%s: page_tokens %d, n_pages %d and max_seq_pages %d must be >= 1, pages and a sequence's positions "
                    "below 2^30",
                    who, c->page_tokens, c->n_pages, c->max_seq_pages);
    if (c->n_pools < 0 || c->n_pools > G4S_PAGES_MAX_POOLS || (c->n_pools && !c->pools))
        return fail(ctx, G4S_ERR_ARG, "%s: n_pools %d outside [0, %d], or pools is NULL", who, c->n_pools,
                    G4S_PAGES_MAX_POOLS);
    memset(&a, 0, sizeof(a));
    a.page_tokens = c->page_tokens;
    a.n_pages = c->n_pages;
    a.width = c->max_seq_pages;
    pools.n = c->n_pools;
    pools.chunks = 1;
    for (int i = 0; i < c->n_pools; i++) {
        const g4s_page_pool &p = c->pools[i];
        if (!p.data || p.segs < 1 || p.token_bytes < 1 || p.page_stride < 1 || p.seg_stride < 0)
            return fail(ctx, G4S_ERR_ARG, "%s: pools[%d]: NULL data, or a size below 1", who, i);
        PoolArg &q = pools.p[i];
        q.width = copy_width((uint64_t)(uintptr_t)p.data | (uint64_t)p.page_stride | (uint64_t)p.token_bytes |
                             (p.segs > 1 ? (uint64_t)p.seg_stride : 0));
        const int64_t vecs = p.token_bytes / q.width;
        if (vecs > 0x7fffffff || vecs * c->page_tokens > 0x7fffffff || vecs * c->page_tokens * p.segs > 0x7fffffff)
            return fail(ctx, G4S_ERR_CAPACITY, "%s: pools[%d]: a page of over 2^31 vectors of %d bytes", who, i, q.width);
        const int64_t seg = p.token_bytes * c->page_tokens;
        if (p.page_stride < seg || (p.segs > 1 && (p.seg_stride < seg || (p.page_stride - seg) / (p.segs - 1) < p.seg_stride)))
            return fail(ctx, G4S_ERR_ARG, "%s: pools[%d]: segments or pages overlap", who, i);
        q.data = (char *)p.data;
        q.page_stride = p.page_stride;
        q.seg_stride = p.seg_stride;
        q.segs = p.segs;
        q.token_vecs = (uint32_t)vecs;
        pools.chunks = std::max<int>(pools.chunks, (int)ceil_div(vecs * c->page_tokens * p.segs, pages_chunk_vecs()));
    }
    return G4S_OK;
}

static int32_t pages_seqs_ok(g4s_ctx *ctx, const char *who, int32_t n, const char *what)
{
    const int most = std::min(ctx->max_rows, G4S_PAGES_MAX_SEQS);
    if (n < 0) return fail(ctx, G4S_ERR_ARG, "%s: %s %d < 0", who, what, n);
    if (n > most) return fail(ctx, G4S_ERR_CAPACITY, "%s: %s %d above %d", who, what, n, most);
    return G4S_OK;
}

static int32_t pages_fork_args(g4s_ctx *ctx, const char *who, const g4s_page_cache *cache, int32_t n_in,
                               const g4s_page_tables *in, int32_t n_out, const int32_t *src, int32_t n_new,
                               const uint8_t *frozen, const g4s_page_tables *out, int32_t *result, PagesArgs &a,
                               PoolArgs &pools)
{
    int32_t rc = pages_cache_args(ctx, who, cache, a, pools);
    if (rc != G4S_OK) return rc;
    if ((rc = pages_seqs_ok(ctx, who, n_in, "n_in")) != G4S_OK || (rc = pages_seqs_ok(ctx, who, n_out, "n_out")) != G4S_OK)
        return rc;
    if (!in || !out || !result || !in->refs || !out->refs || (n_in && (!in->tables || !in->lens)) ||
        (n_out && (!out->tables || !out->lens || !src)))
        return fail(ctx, G4S_ERR_ARG, "%s: in, out, their arrays, src and result must be non-NULL", who);
    if (!aligned4({in->tables, in->lens, in->refs, out->tables, out->lens, out->refs, src, result}))
        return fail(ctx, G4S_ERR_ARG, "%s: tables, lens, refs, src or result are not aligned to their type", who);
    if (n_new < 0 || n_new > 0x3fffffff) return fail(ctx, G4S_ERR_ARG, "%s: n_new %d outside [0, 2^30)", who, n_new);
    const size_t wi = (size_t)n_in * a.width * 4, wo = (size_t)n_out * a.width * 4, np = (size_t)a.n_pages * 4;
    if (n_in && n_out && !aliasing_ok(in->tables, out->tables, wi, wo, false))
        return fail(ctx, G4S_ERR_ARG, "%s: out->tables overlaps in->tables", who);
    if (!aliasing_ok(in->refs, out->refs, np, np, true) ||
        (n_in && n_out && !aliasing_ok(in->lens, out->lens, (size_t)n_in * 4, (size_t)n_out * 4, true)))
        return fail(ctx, G4S_ERR_ARG, "%s: out's refs or lens overlap in's (allowed: the same arrays)", who);
    auto span = [](const void *p, size_t bytes) { return bytes ? Span{p, bytes} : Span{nullptr, 0}; };
    const size_t no = (size_t)n_out, ni = (size_t)n_in * 4;
    if (!spans_apart({span(out->tables, wo), span(out->lens, no * 4), {out->refs, np}, {result, 16}},
                     {span(in->tables, wi), span(in->lens, ni), {in->refs, np}, span(src, no * 4), span(frozen, no)}, 6))
        return fail(ctx, G4S_ERR_ARG, "%s: an array of out, or result, overlaps another array (allowed: in's lens and refs)", who);
    a.n_in = n_in;
    a.n_out = n_out;
    a.n_new = n_new;
    a.max_copies = n_out;
    a.tables_in = in->tables;
    a.lens_in = in->lens;
    a.refs_in = in->refs;
    a.src = src;
    a.frozen = frozen;
    a.tables_out = out->tables;
    a.lens_out = out->lens;
    a.refs_out = out->refs;
    a.result = result;
    a.copies = ctx->pg_copies;
    a.n_copies = ctx->pg_n_copies;
    return G4S_OK;
}

int32_t g4s_beam_select(g4s_ctx *ctx, const void *logits, int32_t dtype, int32_t groups, int32_t vocab,
                        int64_t row_stride, float softcap, const g4s_beam_params *params, const g4s_beam_state *in,
                        const g4s_beam_state *out, int32_t *out_parents, int32_t *out_tokens, void *stream)
{
    static const char *who = "g4s_beam_select";
    if (!ctx) return fail(nullptr, G4S_ERR_ARG, "%s: ctx is NULL", who);
    BeamArgs a;
    bool vec;
    const int32_t rc = beam_select_args(ctx, who, logits, dtype, groups, vocab, row_stride, softcap, params, in, out,
                                        out_parents, out_tokens, a, vec);
    if (rc != G4S_OK) return rc;
    DeviceGuard guard(ctx->device);
    if (!guard.ok) return fail(ctx, G4S_ERR_CUDA, "%s: cannot select device %d", who, ctx->device);
    const cudaError_t e = launch_beam_select(a, dtype, vec, ctx->sm_count, stream ? (cudaStream_t)stream : ctx->stream);
    if (e != cudaSuccess) return fail(ctx, G4S_ERR_CUDA, "%s: launch failed: %s", who, cudaGetErrorString(e));
    return G4S_OK;
}

int32_t g4s_beam_reorder(g4s_ctx *ctx, const int32_t *parents, int32_t groups, int32_t beams,
                         const g4s_beam_tensor *tensors, int32_t n_tensors, void *stream)
{
    static const char *who = "g4s_beam_reorder";
    if (!ctx) return fail(nullptr, G4S_ERR_ARG, "%s: ctx is NULL", who);
    ReorderArgs a;
    int64_t blocks = 0;
    const int32_t rc = beam_reorder_args(ctx, who, parents, groups, beams, tensors, n_tensors, a, blocks);
    if (rc != G4S_OK || blocks == 0) return rc;
    DeviceGuard guard(ctx->device);
    if (!guard.ok) return fail(ctx, G4S_ERR_CUDA, "%s: cannot select device %d", who, ctx->device);
    const cudaError_t e = launch_beam_reorder(a, blocks, stream ? (cudaStream_t)stream : ctx->stream);
    if (e != cudaSuccess) return fail(ctx, G4S_ERR_CUDA, "%s: launch failed: %s", who, cudaGetErrorString(e));
    return G4S_OK;
}

int32_t g4s_pages_fork(g4s_ctx *ctx, const g4s_page_cache *cache, int32_t n_in, const g4s_page_tables *in,
                       int32_t n_out, const int32_t *src, int32_t n_new, const uint8_t *frozen,
                       const g4s_page_tables *out, int32_t *result, void *stream)
{
    static const char *who = "g4s_pages_fork";
    if (!ctx) return fail(nullptr, G4S_ERR_ARG, "%s: ctx is NULL", who);
    PagesArgs a;
    PoolArgs pools;
    const int32_t rc = pages_fork_args(ctx, who, cache, n_in, in, n_out, src, n_new, frozen, out, result, a, pools);
    if (rc != G4S_OK) return rc;
    DeviceGuard guard(ctx->device);
    if (!guard.ok) return fail(ctx, G4S_ERR_CUDA, "%s: cannot select device %d", who, ctx->device);
    const cudaError_t e = launch_pages_fork(a, pools, ctx->sm_count, stream ? (cudaStream_t)stream : ctx->stream);
    if (e != cudaSuccess) return fail(ctx, G4S_ERR_CUDA, "%s: launch failed: %s", who, cudaGetErrorString(e));
    return G4S_OK;
}

int32_t g4s_pages_compact(g4s_ctx *ctx, const g4s_page_cache *cache, int32_t n_seqs, const g4s_page_tables *in,
                          const g4s_page_tables *out, int32_t *page_map, int32_t *moves, int32_t *result, void *stream)
{
    static const char *who = "g4s_pages_compact";
    if (!ctx) return fail(nullptr, G4S_ERR_ARG, "%s: ctx is NULL", who);
    PagesArgs a;
    PoolArgs pools;
    int32_t rc = pages_cache_args(ctx, who, cache, a, pools);
    if (rc != G4S_OK || (rc = pages_seqs_ok(ctx, who, n_seqs, "n_seqs")) != G4S_OK) return rc;
    if (!in || !out || !page_map || !moves || !result || !in->refs || !out->refs ||
        (n_seqs && (!in->tables || !in->lens || !out->tables)))
        return fail(ctx, G4S_ERR_ARG, "%s: in, out, their arrays, page_map, moves and result must be non-NULL", who);
    if (!aligned4({in->tables, in->lens, in->refs, out->tables, out->refs, page_map, result}))
        return fail(ctx, G4S_ERR_ARG, "%s: tables, lens, refs, page_map or result are not aligned to their type", who);
    if ((uintptr_t)moves % 8) return fail(ctx, G4S_ERR_ARG, "%s: moves is not 8-byte aligned", who);
    const size_t w = (size_t)n_seqs * a.width * 4, np = (size_t)a.n_pages * 4;
    if ((n_seqs && !aliasing_ok(in->tables, out->tables, w, w, true)) || !aliasing_ok(in->refs, out->refs, np, np, true))
        return fail(ctx, G4S_ERR_ARG, "%s: out's tables or refs overlap in's (allowed: the same arrays)", who);
    auto span = [](const void *p, size_t bytes) { return bytes ? Span{p, bytes} : Span{nullptr, 0}; };
    if (!spans_apart({span(out->tables, w), {out->refs, np}, {page_map, np}, {moves, np}, {result, 16}},
                     {span(in->tables, w), {in->refs, np}, span(in->lens, (size_t)n_seqs * 4)}, 3))
        return fail(ctx, G4S_ERR_ARG, "%s: an output overlaps another array (allowed: in's tables and refs)", who);
    a.n_in = a.n_out = n_seqs;
    a.max_copies = a.n_pages / 2;
    a.tables_in = in->tables;
    a.lens_in = in->lens;
    a.refs_in = in->refs;
    a.tables_out = out->tables;
    a.refs_out = out->refs;
    a.page_map = page_map;
    a.moves = moves;
    a.result = result;
    DeviceGuard guard(ctx->device);
    if (!guard.ok) return fail(ctx, G4S_ERR_CUDA, "%s: cannot select device %d", who, ctx->device);
    const cudaError_t e = launch_pages_compact(a, pools, ctx->sm_count, stream ? (cudaStream_t)stream : ctx->stream);
    if (e != cudaSuccess) return fail(ctx, G4S_ERR_CUDA, "%s: launch failed: %s", who, cudaGetErrorString(e));
    return G4S_OK;
}

int32_t g4s_beam_step(g4s_ctx *ctx, const void *logits, int32_t dtype, int32_t groups, int32_t vocab,
                      int64_t row_stride, float softcap, const g4s_beam_params *params, const g4s_beam_state *in,
                      const g4s_beam_state *out, int32_t *out_parents, int32_t *out_tokens,
                      const g4s_beam_tensor *tensors, int32_t n_tensors, const g4s_beam_pages *pages, void *stream)
{
    static const char *who = "g4s_beam_step";
    if (!ctx) return fail(nullptr, G4S_ERR_ARG, "%s: ctx is NULL", who);
    BeamArgs a;
    bool vec;
    int32_t rc = beam_select_args(ctx, who, logits, dtype, groups, vocab, row_stride, softcap, params, in, out,
                                  out_parents, out_tokens, a, vec);
    if (rc != G4S_OK) return rc;
    if (params->n_out != params->beams)
        return fail(ctx, G4S_ERR_ARG, "%s: n_out %d is not beams %d", who, params->n_out, params->beams);
    ReorderArgs r;
    int64_t blocks = 0;
    if ((rc = beam_reorder_args(ctx, who, out_parents, groups, params->beams, tensors, n_tensors, r, blocks)) != G4S_OK)
        return rc;
    PagesArgs p;
    PoolArgs pools;
    if (pages && (rc = pages_fork_args(ctx, who, pages->cache, a.rows, &pages->in, a.rows, out_parents, pages->n_new,
                                       out->done, &pages->out, pages->result, p, pools)) != G4S_OK)
        return rc;
    if (pages) {  // the selection writes before the fork reads
        const size_t n = (size_t)a.rows, w = n * p.width * 4, np = (size_t)p.n_pages * 4;
        if (!spans_apart({{out->scores, n * 4}, {out->lens, n * 4}, {out->done, n}, {out_parents, n * 4}, {out_tokens, n * 4}},
                         {{p.tables_in, w}, {p.lens_in, n * 4}, {p.refs_in, np}, {p.tables_out, w}, {p.lens_out, n * 4},
                          {p.refs_out, np}, {p.result, 16}}, 0))
            return fail(ctx, G4S_ERR_ARG, "%s: an output of the selection overlaps an array of the pages", who);
    }
    DeviceGuard guard(ctx->device);
    if (!guard.ok) return fail(ctx, G4S_ERR_CUDA, "%s: cannot select device %d", who, ctx->device);
    cudaStream_t s = stream ? (cudaStream_t)stream : ctx->stream;
    cudaError_t e = launch_beam_select(a, dtype, vec, ctx->sm_count, s);
    if (e == cudaSuccess && blocks) e = launch_beam_reorder(r, blocks, s);
    if (e == cudaSuccess && pages) e = launch_pages_fork(p, pools, ctx->sm_count, s);
    if (e != cudaSuccess) return fail(ctx, G4S_ERR_CUDA, "%s: launch failed: %s", who, cudaGetErrorString(e));
    return G4S_OK;
}

}  // extern "C"
