// g4s_pages.cu -- the pages of a beam search's cache: forking by parents with
// copy on write, allocation and freeing (pages_fork_kernel), compaction
// (pages_compact_kernel), and the copies of page contents that both list
// (pages_copy_kernel).  No counterpart in the reference, whose cache is one
// contiguous ring a layer (src/Gemma4.Model.pas:61-66).
//
// What decides (tables, lengths, counts) is whole numbers and a few hundred
// KiB: one thread-block cluster walks it, its barriers standing between the
// steps, so that a fork is two launches whatever its size.  What moves bytes
// runs over the whole GPU as the first kernel's programmatic dependent.
//
// Measured (one B200): fork of one prompt of 4 beams, 1024 pages, 8.0 us (one CTA decides);
// of 32 prompts of 8 beams, 12288 pages, 14.0 (the cluster); of 8 prompts of 6 beams, up to
// 482 pages each, with 5 new positions, 16.3.  Latency bounds them: a few hundred KiB of
// table entries and counts, about ten dependent steps over them.  Compaction of 8192 pages,
// 258 MB read and written, 48.3 us: 6 the decision, 42 the copies at 6.1 TB/s (5.3 TB/s in
// all, of 6.6 for a plain copy).
#include <cooperative_groups.h>

#include "g4s_device.cuh"
#include "g4s_kernels.cuh"

namespace cg = cooperative_groups;

namespace g4s {

constexpr int PG_CLUSTER = 16;      // CTAs of the cluster that decides (16: a non-portable size)
constexpr int PG_THREADS = 1024;
constexpr int PG_WARPS = PG_THREADS / 32;
constexpr int PG_SLICES = PG_CLUSTER * PG_WARPS;  // a warp's slice of the page counts
constexpr int PC_THREADS = 256;     // CTA of the copies
constexpr int PC_VECS = 4;          // vectors a thread and step
constexpr int PC_CTAS = 4;          // CTAs on an SM (2, 3, 5, 6, 8: slower)

// Exclusive scan over the CTA's PG_THREADS values; *total gets the sum.  sh: PG_WARPS, not
// written again before the next barrier.
__device__ __forceinline__ unsigned long long pg_scan(unsigned long long v, unsigned long long *total, unsigned long long *sh)
{
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const unsigned long long inc = warp_incl_scan(v);
    if (lane == 31) sh[w] = inc;
    __syncthreads();
    const unsigned long long s = sh[lane], si = warp_incl_scan(s);
    *total = __shfl_sync(FULLMASK, si, 31);
    return __shfl_sync(FULLMASK, si - s, w) + inc - v;
}

// Pages of that many positions (each below 2^30, so sums of three fit in 32 bits).
__device__ __forceinline__ int pages_of(int tokens, int page_tokens)
{
    return (int)(((uint32_t)tokens + (uint32_t)page_tokens - 1) / (uint32_t)page_tokens);
}

// A sequence's length, or -1 where the table cannot hold it.
__device__ __forceinline__ int seq_len(const PagesArgs &a, int i)
{
    const int n = a.lens_in[i];
    return n >= 0 && (int64_t)n <= (int64_t)a.width * a.page_tokens ? n : -1;
}

// Fork.  Every CTA of the cluster works out the same sequences and needs in its own shared
// memory; the old sequences' table rows and the pages' counts are split over the warps.
// Up to these one CTA decides: its barriers are cheaper than the cluster's.  One CTA against
// the cluster, us: fork of 1024 table entries with 4096 pages 8.5 / 9.3, 8192 9.7 / 9.4,
// 16384 11.5 / 9.5; of 8192 entries with 1024 pages 9.0 / 10.3, 16384 with 8192 12.1 / 10.7;
// compaction of 2048 pages 7.6 / 9.3, 4096 10.7 / 11.4, 8192 19.4 / 19.1, 32768 67 / 55.
constexpr int PG_ONE_PAGES = 4096, PG_ONE_ENTRIES = 8192;
constexpr int PG_HEADS = 1024;  // lists of the sequences that write to a page, by its id
constexpr int PG_MASKS = 4;     // 32-page masks of its slice that a warp keeps
constexpr int PG_ROW = 4;       // table entries a lane has under way

__global__ void __launch_bounds__(PG_THREADS, 1) pages_fork_kernel(const __grid_constant__ PagesArgs a)
{
    cg::cluster_group cluster = cg::this_cluster();
    extern __shared__ int s_dyn[];
    __shared__ int s_free[PG_WARPS], s_bad, s_over, s_most, s_writers[PG_HEADS];
    __shared__ int4 s_cta[PG_CLUSTER];  // each CTA's free pages, bad entries, short tables
    __shared__ unsigned long long s_sh[2][PG_WARPS];
    const int nc = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int slices = nc * PG_WARPS, gw = rank * PG_WARPS + warp, gt = rank * PG_THREADS + tid;
    const int P = a.page_tokens, nmax = max(a.n_in, a.n_out);
    int *s_len = s_dyn;         // [n_out] length, -1: an empty sequence
    int *s_last = s_len + nmax; // [n_out] the partly filled last page it will write to, or -1
    int *s_next = s_last + nmax;  // [n_out] next of its parent's children
    int *s_also = s_next + nmax;  // [n_out] next of that page's writers
    int *s_off = s_also + nmax; // [n_in] first child of an old sequence; then [n_out] its place in the allocation
    int *s_copy = s_off + nmax; // [n_out] its place among the copies, or -1
    auto sync = [&] {
        if (nc > 1) cluster.sync();
        else __syncthreads();
    };
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

    if (tid == 0) s_bad = s_over = s_most = 0;
    for (int i = tid; i < a.n_in; i += PG_THREADS) s_off[i] = -1;
    s_writers[tid] = -1;
    static_assert(PG_HEADS == PG_THREADS, "one list head a thread");
    touch_params(a);
    asm volatile("griddepcontrol.wait;" ::: "memory");
    __syncthreads();
    if (a.refs_out != a.refs_in)
        for (int p = gt; p < a.n_pages; p += nc * PG_THREADS) a.refs_out[p] = a.refs_in[p];
    for (int j = tid; j < a.n_out; j += PG_THREADS) {
        const int p = a.src[j];
        int len = -1, last = -1;
        if (p >= 0) {
            len = p < a.n_in ? seq_len(a, p) : -1;
            if (len >= 0) s_next[j] = atomicExch(&s_off[p], j);
            else if (rank == 0) atomicAdd(&s_bad, 1);
            if (a.n_new > 0 && len > 0 && len % P && !(a.frozen && a.frozen[j])) {
                last = a.tables_in[(int64_t)p * a.width + len / P];
                if (last < 0 || last >= a.n_pages) last = -1;
                else s_also[j] = atomicExch(&s_writers[last % PG_HEADS], j);
            }
        }
        s_len[j] = len;
        s_last[j] = last;
    }
    for (int i = tid; i < a.n_in; i += PG_THREADS) atomicMax(&s_most, pages_of(max(seq_len(a, i), 0), P));
    sync();  // the counts are copied, the children listed, the longest old row known

    // each old sequence's row goes to its children; its pages lose its hold and gain theirs
    const int chunks = (s_most + PG_ROW * 32 - 1) / (PG_ROW * 32);
    for (int task = gw; task < a.n_in * chunks; task += slices) {  // (a GPU's memory holds under 2^31 chunks)
        const int i = task % a.n_in, c0 = task / a.n_in * (PG_ROW * 32) + lane;
        const int n = pages_of(max(seq_len(a, i), 0), P), first = s_off[i];
        if (c0 - lane >= n) continue;
        const int32_t *row = a.tables_in + (int64_t)i * a.width + c0;
        int v[PG_ROW], bad = 0, kids = 0;
#pragma unroll
        for (int k = 0; k < PG_ROW; k++) v[k] = c0 + k * 32 < n ? row[k * 32] : 0;
        for (int j = first; j >= 0; j = s_next[j], kids++) {
            int32_t *to = a.tables_out + (int64_t)j * a.width + c0;
#pragma unroll
            for (int k = 0; k < PG_ROW; k++)
                if (c0 + k * 32 < n) to[k * 32] = v[k];
        }
#pragma unroll
        for (int k = 0; k < PG_ROW; k++) {
            const bool in = c0 + k * 32 < n, page = v[k] >= 0 && v[k] < a.n_pages;
            if (in && page && kids != 1) atomicAdd(&a.refs_out[v[k]], kids - 1);
            bad += in && !page;
        }
        bad = __reduce_add_sync(FULLMASK, bad);
        if (lane == 0 && bad) atomicAdd(&s_bad, bad * kids);
    }
    sync();  // the counts are the fork's

    // free pages of each warp's slice
    const int per = (a.n_pages + slices - 1) / slices;
    const int64_t lo = (int64_t)gw * per;
    const int n_slice = (int)max((int64_t)0, min((int64_t)per, a.n_pages - lo));
    const int holds0 = tid < a.n_out && s_last[tid] >= 0 ? __ldcg(a.refs_out + s_last[tid]) : 0;  // (under way early)
    unsigned free_mask[PG_MASKS];  // of the slice's first pages
    {
        int n = 0;
#pragma unroll
        for (int k = 0; k < PG_MASKS; k++) {
            const int i = k * 32 + lane;
            free_mask[k] = __ballot_sync(FULLMASK, i < n_slice && __ldcg(a.refs_out + lo + i) <= 0);
            n += __popc(free_mask[k]);
        }
        for (int i0 = PG_MASKS * 32; i0 < n_slice; i0 += 32) {
            const int i = i0 + lane;
            n += __popc(__ballot_sync(FULLMASK, i < n_slice && __ldcg(a.refs_out + lo + i) <= 0));
        }
        if (lane == 0) s_free[warp] = n;
    }
    // every sequence's needs (a page that only one holds stays its own; of w writers of a
    // page with r holds, the first min(w, r - 1) copy it)
    unsigned long long base = 0;  // copies << 40 | pages
    for (int j0 = 0; j0 < a.n_out; j0 += PG_THREADS) {
        const int j = j0 + tid;
        int need = 0, copy = 0;
        if (j < a.n_out && s_len[j] >= 0 && a.n_new > 0 && !(a.frozen && a.frozen[j])) {
            const int len = s_len[j], last = s_last[j];
            if (last >= 0) {
                const int holds = j0 == 0 ? holds0 : __ldcg(a.refs_out + last);
                if (holds > 1) {
                    int before = 0;
                    for (int i = s_writers[last % PG_HEADS]; i >= 0; i = s_also[i]) before += s_last[i] == last && i < j;
                    copy = before < holds - 1;
                }
            }
            const int now = pages_of(len, P), then = pages_of(len + a.n_new, P);
            if (then > a.width) {
                if (rank == 0) atomicAdd(&s_over, 1);
            } else {
                need = copy + (then - now);
            }
        }
        unsigned long long total;
        const unsigned long long off = base + pg_scan((unsigned long long)copy << 40 | (uint32_t)need, &total, s_sh[j0 / PG_THREADS % 2]);
        if (j < a.n_out) {
            s_off[j] = (int)min(off & ((1ull << 40) - 1), 0x7fffffffull);
            s_copy[j] = copy ? (int)(off >> 40) : -1;
        }
        base += total;
    }
    const int64_t taken = (int64_t)(base & ((1ull << 40) - 1));
    __syncthreads();
    // each CTA's free pages, bad entries and short tables into every CTA's shared memory
    if (warp == 0) {
        const int n = __reduce_add_sync(FULLMASK, s_free[lane]);
        if (lane < nc) {
            int4 *to = nc > 1 ? cluster.map_shared_rank(s_cta, lane) : s_cta;
            to[rank] = make_int4(n, s_bad, s_over, 0);
        }
    }
    sync();
    const int4 cta = lane < nc ? s_cta[lane] : make_int4(0, 0, 0, 0);
    const int free_pages = __reduce_add_sync(FULLMASK, cta.x), bad = __reduce_add_sync(FULLMASK, cta.y);
    const int over = __reduce_add_sync(FULLMASK, cta.z);  // (counted by the first CTA alone)
    int k0 = __reduce_add_sync(FULLMASK, (lane < rank ? cta.x : 0) + (lane < warp ? s_free[lane] : 0));
    const bool ok = taken <= free_pages && over == 0 && bad == 0;
    if (ok && k0 < taken) {
        // the k-th free page belongs to the last sequence whose place is at or before k
        for (int i0 = 0; i0 < n_slice && k0 < taken; i0 += 32) {
            const int p = (int)lo + i0 + lane;
            unsigned b = 0;
            if (i0 < PG_MASKS * 32) {
#pragma unroll
                for (int k = 0; k < PG_MASKS; k++) b = i0 == k * 32 ? free_mask[k] : b;
            } else {
                b = __ballot_sync(FULLMASK, i0 + lane < n_slice && __ldcg(a.refs_out + p) <= 0);
            }
            const bool is = b >> lane & 1;
            const int k = k0 + __popc(b & ((1u << lane) - 1));
            k0 += __popc(b);
            if (!is || k >= taken) continue;
            int j = 0, hi = a.n_out - 1;
            while (j < hi) {
                const int mid = (j + hi + 1) / 2;
                if (s_off[mid] <= k) j = mid;
                else hi = mid - 1;
            }
            const int len = s_len[j], t = k - s_off[j], slot = s_copy[j];
            a.refs_out[p] = 1;
            if (slot >= 0 && t == 0) {
                a.tables_out[(int64_t)j * a.width + len / P] = p;
                a.copies[slot] = make_int4(s_last[j], p, len % P, 0);
                atomicSub(&a.refs_out[s_last[j]], 1);
            } else {
                a.tables_out[(int64_t)j * a.width + pages_of(len, P) + t - (slot >= 0)] = p;
            }
        }
    }
    if (rank == 0) {
        for (int j = tid; j < a.n_out; j += PG_THREADS) {
            const int len = max(s_len[j], 0);
            const bool grows = ok && s_len[j] >= 0 && !(a.frozen && a.frozen[j]);
            a.lens_out[j] = len + (grows ? a.n_new : 0);
        }
        if (tid == 0) {
            a.result[0] = ok ? (int)taken : 0;
            a.result[1] = (int)min(max(taken - free_pages, (int64_t)0), (int64_t)0x7fffffff);
            a.result[2] = over;
            a.result[3] = bad;
            *a.n_copies = ok ? (int)(base >> 40) : 0;
        }
    }
}

// Compaction: used pages at or above the number of used pages go to the free pages below
// it, the k-th to the k-th.  A warp walks a slice of the pages; every CTA has every slice's
// count in its shared memory.
__global__ void __launch_bounds__(PG_THREADS, 1) pages_compact_kernel(const __grid_constant__ PagesArgs a)
{
    cg::cluster_group cluster = cg::this_cluster();
    __shared__ int s_used[PG_SLICES];
    const int nc = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int slices = nc * PG_WARPS, gw = rank * PG_WARPS + warp, gt = rank * PG_THREADS + tid;
    const int per = (a.n_pages + slices - 1) / slices;
    const int64_t lo = (int64_t)gw * per;
    const int n_slice = (int)max((int64_t)0, min((int64_t)per, a.n_pages - lo));
    auto sync = [&] {
        if (nc > 1) cluster.sync();
        else __syncthreads();
    };
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    touch_params(a);
    sync();  // (every CTA runs, before any writes to another's shared memory)
    asm volatile("griddepcontrol.wait;" ::: "memory");

    int n = 0;
#pragma unroll 8
    for (int i = lane; i < n_slice; i += 32) n += a.refs_in[lo + i] > 0;
    n = __reduce_add_sync(FULLMASK, n);
    if (lane < nc) (nc > 1 ? cluster.map_shared_rank(s_used, lane) : s_used)[gw] = n;
    sync();
    // pages used, before this warp's slice, and below the border
    int used = 0, before = 0, below = 0;
    for (int i = lane; i < slices; i += 32) {
        used += s_used[i];
        before += i < gw ? s_used[i] : 0;
    }
    used = __reduce_add_sync(FULLMASK, used);
    before = __reduce_add_sync(FULLMASK, before);
    const int cut = used / per;  // the slice that holds the border (every page used: none)
    for (int i = lane; i < min(cut, slices); i += 32) below += s_used[i];
    for (int64_t p = (int64_t)cut * per + lane; p < used; p += 32) below += a.refs_in[p] > 0;
    below = __reduce_add_sync(FULLMASK, below);
    for (int i0 = 0; i0 < n_slice; i0 += 32) {
        const int p = (int)lo + i0 + lane;
        const bool in = i0 + lane < n_slice;
        const int refs = in ? a.refs_in[p] : 0;
        const unsigned b = __ballot_sync(FULLMASK, refs > 0);
        const int u = before + __popc(b & ((1u << lane) - 1));  // used pages below p
        before += __popc(b);
        const bool mv = refs > 0 && p >= used, hole = in && refs <= 0 && p < used;
        if (mv) a.moves[2 * (u - below)] = p;
        if (hole) a.moves[2 * (p - u) + 1] = p;
        if (in && !mv) a.page_map[p] = refs > 0 ? p : -1;
        if (in && !mv && !hole) a.refs_out[p] = refs > 0 ? refs : 0;
    }
    sync();  // the moves are listed
    for (int k = gt; k < used - below; k += nc * PG_THREADS) {
        const int from = __ldcg(a.moves + 2 * k), to = __ldcg(a.moves + 2 * k + 1);
        const int refs = a.refs_in[from];
        a.page_map[from] = to;
        a.refs_out[to] = refs;
        a.refs_out[from] = 0;
    }
    if (gt == 0) {
        a.result[0] = used;
        a.result[1] = used - below;
        a.result[2] = 0;
        a.result[3] = 0;
    }
}

// One chunk of a page: the first `fill` positions of its segments.
template <class V>
__device__ __forceinline__ void copy_chunk(const PoolArg &q, const char *src, char *dst, int fill, int chunk)
{
    const uint32_t cols = (uint32_t)fill * q.token_vecs, all = cols * (uint32_t)q.segs;
    auto place = [&](uint32_t c) {
        if (q.segs == 1) return (int64_t)c * (int64_t)sizeof(V);
        const uint32_t seg = c / cols;
        return (int64_t)seg * q.seg_stride + (int64_t)(c - seg * cols) * (int64_t)sizeof(V);
    };
    const uint32_t c0 = (uint32_t)chunk * (PC_THREADS * PC_VECS) + threadIdx.x;
    V v[PC_VECS];
#pragma unroll
    for (int i = 0; i < PC_VECS; i++)
        if (c0 + i * PC_THREADS < all) v[i] = *(const V *)(src + place(c0 + i * PC_THREADS));
#pragma unroll
    for (int i = 0; i < PC_VECS; i++)
        if (c0 + i * PC_THREADS < all) *(V *)(dst + place(c0 + i * PC_THREADS)) = v[i];
}

template <bool FORK>
__global__ void __launch_bounds__(PC_THREADS, PC_CTAS) pages_copy_kernel(const __grid_constant__ PagesArgs a, const __grid_constant__ PoolArgs pools)
{
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if constexpr (!FORK) {
        // a CTA an eighth of a sequence's entries, every eighth block of them
        for (int w = blockIdx.x; w < a.n_in * 8; w += gridDim.x) {
            const int i = w >> 3;
            const int64_t most = (int64_t)a.width * a.page_tokens;
            const int raw = a.lens_in[i];
            const int len = raw < 0 ? 0 : (int)min((int64_t)raw, most);
            int bad = (w & 7) == 0 && threadIdx.x == 0 && len != raw;
            for (int c = (w & 7) * PC_THREADS + threadIdx.x; c < pages_of(len, a.page_tokens); c += 8 * PC_THREADS) {
                const int64_t o = (int64_t)i * a.width + c;
                int p = a.tables_in[o];
                if (p >= 0 && p < a.n_pages) {
                    p = __ldcg(a.page_map + p);
                    bad += p < 0;
                } else {
                    bad++;
                }
                a.tables_out[o] = p;
            }
            if (bad) atomicAdd(&a.result[3], bad);
        }
    }
    if (pools.n == 0) return;
    const int n = FORK ? __ldcg(a.n_copies) : __ldcg(a.result + 1);
    // work item (k-th copy, pool, chunk), the CTAs' steps carried from digit to digit
    const int step_chunk = (int)(gridDim.x % (unsigned)pools.chunks), step_rest = (int)(gridDim.x / (unsigned)pools.chunks);
    const int step_pool = step_rest % pools.n, step_k = step_rest / pools.n;
    int chunk = (int)(blockIdx.x % (unsigned)pools.chunks), rest = (int)(blockIdx.x / (unsigned)pools.chunks);
    int pool = rest % pools.n, k = rest / pools.n;
    while (k < n) {
        int from, to, fill;
        if constexpr (FORK) {
            const int4 c = __ldcg(a.copies + k);
            from = c.x, to = c.y, fill = c.z;
        } else {
            const int2 c = __ldcg((const int2 *)a.moves + k);
            from = c.x, to = c.y, fill = a.page_tokens;
        }
        const PoolArg &q = pools.p[pool];
        const char *src = q.data + (int64_t)from * q.page_stride;
        char *dst = q.data + (int64_t)to * q.page_stride;
        if (q.width == 16) copy_chunk<uint4>(q, src, dst, fill, chunk);
        else if (q.width == 4) copy_chunk<uint32_t>(q, src, dst, fill, chunk);
        else copy_chunk<uint8_t>(q, src, dst, fill, chunk);
        chunk += step_chunk;
        pool += step_pool;
        k += step_k;
        if (chunk >= pools.chunks) {
            chunk -= pools.chunks;
            pool++;
        }
        if (pool >= pools.n) {
            pool -= pools.n;
            k++;
        }
    }
}

// The deciding kernels: one cluster, a programmatic dependent of what runs before.
static cudaError_t launch_cluster(void (*kernel)(PagesArgs), int ctas, int smem, const PagesArgs &a, cudaStream_t s)
{
    static bool ready[2][MAX_DEVICES] = {};
    const int dev = current_device();
    if (dev < 0 || dev >= MAX_DEVICES) return cudaErrorInvalidDevice;
    bool &done = ready[kernel == pages_fork_kernel][dev];
    if (!done) {
        cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (e == cudaSuccess && kernel == pages_fork_kernel)
            e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     pages_fork_smem(G4S_PAGES_MAX_SEQS, G4S_PAGES_MAX_SEQS));
        if (e != cudaSuccess) return e;
        done = true;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)ctas);
    cfg.blockDim = dim3(PG_THREADS);
    cfg.dynamicSmemBytes = (size_t)smem;
    cfg.stream = s;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned)ctas;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, kernel, a);
}

int pages_chunk_vecs() { return PC_THREADS * PC_VECS; }

int pages_fork_smem(int n_in, int n_out) { return 6 * (n_in > n_out ? n_in : n_out) * (int)sizeof(int); }

template <bool FORK>
static cudaError_t launch_copy(const PagesArgs &a, const PoolArgs &pools, int sms, cudaStream_t s)
{
    int64_t work = (int64_t)a.max_copies * pools.n * pools.chunks;
    if (!FORK && work < a.n_in * 8) work = a.n_in * 8;
    if (work == 0) return cudaSuccess;
    // a compaction's CTAs: as many as fit at once, or four times that where each of these would
    // have 6 pieces or more, so that they end together (one and four times: 2048 pieces 10.6
    // and 11.5 us, 4096 19.0 and 18.6, 16384 52.6 and 48.3; a CTA a piece 61.7).  A fork's
    // copies are few.
    const int64_t fit = (int64_t)sms * PC_CTAS, most = FORK || work < 6 * fit ? fit : 4 * fit;
    return launch_dependent(pages_copy_kernel<FORK>, work < most ? work : most, PC_THREADS, 0, s, a, pools);
}

cudaError_t launch_pages_fork(const PagesArgs &a, const PoolArgs &pools, int sms, cudaStream_t s)
{
    const bool one = a.n_pages <= PG_ONE_PAGES && (int64_t)a.n_in * a.width <= PG_ONE_ENTRIES;
    const cudaError_t e = launch_cluster(pages_fork_kernel, one ? 1 : PG_CLUSTER, pages_fork_smem(a.n_in, a.n_out), a, s);
    if (e != cudaSuccess || a.n_new == 0) return e;
    return launch_copy<true>(a, pools, sms, s);
}

cudaError_t launch_pages_compact(const PagesArgs &a, const PoolArgs &pools, int sms, cudaStream_t s)
{
    const cudaError_t e = launch_cluster(pages_compact_kernel, a.n_pages <= PG_ONE_PAGES ? 1 : PG_CLUSTER, 0, a, s);
    if (e != cudaSuccess) return e;
    return launch_copy<false>(a, pools, sms, s);
}

}  // namespace g4s
