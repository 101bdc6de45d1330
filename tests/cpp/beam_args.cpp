// The argument checks of the beam-search entry points without a GPU: the API's source built
// by the host compiler around a context that was never created (its checks come before any
// CUDA call).  Prints one line a failed check; exits 0 when all hold.
#include "../../gemma4.pas_b200/csrc/g4s_api.cu"

static int bad = 0;
static g4s_ctx C;

static void expect(int line, int32_t rc, int32_t want, const char *text)
{
    if (rc == want && (rc == G4S_OK || strstr(g4s_last_error(&C), text))) return;
    printf("line %d: %d (%s), expected %d with '%s'\n", line, rc, g4s_last_error(&C), want, text);
    bad++;
}
#define EXPECT(rc, want, text) expect(__LINE__, rc, want, text)

// addresses that are never followed
static void *at(uintptr_t a) { return (void *)a; }
static int32_t *ints(uintptr_t a) { return (int32_t *)at(a); }

struct Select {
    const void *logits = at(1 << 20);
    int32_t dtype = G4S_F32, groups = 2, vocab = 100;
    int64_t stride = 100;
    float cap = 30.0f;
    g4s_beam_params p;
    g4s_beam_state in{(float *)at(4096), ints(8192), (uint8_t *)at(12288)};
    g4s_beam_state out{(float *)at(16384), ints(20480), (uint8_t *)at(24576)};
    int32_t *parents = ints(28672), *tokens = ints(32768);
    Select() { g4s_beam_params_defaults(&p); }
    int32_t run()
    {
        BeamArgs a;
        bool vec;
        return beam_select_args(&C, "select", logits, dtype, groups, vocab, stride, cap, &p, &in, &out, parents, tokens, a, vec);
    }
};

struct Fork {
    g4s_page_pool pool{at(1 << 20), 64, 1, 0, 16};
    g4s_page_cache cache{4, 8, 2, 1, &pool};
    g4s_page_tables in{ints(4096), ints(8192), ints(12288)}, out{ints(16384), ints(20480), ints(24576)};
    int32_t n_in = 2, n_out = 2, n_new = 1;
    int32_t *src = ints(28672), *result = ints(32768);
    int32_t run()
    {
        PagesArgs a;
        PoolArgs pools;
        return pages_fork_args(&C, "fork", &cache, n_in, &in, n_out, src, n_new, nullptr, &out, result, a, pools);
    }
};

static int32_t reorder(const g4s_beam_tensor &t, ReorderArgs &a, int64_t &blocks, int groups = 2, int beams = 4)
{
    return beam_reorder_args(&C, "reorder", ints(4096), groups, beams, &t, 1, a, blocks);
}

int main()
{
    C.max_rows = 64;
    C.max_vocab = 1000;
    EXPECT(Select().run(), G4S_OK, "");
#define SELECT(change, want, text) { Select s; s.change; EXPECT(s.run(), want, text); }
    SELECT(logits = nullptr, G4S_ERR_ARG, "non-NULL")
    SELECT(in.scores = nullptr, G4S_ERR_ARG, "non-NULL")
    SELECT(out.scores = nullptr, G4S_ERR_ARG, "non-NULL")
    SELECT(tokens = nullptr, G4S_ERR_ARG, "non-NULL")
    SELECT(dtype = 7, G4S_ERR_ARG, "dtype")
    SELECT(p.beams = 33, G4S_ERR_ARG, "beams")
    SELECT(p.n_out = 65, G4S_ERR_ARG, "n_out")
    SELECT(groups = 0, G4S_ERR_ARG, "groups")
    SELECT(groups = 17, G4S_ERR_CAPACITY, "exceed")
    SELECT(groups = 0x7fffffff, G4S_ERR_CAPACITY, "exceed")
    { Select s; s.vocab = 1001; s.stride = 1001; EXPECT(s.run(), G4S_ERR_CAPACITY, "exceed"); }
    SELECT(stride = 99, G4S_ERR_ARG, "row_stride")
    SELECT(logits = at((1 << 20) + 2), G4S_ERR_ARG, "aligned")
    SELECT(in.scores = (float *)at(4098), G4S_ERR_ARG, "aligned")
    SELECT(out.lens = ints(20481), G4S_ERR_ARG, "aligned")
    SELECT(parents = ints(28674), G4S_ERR_ARG, "aligned")
    SELECT(tokens = ints(32771), G4S_ERR_ARG, "aligned")
    SELECT(in.done = (uint8_t *)at(12289), G4S_OK, "")
    SELECT(p.temperature = 0.0, G4S_ERR_ARG, "temperature")
    SELECT(p.temperature = NAN, G4S_ERR_ARG, "temperature")
    SELECT(p.length_alpha = NAN, G4S_ERR_ARG, "length_alpha")
    SELECT(p.length_alpha = -1.0, G4S_ERR_ARG, "length_alpha")
    SELECT(cap = NAN, G4S_ERR_ARG, "softcap")
    SELECT(cap = INFINITY, G4S_ERR_ARG, "softcap")
    SELECT(cap = -INFINITY, G4S_OK, "")
    SELECT(p.n_eos = 9, G4S_ERR_ARG, "n_eos")
    SELECT(in.lens = nullptr, G4S_ERR_ARG, "lens")
    SELECT(out = s.in, G4S_OK, "")
    { Select s; s.out = s.in; s.p.n_out = 5; EXPECT(s.run(), G4S_ERR_ARG, "overlaps"); }
    SELECT(out.scores = s.in.scores + 7, G4S_ERR_ARG, "overlaps")
    SELECT(out.scores = s.in.scores + 8, G4S_OK, "")
    SELECT(out.done = s.in.done - 7, G4S_ERR_ARG, "overlaps")
    { Select s; s.out.lens = nullptr; s.out.done = nullptr; s.in.lens = nullptr; s.in.done = nullptr; EXPECT(s.run(), G4S_OK, ""); }

    ReorderArgs a;
    int64_t blocks = 0;
    g4s_beam_tensor t{at(1 << 20), at(1 << 21), 1024, 3, 8192, 2, 512, 256};
    EXPECT(reorder(t, a, blocks), G4S_OK, "");
    if (a.n != 1 || a.t[0].width != 16 || a.t[0].seg_cols != 16 || a.t[0].cols != 96 || a.t[0].blocks != 1 || blocks != 2) bad++, puts("columns");
    t.seg_bytes = 252;
    EXPECT(reorder(t, a, blocks), G4S_OK, "");
    if (a.t[0].width != 4 || a.t[0].cols != 6 * 63) bad++, puts("columns of 4");
    t.src = at((1 << 20) + 1);
    EXPECT(reorder(t, a, blocks), G4S_OK, "");
    if (a.t[0].width != 1 || a.t[0].blocks != (6 * 252 + REORDER_THREADS - 1) / REORDER_THREADS) bad++, puts("columns of 1");
    t.seg_bytes = 0;
    EXPECT(reorder(t, a, blocks), G4S_OK, "");
    if (a.n != 0 || blocks != 0) bad++, puts("an empty tensor");
#define REORDER(change, want, text) { g4s_beam_tensor t{at(1 << 20), at(1 << 21), 1024, 3, 8192, 2, 512, 256}; t.change; EXPECT(reorder(t, a, blocks), want, text); }
    REORDER(src = nullptr, G4S_ERR_ARG, "NULL")
    REORDER(row_stride = 255, G4S_ERR_ARG, "row_stride")
    REORDER(stride1 = 255, G4S_ERR_ARG, "overlap")
    REORDER(stride0 = -16, G4S_ERR_ARG, "negative")
    REORDER(segs0 = 0, G4S_ERR_ARG, "no segment")
    REORDER(seg_bytes = -1, G4S_ERR_ARG, "negative")
    { g4s_beam_tensor t{at(1 << 20), at(1 << 21), (int64_t)1 << 41, 1, 0, 1, 0, (int64_t)1 << 40}; EXPECT(reorder(t, a, blocks), G4S_ERR_CAPACITY, "columns"); }
    { g4s_beam_tensor t{at(1 << 20), at(1 << 21), 16, 1, 0, 1, 0, 16}; EXPECT(reorder(t, a, blocks, 1, 33), G4S_ERR_ARG, "beams"); }
    { g4s_beam_tensor t{at(1 << 20), at(1 << 21), (int64_t)1 << 34, 1, 0, 1, 0, (int64_t)1 << 33}; EXPECT(reorder(t, a, blocks, 1 << 20, 32), G4S_ERR_CAPACITY, "blocks"); }
    EXPECT(beam_reorder_args(&C, "reorder", ints(4096), 1, 4, nullptr, 33, a, blocks), G4S_ERR_ARG, "n_tensors");
    EXPECT(beam_reorder_args(&C, "reorder", ints(4098), 1, 4, nullptr, 0, a, blocks), G4S_ERR_ARG, "aligned");
    EXPECT(beam_reorder_args(&C, "reorder", ints(4096), 1, 4, nullptr, 1, a, blocks), G4S_ERR_ARG, "NULL");

    EXPECT(Fork().run(), G4S_OK, "");
#define FORK(change, want, text) { Fork s; s.change; EXPECT(s.run(), want, text); }
    FORK(cache.page_tokens = 0, G4S_ERR_ARG, "page_tokens")
    FORK(cache.n_pages = 1 << 30, G4S_ERR_ARG, "2^30")
    FORK(cache.max_seq_pages = 1 << 29, G4S_ERR_ARG, "2^30")
    FORK(cache.n_pools = 97, G4S_ERR_ARG, "n_pools")
    FORK(cache.pools = nullptr, G4S_ERR_ARG, "n_pools")
    { Fork s; s.cache.n_pools = 0; s.cache.pools = nullptr; EXPECT(s.run(), G4S_OK, ""); }
    FORK(pool.data = nullptr, G4S_ERR_ARG, "NULL data")
    FORK(pool.page_stride = 63, G4S_ERR_ARG, "overlap")
    FORK(pool.token_bytes = 0, G4S_ERR_ARG, "size")
    { Fork s; s.pool.segs = 2; s.pool.seg_stride = 63; s.pool.page_stride = 200; EXPECT(s.run(), G4S_ERR_ARG, "overlap"); }
    { Fork s; s.pool.token_bytes = (int64_t)1 << 36; s.pool.page_stride = (int64_t)1 << 40; EXPECT(s.run(), G4S_ERR_CAPACITY, "vectors"); }
    // strides whose product is beyond 64 bits
    { Fork s; s.pool.segs = 3; s.pool.seg_stride = (int64_t)1 << 62; s.pool.page_stride = 4096; EXPECT(s.run(), G4S_ERR_ARG, "overlap"); }
    { Fork s; s.pool.segs = 5; s.pool.seg_stride = (int64_t)1 << 62; s.pool.page_stride = 4096; EXPECT(s.run(), G4S_ERR_ARG, "overlap"); }
    { Fork s; s.pool.segs = 3; s.pool.seg_stride = 96; s.pool.page_stride = 256; EXPECT(s.run(), G4S_OK, ""); }
    { Fork s; s.pool.segs = 3; s.pool.seg_stride = 96; s.pool.page_stride = 255; EXPECT(s.run(), G4S_ERR_ARG, "overlap"); }
    FORK(in.tables = ints(4097), G4S_ERR_ARG, "aligned")
    FORK(in.refs = ints(12290), G4S_ERR_ARG, "aligned")
    FORK(out.lens = ints(20483), G4S_ERR_ARG, "aligned")
    FORK(src = ints(28673), G4S_ERR_ARG, "aligned")
    FORK(result = ints(32770), G4S_ERR_ARG, "aligned")
    FORK(n_in = -1, G4S_ERR_ARG, "n_in")
    FORK(n_out = 65, G4S_ERR_CAPACITY, "n_out")
    FORK(n_new = -1, G4S_ERR_ARG, "n_new")
    FORK(src = nullptr, G4S_ERR_ARG, "non-NULL")
    FORK(result = nullptr, G4S_ERR_ARG, "non-NULL")
    FORK(out.tables = s.in.tables, G4S_ERR_ARG, "tables")
    FORK(out.tables = s.in.tables + 3, G4S_ERR_ARG, "tables")
    FORK(out.tables = s.in.tables + 4, G4S_OK, "")
    FORK(out.refs = s.in.refs, G4S_OK, "")
    FORK(out.refs = s.in.refs + 7, G4S_ERR_ARG, "refs or lens")
    FORK(out.lens = s.in.lens + 1, G4S_ERR_ARG, "refs or lens")
    { Fork s; s.n_in = s.n_out = 0; s.in.tables = s.in.lens = s.out.tables = s.out.lens = s.src = nullptr; EXPECT(s.run(), G4S_OK, ""); }
    // a compaction's and a step's own checks
    {
        Fork s;
        EXPECT(g4s_pages_compact(&C, &s.cache, 2, &s.in, &s.out, ints(40960), ints(45060), s.result, nullptr), G4S_ERR_ARG, "aligned");
        EXPECT(g4s_pages_compact(&C, &s.cache, 2, &s.in, &s.out, nullptr, ints(45056), s.result, nullptr), G4S_ERR_ARG, "page_map");
        EXPECT(g4s_pages_compact(&C, &s.cache, 2, &s.in, &s.out, ints(40962), ints(45056), s.result, nullptr), G4S_ERR_ARG, "aligned");
        s.out.tables = s.in.tables + 1;
        EXPECT(g4s_pages_compact(&C, &s.cache, 2, &s.in, &s.out, ints(40960), ints(45056), s.result, nullptr), G4S_ERR_ARG, "overlap");
        Select q;
        q.p.n_out = 5;
        EXPECT(g4s_beam_step(&C, q.logits, q.dtype, 2, 100, 100, 30.0f, &q.p, &q.in, &q.out, q.parents, q.tokens, nullptr, 0, nullptr, nullptr),
               G4S_ERR_ARG, "n_out");
        q.p.n_out = 4;
        g4s_beam_pages pages{&s.cache, s.in, s.in, 1, s.result};
        EXPECT(g4s_beam_step(&C, q.logits, q.dtype, 2, 100, 100, 30.0f, &q.p, &q.in, &q.out, q.parents, q.tokens, nullptr, 0, &pages, nullptr),
               G4S_ERR_ARG, "tables");
        EXPECT(g4s_beam_step(&C, q.logits, q.dtype, 2, 100, 100, 30.0f, &q.p, &q.in, &q.out, q.parents, q.tokens, nullptr, 1, nullptr, nullptr),
               G4S_ERR_ARG, "NULL");
    }
    // entry points without a context
    if (g4s_beam_select(nullptr, nullptr, 0, 1, 1, 1, 0, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr) != G4S_ERR_ARG ||
        g4s_beam_reorder(nullptr, nullptr, 1, 1, nullptr, 0, nullptr) != G4S_ERR_ARG ||
        g4s_pages_fork(nullptr, nullptr, 0, nullptr, 0, nullptr, 0, nullptr, nullptr, nullptr, nullptr) != G4S_ERR_ARG ||
        g4s_pages_compact(nullptr, nullptr, 0, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr) != G4S_ERR_ARG ||
        g4s_beam_step(nullptr, nullptr, 0, 1, 1, 1, 0, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, 0, nullptr, nullptr) != G4S_ERR_ARG)
        bad++, puts("a NULL context");
    printf(bad ? "%d failed\n" : "ok\n", bad);
    return bad != 0;
}
