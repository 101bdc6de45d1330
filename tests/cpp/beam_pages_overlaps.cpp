// Overlaps that g4s_pages_fork, g4s_pages_compact and g4s_beam_step refuse, without a GPU: the
// API's source built by the host compiler around a context that was never created (the checks
// come before any CUDA call).  Prints one line a failed check; exits 0 when all hold.
#include "../../gemma4.pas_b200/csrc/g4s_api.cu"

static int bad = 0;
static g4s_ctx C;

static void expect(int line, int a, int b, int32_t rc, int32_t want, const char *text)
{
    if (rc == want && (rc == G4S_OK || strstr(g4s_last_error(&C), text))) return;
    printf("line %d (%d, %d): %d (%s), expected %d with '%s'\n", line, a, b, rc, g4s_last_error(&C), want, text);
    bad++;
}

// addresses that are never followed, 64 KiB apart
static char *at(int i) { return (char *)(uintptr_t)((i + 1) << 16); }

// 4 sequences of up to 6 pages, 50 pages
enum { IT, IL, IR, SRC, FZ, OT, OL, OR, RES, N };
static const int SIZE[N] = {96, 16, 200, 16, 4, 96, 16, 200, 16};
static int32_t fork(char *const (&p)[N])
{
    const g4s_page_cache cache{4, 50, 6, 0, nullptr};
    const g4s_page_tables in{(int32_t *)p[IT], (int32_t *)p[IL], (int32_t *)p[IR]}, out{(int32_t *)p[OT], (int32_t *)p[OL], (int32_t *)p[OR]};
    PagesArgs a;
    static PoolArgs pools;
    return pages_fork_args(&C, "fork", &cache, 4, &in, 4, (int32_t *)p[SRC], 1, (uint8_t *)p[FZ], &out, (int32_t *)p[RES], a, pools);
}

int main()
{
    C.max_rows = 64;
    C.max_vocab = 1000;
    char *base[N], *p[N];
    auto reset = [&] { for (int i = 0; i < N; i++) p[i] = base[i] = at(i); };
    reset();
    expect(__LINE__, 0, 0, fork(p), G4S_OK, "");
    for (int o = OT; o < N; o++) {
        for (int i = 0; i < N; i++) {
            if (i == o) continue;
            reset();
            p[o] = base[i];
            const bool same = (o == OL && i == IL) || (o == OR && i == IR);
            expect(__LINE__, o, i, fork(p), same ? G4S_OK : G4S_ERR_ARG, "overlap");
            p[o] = base[i] + (SIZE[i] - 1) / 4 * 4;  // its last element
            expect(__LINE__, o, i, fork(p), G4S_ERR_ARG, "overlap");
            p[o] = base[i] + SIZE[i];
            expect(__LINE__, o, i, fork(p), G4S_OK, "");
            p[o] = base[i] - SIZE[o];
            expect(__LINE__, o, i, fork(p), G4S_OK, "");
        }
    }
    reset();
    p[FZ] = nullptr;
    p[SRC] = p[IL];  // inputs may share
    expect(__LINE__, 0, 0, fork(p), G4S_OK, "");
    // nothing is compared with arrays of no sequence
    {
        const g4s_page_cache cache{4, 50, 6, 0, nullptr};
        const g4s_page_tables in{(int32_t *)at(0), (int32_t *)at(0), (int32_t *)at(2)}, out{(int32_t *)at(2), (int32_t *)at(2), (int32_t *)at(2)};
        PagesArgs a;
        static PoolArgs pools;
        expect(__LINE__, 0, 0, pages_fork_args(&C, "fork", &cache, 0, &in, 0, nullptr, 1, nullptr, &out, (int32_t *)at(8), a, pools), G4S_OK, "");
    }
    // compaction (its checks end in a launch, so only refusals)
    {
        const g4s_page_cache cache{4, 50, 6, 0, nullptr};
        char *q[8] = {at(0), at(1), at(2), at(3), at(4), at(5), at(6), at(7)};  // in: tables lens refs; out: tables refs; map moves result
        static const int size[8] = {96, 16, 200, 96, 200, 200, 200, 16};
        for (int o = 3; o < 8; o++)
            for (int i = 0; i < 8; i++) {
                char *r[8];
                memcpy(r, q, sizeof(q));
                if (i == o) continue;
                r[o] = q[i] + size[i] - 8;
                const g4s_page_tables in{(int32_t *)r[0], (int32_t *)r[1], (int32_t *)r[2]}, out{(int32_t *)r[3], nullptr, (int32_t *)r[4]};
                expect(__LINE__, o, i, g4s_pages_compact(&C, &cache, 4, &in, &out, (int32_t *)r[5], (int32_t *)r[6], (int32_t *)r[7], nullptr),
                       G4S_ERR_ARG, "overlap");
            }
    }
    // a step: what the selection writes against what the fork reads and writes
    {
        g4s_beam_params par;
        g4s_beam_params_defaults(&par);
        for (int o = 0; o < 5; o++)
            for (int i = 0; i < 7; i++) {
                reset();
                char *s[5] = {at(20), at(21), at(22), at(23), at(24)};
                const int arrays[7] = {IT, IL, IR, OT, OL, OR, RES};
                s[o] = p[arrays[i]] + SIZE[arrays[i]] - 4;
                const g4s_beam_state before{(float *)at(25), (int32_t *)at(26), (uint8_t *)at(27)};
                const g4s_beam_state after{(float *)s[0], (int32_t *)s[1], (uint8_t *)s[2]};
                const g4s_page_cache cache{4, 50, 6, 0, nullptr};
                const g4s_beam_pages pages{&cache, {(int32_t *)p[IT], (int32_t *)p[IL], (int32_t *)p[IR]},
                                           {(int32_t *)p[OT], (int32_t *)p[OL], (int32_t *)p[OR]}, 1, (int32_t *)p[RES]};
                expect(__LINE__, o, i, g4s_beam_step(&C, at(30), G4S_F32, 1, 100, 100, 30.0f, &par, &before, &after, (int32_t *)s[3],
                                                     (int32_t *)s[4], nullptr, 0, &pages, nullptr), G4S_ERR_ARG, "overlap");
            }
    }
    printf(bad ? "%d failed\n" : "ok\n", bad);
    return bad != 0;
}
