// Overlaps (and ranges) that the beam selection refuses, without a GPU: the API's source built by
// the host compiler around a context that was never created (the checks come before any CUDA
// call).  Prints one line a failed check; exits 0 when all hold.
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
static char *at(uintptr_t a) { return (char *)a; }

// 8 rows of 100 logits, 120 apart: 8 * 4 bytes of scores and lens, 8 of done
struct Select {
    char *logits = at(1 << 20), *in[3] = {at(4096), at(8192), at(12288)};
    char *out[5] = {at(16384), at(20480), at(24576), at(28672), at(32768)};  // scores, lens, done, parents, tokens
    int32_t dtype = G4S_F32;
    int64_t stride = 120;
    float cap = 30.0f;
    g4s_beam_params p;
    Select() { g4s_beam_params_defaults(&p); }
    int32_t run()
    {
        BeamArgs a;
        bool vec;
        const g4s_beam_state i{(float *)in[0], (int32_t *)in[1], (uint8_t *)in[2]}, o{(float *)out[0], (int32_t *)out[1], (uint8_t *)out[2]};
        return beam_select_args(&C, "select", logits, dtype, 2, 100, stride, cap, &p, &i, &o, (int32_t *)out[3],
                                (int32_t *)out[4], a, vec);
    }
};
static const int SIZE[5] = {32, 32, 8, 32, 32};  // bytes of the outputs, and of in's by the same name

int main()
{
    C.max_rows = 64;
    C.max_vocab = 1000;
    EXPECT(Select().run(), G4S_OK, "");
    // an output against every input: the last byte of it, the first, right behind, right before
    for (int o = 0; o < 5; o++) {
        for (int i = 0; i < 3; i++) {
            const int step = o == 2 ? 1 : 4;
            for (int64_t by : {(int64_t)0, (int64_t)SIZE[i] - step, (int64_t)SIZE[i], (int64_t)step - SIZE[o], -(int64_t)SIZE[o]}) {
                Select s;
                s.out[o] = s.in[i] + by;
                const bool apart = by >= SIZE[i] || by <= -SIZE[o], same = by == 0 && o == i;
                EXPECT(s.run(), apart || same ? G4S_OK : G4S_ERR_ARG, "overlaps");
                s.p.n_out = 3;  // (8 rows in, 6 out: in place no more)
                if (same) EXPECT(s.run(), G4S_ERR_ARG, "overlaps");
            }
        }
        for (int q = 0; q < 5; q++) {
            if (q == o) continue;
            Select s;
            s.out[o] = s.out[q];
            EXPECT(s.run(), G4S_ERR_ARG, "overlaps");
            s.out[o] = s.out[q] + SIZE[q];
            EXPECT(s.run(), G4S_OK, "");
            s.out[o] = s.out[q] + SIZE[q] - (o == 2 ? 1 : 4);
            EXPECT(s.run(), G4S_ERR_ARG, "overlaps");
        }
        // against the logits: a row's first and last byte, between two rows, behind the last
        for (int row : {0, 1, 7}) {
            Select s;
            char *r = s.logits + row * 480;
            s.out[o] = r;
            EXPECT(s.run(), G4S_ERR_ARG, "overlaps");
            s.out[o] = r + 396;
            EXPECT(s.run(), G4S_ERR_ARG, "overlaps");
            s.out[o] = r + 400;
            EXPECT(s.run(), G4S_OK, "");
            s.out[o] = r - SIZE[o];
            EXPECT(s.run(), G4S_OK, "");
            s.out[o] = r - SIZE[o] + (o == 2 ? 1 : 4);
            EXPECT(s.run(), G4S_ERR_ARG, "overlaps");
        }
    }
    {
        Select s;  // in place, and lens and done left out
        for (int i = 0; i < 3; i++) s.out[i] = s.in[i];
        EXPECT(s.run(), G4S_OK, "");
        s.in[1] = s.in[2] = s.out[1] = s.out[2] = nullptr;
        EXPECT(s.run(), G4S_OK, "");
        s.in[1] = s.in[0];  // inputs may share
        EXPECT(s.run(), G4S_ERR_ARG, "overlaps");  // (but not with an output that is another of them)
        s.out[0] = at(16384);
        EXPECT(s.run(), G4S_OK, "");
    }
    // a softcap beyond 1e8 temperatures
    { Select s; s.cap = 200.0f; s.p.temperature = 1e-6; EXPECT(s.run(), G4S_ERR_ARG, "temperature"); }
    { Select s; s.cap = 1e6f; s.p.temperature = 0.0099; EXPECT(s.run(), G4S_ERR_ARG, "temperature"); }
    { Select s; s.cap = 1e6f; s.p.temperature = 0.01; EXPECT(s.run(), G4S_OK, ""); }
    { Select s; s.cap = 100.0f; s.p.temperature = 1e-6; EXPECT(s.run(), G4S_OK, ""); }
    { Select s; s.cap = 0.0f; s.p.temperature = 1e-6; EXPECT(s.run(), G4S_OK, ""); }
    { Select s; s.stride = (int64_t)1 << 58; EXPECT(s.run(), G4S_ERR_ARG, "row_stride"); }
    { Select s; s.stride = (int64_t)1 << 62; EXPECT(s.run(), G4S_ERR_ARG, "row_stride"); }
    { Select s; s.stride = (int64_t)1 << 40; EXPECT(s.run(), G4S_OK, ""); }
    printf(bad ? "%d failed\n" : "ok\n", bad);
    return bad != 0;
}
