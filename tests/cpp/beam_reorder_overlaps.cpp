// Which layouts of dense states g4s_beam_reorder takes for overlapping, without a GPU: the
// API's source built by the host compiler, its arguments' check against a byte-by-byte count
// over random small layouts.  Prints one line a failed check; exits 0 when all hold.
#include "../../gemma4.pas_b200/csrc/g4s_api.cu"

#include <map>
#include <random>

static int bad = 0;
static g4s_ctx C;

static int32_t reorder(const std::vector<g4s_beam_tensor> &t, int groups, int beams)
{
    static ReorderArgs a;
    int64_t blocks = 0;
    return beam_reorder_args(&C, "reorder", (int32_t *)4096, groups, beams, t.data(), (int)t.size(), a, blocks);
}

static void expect(int line, const std::vector<g4s_beam_tensor> &t, int groups, int beams, int32_t want, const char *text)
{
    const int32_t rc = reorder(t, groups, beams);
    if (rc == want && (rc == G4S_OK || strstr(g4s_last_error(&C), text))) return;
    printf("line %d: %d (%s), expected %d with '%s'\n", line, rc, g4s_last_error(&C), want, text);
    bad++;
}
#define EXPECT(t, groups, beams, want, text) expect(__LINE__, std::vector<g4s_beam_tensor> t, groups, beams, want, text)

// every byte of a tensor's segments, counted
static void bytes(const g4s_beam_tensor &t, const void *p, int rows, std::map<int64_t, int> &m)
{
    for (int64_t r = 0; r < rows; r++)
        for (int64_t i = 0; i < t.segs0; i++)
            for (int64_t j = 0; j < t.segs1; j++)
                for (int64_t b = 0; b < t.seg_bytes; b++)
                    m[(int64_t)(intptr_t)p + r * t.row_stride + i * t.stride0 + j * t.stride1 + b]++;
}

static bool overlap(const std::vector<g4s_beam_tensor> &ts, int rows)
{
    for (size_t i = 0; i < ts.size(); i++) {
        std::map<int64_t, int> d;
        bytes(ts[i], ts[i].dst, rows, d);
        for (auto &k : d)
            if (k.second > 1) return true;
        for (size_t j = 0; j < ts.size(); j++) {
            std::map<int64_t, int> o;
            if (j != i) bytes(ts[j], ts[j].dst, rows, o);
            if (j != i || ts[i].src != ts[i].dst) bytes(ts[j], ts[j].src, rows, o);
            for (auto &k : o)
                if (d.count(k.first)) return true;
        }
    }
    return false;
}

int main()
{
    char *A = (char *)(1 << 20), *B = (char *)(1 << 22);
    // [layers][rows][heads][max_len][dim] and its orders: 8 rows of 2 heads of 512 bytes, 256 in use, 3 layers
    EXPECT(({{A, B, 1024, 3, 8192, 2, 512, 256}}), 2, 4, G4S_OK, "");
    EXPECT(({{A, A, 1024, 3, 8192, 2, 512, 512}}), 2, 4, G4S_OK, "");
    EXPECT(({{A, A, 5120, 5, 1024, 2, 512, 512}}), 2, 4, G4S_OK, "");
    EXPECT(({{A, A, 512, 3, 8192, 2, 4096, 512}}), 2, 4, G4S_OK, "");
    EXPECT(({{A, A, 1023, 3, 8192, 2, 512, 512}}), 2, 4, G4S_ERR_ARG, "rows overlap");
    EXPECT(({{A, A, 1024, 3, 8191, 2, 512, 512}}), 2, 4, G4S_ERR_ARG, "rows overlap");
    EXPECT(({{A, A, 1024, 3, 1024, 2, 512, 512}}), 2, 4, G4S_ERR_ARG, "rows overlap");
    // two axes of one stride, where one counts 1
    EXPECT(({{A, A, 512, 1, 512, 1, 512, 512}}), 2, 4, G4S_OK, "");
    EXPECT(({{A, A, 0, 4, 512, 1, 0, 512}}), 1, 1, G4S_OK, "");
    // dst a byte off src, between src's rows, in the next layer
    EXPECT(({{A, A + 1, 1024, 1, 0, 1, 0, 1000}}), 2, 4, G4S_ERR_ARG, "dst overlaps src");
    EXPECT(({{A, A + 512, 1024, 1, 0, 1, 0, 512}}), 2, 4, G4S_OK, "");
    EXPECT(({{A, A + 512, 1024, 1, 0, 1, 0, 513}}), 2, 4, G4S_ERR_ARG, "dst overlaps src");
    EXPECT(({{A, A + 1024, 1024, 1, 0, 1, 0, 512}}), 2, 4, G4S_ERR_ARG, "dst overlaps src");
    EXPECT(({{A, A + 8192, 1024, 3, 16384, 2, 512, 512}}), 2, 4, G4S_OK, "");  // two buffers, layer by layer
    EXPECT(({{A, A + 8191, 1024, 3, 16384, 2, 512, 512}}), 2, 4, G4S_ERR_ARG, "dst overlaps src");
    // K and V side by side in each row
    EXPECT(({{A, A, 2048, 3, 16384, 2, 512, 512}, {A + 1024, A + 1024, 2048, 3, 16384, 2, 512, 512}}), 2, 4, G4S_OK, "");
    EXPECT(({{A, A, 2048, 3, 16384, 2, 512, 512}, {A + 1023, A + 1023, 2048, 3, 16384, 2, 512, 512}}), 2, 4, G4S_ERR_ARG, "where one is written");
    EXPECT(({{A, B, 64, 1, 0, 1, 0, 64}, {A, B + 4096, 64, 1, 0, 1, 0, 64}}), 2, 4, G4S_OK, "");  // one source, read twice
    EXPECT(({{A, B, 64, 1, 0, 1, 0, 64}, {A + 4096, B + 448, 64, 1, 0, 1, 0, 64}}), 2, 4, G4S_ERR_ARG, "where one is written");
    EXPECT(({{A, B, 64, 1, 0, 1, 0, 64}, {B, B + 4096, 64, 1, 0, 1, 0, 64}}), 2, 4, G4S_ERR_ARG, "where one is written");
    EXPECT(({{A, A, 64, 1, 0, 1, 0, 64}, {A, A, 64, 1, 0, 1, 0, 0}}), 2, 4, G4S_OK, "");  // an empty one
    // over the parents (8 numbers at 4096), and with them between two rows
    EXPECT(({{A, (void *)4096, 64, 1, 0, 1, 0, 64}}), 2, 4, G4S_ERR_ARG, "parents");
    EXPECT(({{A, (void *)4124, 64, 1, 0, 1, 0, 64}}), 2, 4, G4S_ERR_ARG, "parents");
    EXPECT(({{A, (void *)4128, 64, 1, 0, 1, 0, 64}}), 2, 4, G4S_OK, "");
    EXPECT(({{A, (void *)4064, 64, 1, 0, 1, 0, 32}}), 2, 4, G4S_OK, "");
    EXPECT(({{A, (void *)4064, 64, 1, 0, 1, 0, 33}}), 2, 4, G4S_ERR_ARG, "parents");
    EXPECT(({{(void *)4096, A, 4, 1, 0, 1, 0, 4}}), 2, 4, G4S_OK, "");  // read they may be
    // beyond 2^60 bytes
    EXPECT(({{A, A, (int64_t)1 << 61, 1, 0, 1, 0, 64}}), 2, 4, G4S_ERR_ARG, "2^60");
    EXPECT(({{A, A, INT64_MAX, 1, 0, 1, 0, 64}}), 2, 4, G4S_ERR_ARG, "2^60");
    EXPECT(({{A, A, 64, 0x7fffffff, INT64_MAX, 1, 0, 1}}), 1, 1, G4S_ERR_ARG, "2^60");
    EXPECT(({{A, A, (int64_t)1 << 50, 2, 64, 1, 0, 64}}), 2, 4, G4S_OK, "");

    // random small layouts, nested and not, one tensor and two
    std::mt19937 rng(1);
    auto upto = [&](int n) { return (int)(rng() % (unsigned)n); };
    int kinds[2] = {};
    for (int k = 0; k < 40000; k++) {
        const int groups = 1 + upto(2), beams = 1 + upto(3), rows = groups * beams;
        auto any = [&] {
            g4s_beam_tensor t{};
            t.seg_bytes = 1 + upto(4);
            t.segs0 = 1 + upto(3);
            t.segs1 = 1 + upto(3);
            if (upto(2)) {  // nested, in some order, with gaps
                int64_t s = t.seg_bytes + upto(3);
                int order[3] = {0, 1, 2};
                std::shuffle(order, order + 3, rng);
                for (int o : order) {
                    (o == 0 ? t.row_stride : o == 1 ? t.stride0 : t.stride1) = s;
                    s = s * (o == 0 ? rows : o == 1 ? t.segs0 : t.segs1) + upto(3) - (upto(8) == 0);
                    if (s < t.seg_bytes) s = t.seg_bytes;
                }
            } else {
                t.row_stride = t.seg_bytes + upto(40);
                t.stride0 = t.seg_bytes + upto(40);
                t.stride1 = t.seg_bytes + upto(40);
            }
            t.src = A + upto(120);
            t.dst = upto(3) ? A + upto(200) : (char *)t.src;
            return t;
        };
        std::vector<g4s_beam_tensor> ts{any()};
        if (upto(3) == 0) ts.push_back(any());
        const bool want = overlap(ts, rows);
        kinds[want]++;
        if ((reorder(ts, groups, beams) != G4S_OK) != want) {
            const g4s_beam_tensor &t = ts[0];
            printf("layout %d of %zu: rows %d x %lld, %d x %lld, %d x %lld, %lld bytes, dst %+lld: expected %d (%s)\n", k, ts.size(),
                   rows, (long long)t.row_stride, t.segs0, (long long)t.stride0, t.segs1, (long long)t.stride1,
                   (long long)t.seg_bytes, (long long)((char *)t.dst - (char *)t.src), want, g4s_last_error(&C));
            bad++;
        }
    }
    if (kinds[0] < 4000 || kinds[1] < 4000) bad++, printf("kinds %d %d\n", kinds[0], kinds[1]);

    // what the check costs: two tensors, every tensor there can be, side by side and interleaved
    for (int kind = 0; kind < 3; kind++) {
        std::vector<g4s_beam_tensor> ts;
        for (int i = 0; i < (kind ? G4S_BEAM_MAX_TENSORS : 2); i++) {
            char *p = kind == 2 ? A + i * 512 : A + (int64_t)i * (8 << 20);
            ts.push_back({p, p, 32 * 512, 8, 1 << 20, 2, 256, 256});
        }
        const auto t0 = std::chrono::steady_clock::now();
        for (int i = 0; i < 1000; i++)
            if (reorder(ts, 8, 8) != G4S_OK) bad++, puts(g4s_last_error(&C));
        printf("%.2f us for %zu tensors\n", std::chrono::duration<double>(std::chrono::steady_clock::now() - t0).count() * 1e3, ts.size());
    }
    printf(bad ? "%d failed\n" : "ok\n", bad);
    return bad != 0;
}
