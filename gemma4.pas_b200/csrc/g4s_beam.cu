// g4s_beam.cu -- beam search beside the sampler: the selection over beams x
// vocabulary (beam_stream_kernel, beam_combine_kernel) and the reordering of
// the beams' dense states (beam_reorder_kernel).  No counterpart in the
// reference, whose TModel.Generate (src/Gemma4.Model.pas:2829-2938) keeps one
// sequence.
//
// Selection.  With x_i = cap * tanh(l_i / cap) / T (masked logits left out) and
// lse = log sum_i exp(x_i), token i continues beam w with the score
//   scores[w] + x_i - lse,   ranked by  score / max(len, 1)^alpha,
// and a prompt's n_out best continuations over its beams are wanted.  Within a
// beam the rank is increasing in the raw logit, so only raw comparisons order
// a beam's tokens; the beams' own scores meet in 64 bits, for the few tokens
// that can be among the best.
//
// beam_stream_kernel: one pass over the logits.  An item is a whole number of
//   2 KiB units of one row (one unit up to 512 units a row); a warp reduces it
//   to (largest raw logit m, its softcapped value c, S = sum 2^((s_i - c) k)),
//   k = log2(e) / T.  The difference s_i - c is taken before the product with
//   k, so that k's rounding acts on the distance from the maximum only.
// beam_combine_kernel: one CTA a prompt.
//   1. a warp a beam: lse from the items in 64 bits, and the beam's n_out
//      items with the largest (m, then lowest item);
//   2. those items' best tokens ranked over the beams: the n_out best tokens
//      lie in the n_out items that rank first (each item that ranks before
//      another holds a token that beats all of the other's);
//   3. these items reread, their tokens above the beam's best item left out
//      collected (at most n_out - j from the item in place j), ranked, sorted.
#include "g4s_device.cuh"
#include "g4s_kernels.cuh"

namespace g4s {

constexpr int BS_THREADS = 256;  // CTA of the streaming pass
constexpr int BC_THREADS = 512;  // CTA of the combine
constexpr int BC_WARPS = BC_THREADS / 32;
constexpr int BNV = 4;           // 16-byte vectors a lane and unit (2 KiB a unit)
constexpr int BIPL = BEAM_MAX_ITEMS / 32;  // a row's items a lane of its warp

template <int DT>
struct BeamGeo {
    static constexpr int VW = DtypeTraits<DT>::VW;
    static constexpr int EPL = BNV * VW;    // a lane's logits of a unit
    static constexpr int UNIT = 32 * EPL;   // 512 fp32 or 1024 bf16 logits
};

int beam_unit_logits(int dtype) { return dtype == G4S_F32 ? BeamGeo<G4S_F32>::UNIT : BeamGeo<G4S_BF16>::UNIT; }

// A masked logit (NaN, or at or below -1e30 as on the top-K path) is -inf; +inf counts
// as the largest finite number, so that differences stay defined; -0 is +0.
__device__ __forceinline__ float beam_raw(float v)
{
    return v > -1e30f ? fminf(v, 3.402823466e38f) + 0.0f : -__uint_as_float(0x7f800000u);
}
__device__ __forceinline__ uint32_t beam_key(float v) { return cand_key(beam_raw(v)); }

// cap * tanh(v / cap) in fp32: the polynomial up to |q| = 1, 1 - 2 / (e^2q + 1) beyond
// (2 / (e^2q + 1) < 0.24 there, so the approximate exponential and quotient cost less
// than half an ulp of the result).
template <bool CAP>
__device__ __forceinline__ float beam_soft(float v, const BeamArgs &a)
{
    if (!CAP) return v;
    const float q = __fmul_rn(v, a.invcap), aq = fabsf(q);
    const float w = 1.0f - __fdividef(2.0f, ex2_approx(aq * (2.0f * G4_L2E)) + 1.0f);
    return __fmul_rn(aq <= 1.0f ? tanh_poly(q) : copysignf(w, q), a.softcap);
}

// One unit's vectors of this lane: logit (j, k) is unit position (j * 32 + lane) * VW + k.
// Rows that are not 16-byte aligned are gathered element by element into the same places,
// so that a row's sums do not depend on its alignment.
template <int DT, bool VEC>
__device__ __forceinline__ void load_unit(const char *p, int lane, uint4 (&r)[BNV])
{
    using T = DtypeTraits<DT>;
#pragma unroll
    for (int j = 0; j < BNV; j++) {
        const int e0 = (j * 32 + lane) * T::VW;
        if constexpr (VEC) {
            r[j] = ld_stream_v4(p + (int64_t)e0 * T::ESIZE);
        } else if constexpr (DT == G4S_F32) {
            const float *f = (const float *)p + e0;
            r[j] = make_uint4(__float_as_uint(__ldg(f)), __float_as_uint(__ldg(f + 1)), __float_as_uint(__ldg(f + 2)),
                              __float_as_uint(__ldg(f + 3)));
        } else {
            const unsigned short *h = (const unsigned short *)p + e0;
            uint32_t w[4];
#pragma unroll
            for (int k = 0; k < 4; k++) w[k] = (uint32_t)__ldg(h + 2 * k) | ((uint32_t)__ldg(h + 2 * k + 1) << 16);
            r[j] = make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
}

struct UnitStat {
    float m, c, S;
};

// Any unit, element by element: masked logits, |q| > 1, a row's ragged end.
template <int DT, bool CAP>
__device__ __forceinline__ UnitStat unit_general(const char *p, int n, int lane, const BeamArgs &a)
{
    const float NEG_INF = -__uint_as_float(0x7f800000u);
    float mx = NEG_INF;
#pragma unroll 4
    for (int i = lane; i < n; i += 32) mx = fmaxf(mx, beam_raw(DtypeTraits<DT>::load1(p, i)));
    UnitStat u{warp_max_redux(mx), 0.0f, 0.0f};
    if (u.m == NEG_INF) return u;
    u.c = beam_soft<CAP>(u.m, a);
    float s = 0.0f;
#pragma unroll 4
    for (int i = lane; i < n; i += 32) {
        const float v = beam_raw(DtypeTraits<DT>::load1(p, i));
        const float e = ex2_approx((beam_soft<CAP>(v, a) - u.c) * a.k);
        s += v == NEG_INF ? 0.0f : e;
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(FULLMASK, s, d);
    u.S = s;
    return u;
}

// A whole unit from registers; false when an element needs unit_general.
template <int DT, bool CAP>
__device__ __forceinline__ bool unit_fast(const uint4 (&r)[BNV], const BeamArgs &a, UnitStat &u)
{
    using T = DtypeTraits<DT>;
    float mx, mn;
    if constexpr (DT == G4S_BF16) {
        uint32_t x = r[0].x, y = x;
#pragma unroll
        for (int j = 0; j < BNV; j++) {
            x = bmax2_nan(x, bmax2_nan(bmax2_nan(r[j].x, r[j].y), bmax2_nan(r[j].z, r[j].w)));
            y = bmin2_nan(y, bmin2_nan(bmin2_nan(r[j].x, r[j].y), bmin2_nan(r[j].z, r[j].w)));
        }
        mx = fmax_nan(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u));
        mn = fmin_nan(__uint_as_float(y << 16), __uint_as_float(y & 0xffff0000u));
    } else {
        mx = mn = __uint_as_float(r[0].x);
#pragma unroll
        for (int j = 0; j < BNV; j++) {
            mx = fmax3_nan(fmax3_nan(mx, __uint_as_float(r[j].x), __uint_as_float(r[j].y)), __uint_as_float(r[j].z),
                           __uint_as_float(r[j].w));
            mn = fmin3_nan(fmin3_nan(mn, __uint_as_float(r[j].x), __uint_as_float(r[j].y)), __uint_as_float(r[j].z),
                           __uint_as_float(r[j].w));
        }
    }
    const float lim = CAP ? fminf(a.softcap, 1e30f) : 3.402823466e38f;
    const bool ok = mx <= lim && mn > (CAP ? -lim : -1e30f);  // a NaN fails both
    if (!__all_sync(FULLMASK, ok)) return false;
    u.m = warp_max_redux(mx);
    u.c = beam_soft<CAP>(u.m, a);
    const float2 ic = make_float2(a.invcap, a.invcap);
    const float2 cap2 = make_float2(a.softcap, a.softcap);
    const float2 nc = make_float2(-u.c, -u.c), k2 = make_float2(a.k, a.k);
    float2 acc0 = make_float2(0.0f, 0.0f), acc1 = acc0;
#pragma unroll
    for (int j = 0; j < BNV; j++) {
        float x[T::VW];
        T::unpack(r[j], x);
#pragma unroll
        for (int k = 0; k < T::VW; k += 2) {
            const float2 v = make_float2(x[k], x[k + 1]);
            float2 d;
            if constexpr (CAP) d = __ffma2_rn(tanh_poly2(__fmul2_rn(v, ic)), cap2, nc);
            else d = __fadd2_rn(v, nc);
            const float2 y = __fmul2_rn(d, k2);
            const float2 e = make_float2(ex2_approx(y.x), ex2_approx(y.y));
            if ((k >> 1) & 1) acc1 = __fadd2_rn(acc1, e);
            else acc0 = __fadd2_rn(acc0, e);
        }
    }
    acc0 = __fadd2_rn(acc0, acc1);
    float s = acc0.x + acc0.y;
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(FULLMASK, s, d);
    u.S = s;
    return true;
}

// A beam that continues: a finite or infinite score (not -inf, not NaN) and not ended.
__device__ __forceinline__ bool beam_live(const BeamArgs &a, int row)
{
    return a.scores[row] > -__uint_as_float(0x7f800000u) && !(a.done && a.done[row]);
}

// Persistent warps over the live rows' items; a unit's vectors are loaded while the
// one before is reduced.
template <int DT, bool VEC, bool CAP>
__global__ void __launch_bounds__(BS_THREADS) beam_stream_kernel(const BeamArgs a)
{
    using T = DtypeTraits<DT>;
    constexpr int UNIT = BeamGeo<DT>::UNIT;
    const float NEG_INF = -__uint_as_float(0x7f800000u);
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int lane = threadIdx.x & 31;
    const int nw = (int)gridDim.x * (BS_THREADS / 32);
    const int it0 = (int)blockIdx.x * (BS_THREADS / 32) + (threadIdx.x >> 5);
    const int step_row = nw / a.ipr, step_sub = nw % a.ipr;
    struct Cursor {
        int row, item, u;  // u: unit within the item
    };
    const int upr = (a.vocab + UNIT - 1) / UNIT;
    auto skip_dead = [&](Cursor &c) {
        while (c.row < a.rows && !beam_live(a, c.row)) {
            c.item += step_sub;
            c.row += step_row;
            if (c.item >= a.ipr) {
                c.item -= a.ipr;
                c.row++;
            }
        }
    };
    auto next = [&](Cursor c) {
        if (c.u + 1 < a.upi && c.item * a.upi + c.u + 1 < upr) {
            c.u++;
            return c;
        }
        c.u = 0;
        c.item += step_sub;
        c.row += step_row;
        if (c.item >= a.ipr) {
            c.item -= a.ipr;
            c.row++;
        }
        skip_dead(c);
        return c;
    };
    auto at = [&](const Cursor &c) {
        return (const char *)a.logits +
               ((int64_t)c.row * a.row_stride + (int64_t)(c.item * a.upi + c.u) * UNIT) * T::ESIZE;
    };
    auto left = [&](const Cursor &c) { return a.vocab - (c.item * a.upi + c.u) * UNIT; };
    Cursor cur{it0 / a.ipr, it0 % a.ipr, 0};
    skip_dead(cur);
    uint4 r[BNV] = {};
    if (cur.row < a.rows && left(cur) >= UNIT) load_unit<DT, VEC>(at(cur), lane, r);
    UnitStat acc{NEG_INF, 0.0f, 0.0f};
    while (cur.row < a.rows) {
        const Cursor nx = next(cur);
        uint4 rn[BNV] = {};
        if (nx.row < a.rows && left(nx) >= UNIT) load_unit<DT, VEC>(at(nx), lane, rn);
        UnitStat u;
        const int n = min(UNIT, left(cur));
        if (n < UNIT || !unit_fast<DT, CAP>(r, a, u)) u = unit_general<DT, CAP>(at(cur), n, lane, a);
        if (cur.u == 0) {
            acc = u;
        } else if (u.m > NEG_INF) {
            if (u.m > acc.m) {
                u.S += acc.m > NEG_INF ? acc.S * ex2_approx((acc.c - u.c) * a.k) : 0.0f;
                acc = u;
            } else {
                acc.S += u.S * ex2_approx((u.c - acc.c) * a.k);
            }
        }
        if (nx.u == 0 && lane == 0)
            a.istat[(int64_t)cur.row * a.ipr + cur.item] = make_float4(acc.m, acc.c, acc.S, 0.0f);
        cur = nx;
#pragma unroll
        for (int j = 0; j < BNV; j++) r[j] = rn[j];
    }
}

// ---------------------------------------------------------------------------
// combine
// ---------------------------------------------------------------------------
struct BeamRow {
    double ln, inv;  // log of the row's sum (in units of c), 1 / max(length, 1)^alpha
    float score, c;
    int len, kind;   // kind: BEAM_DEAD, BEAM_LIVE, BEAM_DONE
};
enum { BEAM_DEAD = 0, BEAM_LIVE = 1, BEAM_DONE = 2 };

__device__ __forceinline__ double beam_score(const BeamArgs &a, const BeamRow &r, uint32_t key)
{
    if (r.kind == BEAM_DONE) return (double)r.score;
    double s = (double)key2f(key);
    if (a.softcap > 0.0f) s = (double)a.softcap * tanh(s / (double)a.softcap);
    return (double)r.score + ((s - (double)r.c) / a.temperature - r.ln);
}

// Order of two continuations: rank, then the lower beam, the larger raw logit, the lower
// id (item): the latter three in one number, larger first.
__device__ __forceinline__ uint64_t beam_tie(int w, uint32_t key, uint32_t id)
{
    return ((uint64_t)(255 - w) << 56) | ((uint64_t)key << 24) | (0xffffffu - id);
}
__device__ __forceinline__ int tie_beam(uint64_t t) { return 255 - (int)(t >> 56); }
__device__ __forceinline__ uint32_t tie_key(uint64_t t) { return (uint32_t)(t >> 24); }
__device__ __forceinline__ uint32_t tie_id(uint64_t t) { return 0xffffffu - (uint32_t)(t & 0xffffffu); }

// Sorts P (a power of two) pairs in shared memory, first in order first.
__device__ __forceinline__ void beam_sort(double *rank, uint64_t *tie, int P)
{
    for (int k = 2; k <= P; k <<= 1) {
        for (int j = k >> 1; j > 0; j >>= 1) {
            for (int t = threadIdx.x; t < P / 2; t += BC_THREADS) {
                const int i = 2 * t - (t & (j - 1)), o = i + j;
                const double ri = rank[i], ro = rank[o];
                const uint64_t ti = tie[i], to = tie[o];
                const bool o_first = ro > ri || (ro == ri && to > ti);
                if (o_first == ((i & k) == 0)) {
                    rank[i] = ro;
                    rank[o] = ri;
                    tie[i] = to;
                    tie[o] = ti;
                }
            }
            __syncthreads();
        }
    }
}

// The keys of unit u of an item (0: masked or past the row).
template <int DT, bool VEC>
__device__ __forceinline__ void unit_keys(const char *p, int n, int lane, uint32_t (&key)[BeamGeo<DT>::EPL])
{
    using T = DtypeTraits<DT>;
    if (n >= BeamGeo<DT>::UNIT) {
        uint4 r[BNV];
        load_unit<DT, VEC>(p, lane, r);
#pragma unroll
        for (int j = 0; j < BNV; j++) {
            float x[T::VW];
            T::unpack(r[j], x);
#pragma unroll
            for (int k = 0; k < T::VW; k++) key[j * T::VW + k] = beam_key(x[k]);
        }
    } else {
#pragma unroll
        for (int j = 0; j < BNV; j++)
#pragma unroll
            for (int k = 0; k < T::VW; k++) {
                const int e = (j * 32 + lane) * T::VW + k;
                key[j * T::VW + k] = e < n ? beam_key(T::load1(p, e)) : 0u;
            }
    }
}

template <int DT, bool VEC>
__global__ void __launch_bounds__(BC_THREADS) beam_combine_kernel(const BeamArgs a)
{
    using T = DtypeTraits<DT>;
    constexpr int UNIT = BeamGeo<DT>::UNIT, EPL = BeamGeo<DT>::EPL;
    const double NEG_INF = -__longlong_as_double(0x7ff0000000000000ll);
    extern __shared__ double s_mem[];
    double *e_rank = s_mem;                              // [pe] the beams' items
    uint64_t *e_tie = (uint64_t *)(e_rank + a.pe);
    double *c_rank = (double *)(e_tie + a.pe);           // [pc] collected tokens
    uint64_t *c_tie = (uint64_t *)(c_rank + a.pc);
    __shared__ BeamRow s_row[G4S_BEAM_MAX];
    __shared__ int s_cnt[G4S_BEAM_MAX], s_sel[G4S_BEAM_MAX];
    __shared__ unsigned long long s_thr[G4S_BEAM_MAX];
    __shared__ int s_m;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int W = a.beams, N = a.n_out, row0 = (int)blockIdx.x * W;

    for (int e = tid; e < a.pe; e += BC_THREADS) {
        e_rank[e] = NEG_INF;
        e_tie[e] = 0;
    }
    for (int e = tid; e < a.pc; e += BC_THREADS) {
        c_rank[e] = NEG_INF;
        c_tie[e] = 0;
    }
    if (tid < G4S_BEAM_MAX) {
        s_thr[tid] = 0;
        s_sel[tid] = 0;
        s_cnt[tid] = 0;
    }
    if (tid == 0) s_m = 0;
    __syncthreads();
    asm volatile("griddepcontrol.wait;" ::: "memory");

    // 1. a warp a beam: the row's sum, its n_out largest items
    for (int w = warp; w < W; w += BC_WARPS) {
        const int row = row0 + w;
        BeamRow r;
        r.score = a.scores[row];
        r.len = a.lens ? a.lens[row] : 0;
        r.kind = !(r.score > -__uint_as_float(0x7f800000u)) ? BEAM_DEAD : (a.done && a.done[row]) ? BEAM_DONE : BEAM_LIVE;
        r.c = 0.0f;
        r.ln = 0.0;
        const int length = r.kind == BEAM_LIVE ? r.len + 1 : r.len;
        r.inv = a.alpha == 0.0 ? 1.0 : pow((double)max(length, 1), -a.alpha);
        int cnt = 0;
        if (r.kind == BEAM_DONE) {
            cnt = 1;
            if (lane == 0) e_tie[w * N] = beam_tie(w, 0u, 0u);
        } else if (r.kind == BEAM_LIVE) {
            const float4 *st = a.istat + (int64_t)row * a.ipr;
            uint32_t key[BIPL];
            float c = -__uint_as_float(0x7f800000u);
            uint32_t kmax = 0;
            int nv = 0;
#pragma unroll
            for (int j = 0; j < BIPL; j++) {
                const int i = j * 32 + lane;
                key[j] = 0;
                if (i < a.ipr) {
                    const float4 q = __ldcg(st + i);
                    key[j] = beam_key(q.x);
                    if (key[j]) c = fmaxf(c, q.y);
                }
                kmax = max(kmax, key[j]);
                nv += key[j] != 0;
            }
            const uint32_t kmin = __reduce_min_sync(FULLMASK, kmax);  // every lane holds an item at or above it
            kmax = __reduce_max_sync(FULLMASK, kmax);
            nv = __reduce_add_sync(FULLMASK, nv);
            if (nv == 0) {
                r.kind = BEAM_DEAD;
            } else {
                c = warp_max_redux(c);
                double sum = 0.0;
#pragma unroll
                for (int j = 0; j < BIPL; j++) {
                    if (key[j]) {
                        const float4 q = __ldcg(st + j * 32 + lane);
                        // 2^((c_i - c) k): whole and fractional part, the difference exact in 64 bits
                        const double y = ((double)q.y - (double)c) * a.k64;
                        const double whole = rint(fmax(y, -1000.0));
                        sum += (double)q.z * (double)ex2_approx((float)(y - whole < -1.0 ? -1.0 : y - whole)) *
                               __longlong_as_double((long long)(1023 + (int)whole) << 52);
                    }
                }
#pragma unroll
                for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(FULLMASK, sum, d);
                r.c = c;
                r.ln = log(sum);
                // the largest thr with at least N items at or above it
                cnt = min(N, nv);
                uint32_t thr = 0;  // keys above thr are taken, then those equal to it
                int eq = 0;
                if (nv > N) {
                    uint32_t lo = N <= 32 ? kmin : 0u, hi = kmax;  // count(>= lo) >= N
                    if (lo == 0) lo = 1;
                    bool exact = false;
                    while (lo < hi) {
                        const uint32_t mid = lo + (hi - lo + 1) / 2;
                        int n = 0;
#pragma unroll
                        for (int j = 0; j < BIPL; j++) n += key[j] >= mid;
                        n = __reduce_add_sync(FULLMASK, n);
                        if (n == N) {
                            thr = mid - 1;
                            exact = true;
                            break;
                        }
                        if (n > N) lo = mid;
                        else hi = mid - 1;
                    }
                    if (!exact) {
                        thr = lo;
                        eq = 1;
                    }
                }
                int base = w * N;
#pragma unroll
                for (int j = 0; j < BIPL; j++) {
                    const bool take = key[j] > thr;
                    const unsigned b = __ballot_sync(FULLMASK, take);
                    if (take) e_tie[base + __popc(b & ((1u << lane) - 1))] = beam_tie(w, key[j], (uint32_t)(j * 32 + lane));
                    base += __popc(b);
                }
                if (eq) {
#pragma unroll
                    for (int j = 0; j < BIPL; j++) {
                        const bool take = key[j] == thr;
                        const unsigned b = __ballot_sync(FULLMASK, take);
                        const int o = base + __popc(b & ((1u << lane) - 1));
                        if (take && o < w * N + cnt) e_tie[o] = beam_tie(w, key[j], (uint32_t)(j * 32 + lane));
                        base += __popc(b);
                    }
                }
            }
        }
        if (lane == 0) {
            s_row[w] = r;
            s_cnt[w] = cnt;
        }
    }
    __syncthreads();

    // 2. the items by their best token
    for (int e = tid; e < W * N; e += BC_THREADS) {
        const uint64_t t = e_tie[e];
        if (t) {
            const BeamRow &r = s_row[tie_beam(t)];
            e_rank[e] = beam_score(a, r, tie_key(t)) * r.inv;
        }
    }
    __syncthreads();
    beam_sort(e_rank, e_tie, a.pe);
    int total = 0;
    for (int w = 0; w < W; w++) total += s_cnt[w];
    const int nsel = min(N, total);
    // a beam's tokens count from its best item left out; where all of its N items are
    // in, from the last of them; where it has no more, all
    for (int e = tid; e < total; e += BC_THREADS) {
        const int w = tie_beam(e_tie[e]);
        if (e < nsel) atomicAdd(&s_sel[w], 1);
        else atomicMax(&s_thr[w], (unsigned long long)e_tie[e]);
    }
    __syncthreads();
    if (tid == 0 && nsel == N && s_sel[tie_beam(e_tie[N - 1])] == N) s_thr[tie_beam(e_tie[N - 1])] = e_tie[N - 1] - 1;
    __syncthreads();

    // 3. their tokens
    for (int j = warp; j < nsel; j += BC_WARPS) {
        const uint64_t t = e_tie[j];
        const int w = tie_beam(t), quota = N - j;
        if (s_row[w].kind == BEAM_DONE) {
            if (lane == 0) c_tie[atomicAdd(&s_m, 1)] = t;
            continue;
        }
        const uint32_t item = tie_id(t);
        const uint64_t thr = s_thr[w];
        const int64_t e0 = (int64_t)item * a.upi * UNIT;
        const int n = (int)min((int64_t)a.upi * UNIT, a.vocab - e0);
        const char *p = (const char *)a.logits + ((int64_t)(row0 + w) * a.row_stride + e0) * T::ESIZE;
        uint32_t first[EPL];  // the first unit's keys; 0: not wanted
        auto want = [&](uint32_t key) { return key && beam_tie(w, key, item) > thr; };
        auto load = [&](int u, uint32_t(&key)[EPL]) {
            unit_keys<DT, VEC>(p + (int64_t)u * UNIT * T::ESIZE, n - u * UNIT, lane, key);
#pragma unroll
            for (int i = 0; i < EPL; i++)
                if (!want(key[i])) key[i] = 0;
        };
        // each unit's keys and the position of the lane's first logit in the item
        auto for_units = [&](auto &&f) {
            f(first, 0);
            for (int u = 1; u * UNIT < n; u++) {
                uint32_t key[EPL];
                load(u, key);
                f(key, u * UNIT);
            }
        };
        load(0, first);
        auto pos = [&](int i) { return ((i / T::VW) * 32 + lane) * T::VW + i % T::VW; };
        auto count = [&](uint32_t least) {  // wanted keys at or above `least`
            int c = 0;
            for_units([&](const uint32_t(&key)[EPL], int) {
#pragma unroll
                for (int i = 0; i < EPL; i++) c += key[i] >= least;
            });
            return (int)__reduce_add_sync(FULLMASK, c);
        };
        auto push = [&](uint32_t above, uint32_t equal, int last) {  // keys > above; == equal up to position `last`
            for_units([&](const uint32_t(&key)[EPL], int at) {
#pragma unroll
                for (int i = 0; i < EPL; i++)
                    if (key[i] > above || (equal && key[i] == equal && at + pos(i) <= last))
                        c_tie[atomicAdd(&s_m, 1)] = beam_tie(w, key[i], (uint32_t)(e0 + at + pos(i)));
            });
        };
        if (count(1u) <= quota) {
            push(0u, 0u, 0);
        } else {
            // only quota of them can count (the j items before hold a better token each): the
            // quota-th largest key, then the position up to which its equals are taken
            uint32_t lo = 1u, hi = 0xffffffffu;
            while (lo < hi) {
                const uint32_t mid = lo + (hi - lo) / 2 + 1;
                if (count(mid) >= quota) lo = mid;
                else hi = mid - 1;
            }
            const int need = quota - (lo == 0xffffffffu ? 0 : count(lo + 1));
            int p0 = 0, p1 = n - 1;
            while (p0 < p1) {
                const int mid = (p0 + p1) / 2;
                int c = 0;
                for_units([&](const uint32_t(&key)[EPL], int at) {
#pragma unroll
                    for (int i = 0; i < EPL; i++) c += key[i] == lo && at + pos(i) <= mid;
                });
                if ((int)__reduce_add_sync(FULLMASK, c) >= need) p1 = mid;
                else p0 = mid + 1;
            }
            push(lo, lo, p0);
        }
    }
    __syncthreads();
    const int m = s_m;
    for (int e = tid; e < m; e += BC_THREADS) {
        const BeamRow &r = s_row[tie_beam(c_tie[e])];
        c_rank[e] = beam_score(a, r, tie_key(c_tie[e])) * r.inv;
    }
    __syncthreads();
    beam_sort(c_rank, c_tie, next_pow2(max(m, 2)));
    if (tid < N) {
        const int64_t o = (int64_t)blockIdx.x * N + tid;
        float score = -__uint_as_float(0x7f800000u);
        int parent = -1, token = -1, len = 0, done = 0;
        if (tid < m) {
            const uint64_t t = c_tie[tid];
            const int w = tie_beam(t);
            const BeamRow &r = s_row[w];
            score = (float)(a.alpha == 0.0 ? c_rank[tid] : beam_score(a, r, tie_key(t)));
            parent = row0 + w;
            if (r.kind == BEAM_DONE) {
                token = a.pad_token;
                len = r.len;
                done = 1;
            } else {
                token = (int)tie_id(t);
                len = r.len + 1;
                for (int i = 0; i < a.n_eos; i++) done |= token == a.eos[i];
            }
        }
        a.out_scores[o] = score;
        a.out_parents[o] = parent;
        a.out_tokens[o] = token;
        if (a.out_lens) a.out_lens[o] = len;
        if (a.out_done) a.out_done[o] = (uint8_t)done;
    }
}

template <int DT, bool VEC, bool CAP>
static cudaError_t launch_beam_t(const BeamArgs &a, int sms, cudaStream_t s)
{
    static int bps[MAX_DEVICES] = {};
    static bool ready[MAX_DEVICES] = {};
    const int dev = current_device();
    if (dev < 0 || dev >= MAX_DEVICES) return cudaErrorInvalidDevice;
    cudaError_t e;
    if (!ready[dev]) {
        e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&bps[dev], beam_stream_kernel<DT, VEC, CAP>, BS_THREADS, 0);
        if (e != cudaSuccess) return e;
        e = cudaFuncSetAttribute(beam_combine_kernel<DT, VEC>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 BEAM_COMBINE_SMEM_MAX);
        if (e != cudaSuccess) return e;
        ready[dev] = true;
    }
    const int64_t items = (int64_t)a.rows * a.ipr, per = BS_THREADS / 32;
    const int64_t blocks = (items + per - 1) / per, most = (int64_t)bps[dev] * sms;
    beam_stream_kernel<DT, VEC, CAP><<<(unsigned)(blocks < most ? blocks : most), BS_THREADS, 0, s>>>(a);
    e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(a.rows / a.beams));
    cfg.blockDim = dim3(BC_THREADS);
    cfg.dynamicSmemBytes = (size_t)(a.pe + a.pc) * 16;
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, beam_combine_kernel<DT, VEC>, a);
}

template <int DT>
static cudaError_t launch_beam_dt(const BeamArgs &a, bool vec, int sms, cudaStream_t s)
{
    if (a.softcap > 0.0f) return vec ? launch_beam_t<DT, true, true>(a, sms, s) : launch_beam_t<DT, false, true>(a, sms, s);
    return vec ? launch_beam_t<DT, true, false>(a, sms, s) : launch_beam_t<DT, false, false>(a, sms, s);
}

cudaError_t launch_beam_select(const BeamArgs &a, int dtype, bool vec, int sms, cudaStream_t s)
{
    return dtype == G4S_F32 ? launch_beam_dt<G4S_F32>(a, vec, sms, s) : launch_beam_dt<G4S_BF16>(a, vec, sms, s);
}

// ---------------------------------------------------------------------------
// reordering of dense states
// ---------------------------------------------------------------------------
// A thread moves one column (sizeof(V) bytes at one place of a segment) of all of a
// group's rows: every row that is wanted is read before any is written, so that source
// and destination may be the same memory without a copy or a barrier, and a parent of
// several rows is read once.
template <class V, int WMAX>
__device__ __forceinline__ void reorder_column(const ReorderTensor &t, int row0, uint32_t c, const uint32_t *child)
{
    const uint32_t seg = c / t.seg_cols, col = c % t.seg_cols;
    const int64_t off = (int64_t)(seg / t.segs1) * t.stride0 + (int64_t)(seg % t.segs1) * t.stride1 +
                        (int64_t)col * (int64_t)sizeof(V) + (int64_t)row0 * t.row_stride;
    const char *src = t.src + off;
    char *dst = t.dst + off;
    V v[WMAX];
#pragma unroll
    for (int p = 0; p < WMAX; p++)
        if (child[p]) v[p] = *(const V *)(src + p * t.row_stride);
#pragma unroll
    for (int p = 0; p < WMAX; p++)
        for (uint32_t m = child[p]; m; m &= m - 1) *(V *)(dst + (__ffs(m) - 1) * t.row_stride) = v[p];
}

template <int WMAX>
__global__ void __launch_bounds__(REORDER_THREADS) beam_reorder_kernel(const ReorderArgs a)
{
    __shared__ uint32_t s_child[WMAX];  // rows of the group that take row p's state
    const int W = a.beams;
    int i = 0;
    while (i + 1 < a.n && (int64_t)blockIdx.x >= a.first[i + 1]) i++;
    const ReorderTensor &t = a.t[i];
    const int64_t b = (int64_t)blockIdx.x - a.first[i];
    const int row0 = (int)(b / t.blocks) * W;
    if (threadIdx.x < WMAX) {
        uint32_t m = 0;
        for (int j = 0; j < W; j++) {
            const int p = a.parents[row0 + j] - row0;
            if (p == (int)threadIdx.x && !(t.src == t.dst && p == j)) m |= 1u << j;
        }
        s_child[threadIdx.x] = (int)threadIdx.x < W ? m : 0u;
    }
    __syncthreads();
    const uint32_t c = (uint32_t)(b % t.blocks) * REORDER_THREADS + threadIdx.x;
    if (c >= t.cols) return;
    if (t.width == 16) reorder_column<uint4, WMAX>(t, row0, c, s_child);
    else if (t.width == 4) reorder_column<uint32_t, WMAX>(t, row0, c, s_child);
    else reorder_column<uint8_t, WMAX>(t, row0, c, s_child);
}

cudaError_t launch_beam_reorder(const ReorderArgs &a, int64_t blocks, cudaStream_t s)
{
    const unsigned g = (unsigned)blocks;
    if (a.beams <= 4) beam_reorder_kernel<4><<<g, REORDER_THREADS, 0, s>>>(a);
    else if (a.beams <= 8) beam_reorder_kernel<8><<<g, REORDER_THREADS, 0, s>>>(a);
    else if (a.beams <= 16) beam_reorder_kernel<16><<<g, REORDER_THREADS, 0, s>>>(a);
    else beam_reorder_kernel<32><<<g, REORDER_THREADS, 0, s>>>(a);
    return cudaGetLastError();
}

}  // namespace g4s
