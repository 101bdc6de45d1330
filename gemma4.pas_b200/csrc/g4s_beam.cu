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
// a beam's tokens; the beams' scores meet in pairs of fp32 numbers, for the
// few tokens that can be among the best.
//
// beam_stream_kernel: one pass over the logits.  A row has up to 128 items of one length
//   (a whole number of 4 KiB loads, or for short rows 1/2 to 1/8 of one); an item is
//   reduced to (m, ref, S): the largest raw logit, a reference in powers of two (ref =
//   s(m) k with the softcap, else m), and S = sum 2^(s_i k - ref) (2^((l_i - ref) k)),
//   k = log2(e) / T.  Items of one load share ref and S, which stands with the largest m.
//   ref is a rounded number: what it is off by is in every term alike, and the combine
//   takes it out again, so that a score is base + x(l) - x(row's largest) with both x exact.
// beam_combine_kernel: one CTA a prompt.
//   1. a warp a beam: the row's sum from its items (as pairs), and its n_out items with the
//      largest (m, then lowest item);
//   2. those items' best tokens ranked over the beams: the n_out best tokens
//      lie in the n_out items that rank first (each item that ranks before
//      another holds a token that beats all of the other's);
//   3. these items reread, their tokens above the beam's best item left out
//      collected (at most n_out - j from the item in place j), ranked, sorted.
//
// Measured (one B200, copy bandwidth 6570 GB/s), the whole selection: 256 bf16 rows of
// 262144 logits, 8 beams, 16 continuations 42 us (3.2 TB/s; the streaming pass 32, without
// its sums 23); 205 live fp32 rows 45 us (4.8 TB/s; 37, 35); 4 fp32 rows 9.3 us (5.0); 30
// live fp32 rows of 32003 logits 10.0 us (4.2).  The streaming pass is bound by
// instructions for bf16 rows (issue slots 57 %, the exponentials' unit 51 %, fp32 pipe
// 48 % busy at 21 warps an SM) and by memory for fp32; the combine, 4 us for 4 beams and
// 10 for 8 beams and 16 continuations, by the latency of dependent steps: its one CTA a
// prompt leaves most of the GPU idle, and waits for barriers and instruction fetches.
#include "g4s_device.cuh"
#include "g4s_kernels.cuh"

namespace g4s {

constexpr int BS_THREADS = 32;   // CTA of the streaming pass: a warp, which shares nothing with another
constexpr int BS_CTAS = 24;      // of them on an SM: 80 registers a thread (the bf16 variants of
                                 // unaligned rows spill 8 to 40 bytes, the aligned softcap one 4), 8 KiB a CTA
constexpr int BS_STAGES = 2;     // loads a warp's ring in shared memory holds
constexpr int BS_NV = 8;         // 16-byte vectors a lane and load (4 KiB, two units)
constexpr int LINE = 128;        // loads of unaligned rows are copied from the line's start
constexpr int BC_THREADS = 1024; // CTA of the combine
constexpr int BC_WARPS = BC_THREADS / 32;
constexpr int BEAM_PART_ITEMS = 64;
constexpr int BIPL = BEAM_MAX_ITEMS / 32;  // a row's items a lane of its warp
constexpr int BNV = 4;           // 16-byte vectors a lane and unit (2 KiB a unit)

template <int DT>
struct BeamGeo {
    static constexpr int VW = DtypeTraits<DT>::VW;
    static constexpr int EPL = BNV * VW;    // a lane's logits of a unit
    static constexpr int UNIT = 32 * EPL;   // 512 fp32 or 1024 bf16 logits
};

// A masked logit (NaN, or at or below -1e30 as on the top-K path) is -inf; +inf counts
// as the type's largest finite number, so that differences stay defined; -0 is +0.
template <int DT>
__device__ __forceinline__ float beam_max()
{
    return __uint_as_float(DT == G4S_BF16 ? 0x7f7f0000u : 0x7f7fffffu);
}
template <int DT>
__device__ __forceinline__ float beam_raw(float v)
{
    return v > -1e30f ? fminf(v, beam_max<DT>()) + 0.0f : -__uint_as_float(0x7f800000u);
}
template <int DT>
__device__ __forceinline__ uint32_t beam_key(float v)
{
    return cand_key(beam_raw<DT>(v));
}

// cap * tanh(v / cap) in fp32: the polynomial up to |q| = 1, 1 - 2 / (e^2q + 1) beyond
// (2 / (e^2q + 1) < 0.24 there, so the approximate exponential and quotient cost less
// than half an ulp of the result).
__device__ __forceinline__ float beam_soft(float v, const BeamArgs &a)
{
    const float q = __fmul_rn(v, a.invcap), aq = fabsf(q);
    const float w = 1.0f - __fdividef(2.0f, ex2_approx(aq * (2.0f * G4_L2E)) + 1.0f);
    return __fmul_rn(aq <= 1.0f ? tanh_poly(q) : copysignf(w, q), a.softcap);
}

// The softcap's kinds.  CAP_FOLD, cap / T up to BEAM_FOLD: s(l) k to a few fp32 steps, so that a
// term is off by up to 4 * 2^-24 cap / T of itself.  CAP_FAR, beyond: what a term is off by goes
// with its distance from the maximum and not with the size of the numbers.
enum { CAP_NONE = 0, CAP_FOLD = 1, CAP_FAR = 2 };

// s(m) k - minus by the very operations that a term takes: with it for a reference and for
// what the maximum's own term is off by, an error common to the terms falls out.
template <int CAP>
__device__ __forceinline__ float beam_value(const BeamArgs &a, float m, float minus)
{
    const float q = __fmul_rn(m, m);
    if constexpr (CAP == CAP_FAR) {
        float p = a.h1[BEAM_H1 - 1];
#pragma unroll
        for (int i = BEAM_H1 - 2; i > 0; i--) p = __fmaf_rn(p, q, a.h1[i]);
        return __fmaf_rn(__fmul_rn(m, q), p, __fmaf_rn(m, a.h1[0], -minus));
    }
    if (fabsf(m) <= a.lim1) {
        float p = a.h1[BEAM_H1 - 1];
#pragma unroll
        for (int i = BEAM_H1 - 2; i >= 0; i--) p = __fmaf_rn(p, q, a.h1[i]);
        return __fmaf_rn(m, p, -minus);
    }
    if (fabsf(m) <= a.lim2) {
        float p = a.h2[BEAM_H2 - 1];
#pragma unroll
        for (int i = BEAM_H2 - 2; i >= 0; i--) p = __fmaf_rn(p, q, a.h2[i]);
        return __fmaf_rn(m, p, -minus);
    }
    return __fmaf_rn(beam_soft(m, a), a.k, -minus);
}

// CAP_FAR: sums whose maximum the polynomial reaches stand against its value there, rounded
// (ref), the others against s(m) k itself; the former's own maximum is 2^this.
__device__ __forceinline__ float beam_off(const BeamArgs &a, float m, float ref)
{
    return fabsf(m) <= a.lim1 ? beam_value<CAP_FAR>(a, m, ref) : 0.0f;
}

// (s(m) - s(l)) k for m >= l to some 2^-21 of itself, whatever cap, T, m and l: with
// a = m / cap, b = l / cap
//   tanh a - tanh b = sinh(a - b) / (cosh a cosh b)
//                   = 2 F (1 - e^-2(a - b)) / ((1 + e^-2|a|) (1 + e^-2|b|)),
// F = e^-2 min(|a|, |b|) where a and b are on one side of 0, else 1.
__device__ __forceinline__ float beam_e2(const BeamArgs &a, float v)  // e^-2|v / cap|
{
    const float x = fminf(fabsf(v), a.sat), h = __fmul_rn(x, a.two2[0]);
    const float l = __fmaf_rn(x, a.two2[1], __fmaf_rn(x, a.two2[0], -h));
    const float e = ex2_approx(-h);
    return __fmaf_rn(e, -l * 0.693147182f, e);
}
__device__ __forceinline__ float beam_below(const BeamArgs &a, float m, float l)
{
    const float em = beam_e2(a, m), el = beam_e2(a, l), d = __fmul_rn(__fsub_rn(m, l), a.invcap);
    const float t = tanh_poly(fminf(d, 1.0f));
    float num = d <= 1.0f ? 2.0f * t : 1.0f - ex2_approx(d * (-2.0f * G4_L2E));
    float den = d <= 1.0f ? 1.0f + t : 1.0f;
    num *= l >= 0.0f ? el : m <= 0.0f ? em : 1.0f;
    den *= (1.0f + em) * (1.0f + el);
    return __fmul_rn(a.capk2, __fdividef(num, den));
}
// A logit below which (s(m) - s(l)) k is over 64 (set for 96; a term is under 2^-64 of the
// maximum's, all of a row's together under 2^-41 of its sum): tanh a - tanh b = 192 / (2 cap k).
__device__ __forceinline__ float beam_nothing(const BeamArgs &a, float m)
{
    const float em = beam_e2(a, m), u = (m >= 0.0f ? 2.0f * em : 2.0f) / (1.0f + em) + 192.0f / a.capk2;
    float lg;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(lg) : "f"((2.0f - u) / u));
    return u < 2.0f ? 0.346573591f * a.softcap * lg : -__uint_as_float(0x7f800000u);
}

// Two fp32 numbers in a 64-bit register: the packed operations' operands.  two() is volatile
// so that a constant stays in its register instead of being rebuilt at every use.
__device__ __forceinline__ uint64_t two(float x)
{
    uint64_t r;
    asm volatile("mov.b64 %0, {%1, %1};" : "=l"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ uint64_t two(float x, float y)
{
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
    return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c)
{
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b)
{
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b)
{
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ float2 halves(uint64_t v)
{
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}

// This lane's largest and smallest logit of a load; a NaN comes through.
template <int DT>
__device__ __forceinline__ float lane_max(const uint4 (&r)[BS_NV])
{
    if constexpr (DT == G4S_BF16) {
        uint32_t x = bmax2_nan(bmax2_nan(r[0].x, r[0].y), bmax2_nan(r[0].z, r[0].w));
#pragma unroll
        for (int j = 1; j < BS_NV; j++) x = bmax2_nan(x, bmax2_nan(bmax2_nan(r[j].x, r[j].y), bmax2_nan(r[j].z, r[j].w)));
        return fmax_nan(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u));
    } else {
        float m = __uint_as_float(r[0].x);
#pragma unroll
        for (int j = 0; j < BS_NV; j++)
            m = fmax3_nan(fmax3_nan(m, __uint_as_float(r[j].x), __uint_as_float(r[j].y)), __uint_as_float(r[j].z),
                          __uint_as_float(r[j].w));
        return m;
    }
}
template <int DT>
__device__ __forceinline__ float lane_min(const uint4 (&r)[BS_NV])
{
    if constexpr (DT == G4S_BF16) {
        uint32_t x = bmin2_nan(bmin2_nan(r[0].x, r[0].y), bmin2_nan(r[0].z, r[0].w));
#pragma unroll
        for (int j = 1; j < BS_NV; j++) x = bmin2_nan(x, bmin2_nan(bmin2_nan(r[j].x, r[j].y), bmin2_nan(r[j].z, r[j].w)));
        return fmin_nan(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u));
    } else {
        float m = __uint_as_float(r[0].x);
#pragma unroll
        for (int j = 0; j < BS_NV; j++)
            m = fmin3_nan(fmin3_nan(m, __uint_as_float(r[j].x), __uint_as_float(r[j].y)), __uint_as_float(r[j].z),
                          __uint_as_float(r[j].w));
        return m;
    }
}

// The same of the logits that are not masked (-inf and +inf for none).
template <int DT>
__device__ __forceinline__ void lane_extremes_open(const uint4 (&r)[BS_NV], float &mx, float &mn)
{
    using T = DtypeTraits<DT>;
    mx = -__uint_as_float(0x7f800000u);
    mn = -mx;
#pragma unroll
    for (int j = 0; j < BS_NV; j++) {
        float x[T::VW];
        T::unpack(r[j], x);
#pragma unroll
        for (int i = 0; i < T::VW; i++) {
            const bool open = x[i] > -1e30f;
            mx = open ? fmaxf(mx, x[i]) : mx;
            mn = open ? fminf(mn, x[i]) : mn;
        }
    }
}

// Adds 2^(s_i k - ref) (without softcap 2^((l_i - ref) k): the difference first, so that
// k's rounding acts on the distance only) of a load to the lane's sums.  With the softcap
// s k = l H(l^2), H a polynomial of NH coefficients with k and the cap folded in.  MASKED:
// some logits add nothing.  APART: the linear part against ref by itself, so that only the
// rest (under a thirteenth of s k below cap / 2) is rounded before its difference is taken.
template <int DT, int NH, bool MASKED, bool APART = false>
__device__ __forceinline__ void load_sum(const uint4 (&r)[BS_NV], const uint64_t *h, uint64_t k, float ref, uint64_t &s0, uint64_t &s1)
{
    using T = DtypeTraits<DT>;
    const uint64_t nref = two(-ref, -ref);
#pragma unroll
    for (int j = 0; j < BS_NV; j++) {
        float x[T::VW];
        T::unpack(r[j], x);
#pragma unroll
        for (int i = 0; i < T::VW; i += 2) {
            const uint64_t v = two(x[i], x[i + 1]);
            uint64_t y;
            if constexpr (NH > 0) {
                const uint64_t q = mul2(v, v);
                uint64_t p = h[NH - 1];
#pragma unroll
                for (int c = NH - 2; c >= (APART ? 1 : 0); c--) p = fma2(p, q, h[c]);
                y = APART ? fma2(mul2(v, q), p, fma2(v, h[0], nref)) : fma2(v, p, nref);
            } else {
                y = mul2(add2(v, nref), k);
            }
            const float2 z = halves(y);
            float e0 = ex2_approx(z.x), e1 = ex2_approx(z.y);
            if (MASKED) {
                e0 = x[i] > -1e30f ? e0 : 0.0f;
                e1 = x[i + 1] > -1e30f ? e1 : 0.0f;
            }
            const uint64_t e = two(e0, e1);
            if ((i >> 1) & 1) s1 = add2(s1, e);
            else s0 = add2(s0, e);
        }
    }
}

// Vector J of a load: its copy into the ring, its way out of it.
template <int J>
__device__ __forceinline__ void ring_copy(uint32_t to, const char *p)
{
    asm volatile("cp.async.cg.shared.global [%0+%2], [%1+%2], 16;" ::"r"(to), "l"(p), "n"(J * 512) : "memory");
    if constexpr (J + 1 < BS_NV) ring_copy<J + 1>(to, p);
}
template <int J>
__device__ __forceinline__ void ring_read(uint32_t from, uint4 (&r)[BS_NV])
{
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4+%5];"
                 : "=r"(r[J].x), "=r"(r[J].y), "=r"(r[J].z), "=r"(r[J].w)
                 : "r"(from), "n"(J * 512)
                 : "memory");
    if constexpr (J + 1 < BS_NV) ring_read<J + 1>(from, r);
}

// The same of a row that is not 16-byte aligned: its bytes stand `shift` into the ring, and
// word i of the lane is word i * 32 + lane of the load (two bf16 logits side by side; where
// they do not share an aligned word, cut from two).
template <int DT>
__device__ __forceinline__ void ring_read_shifted(uint32_t from, uint32_t shift, int lane, uint4 (&r)[BS_NV])
{
    const uint32_t a = from + (shift & ~3u) + lane * 4;
    uint32_t w[BS_NV * 4];
#pragma unroll
    for (int i = 0; i < BS_NV * 4; i++) asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w[i]) : "r"(a + i * 128) : "memory");
    if (DT == G4S_BF16 && (shift & 2)) {
#pragma unroll
        for (int i = 0; i < BS_NV * 4; i++) {
            uint32_t next;
            asm volatile("ld.shared.u32 %0, [%1];" : "=r"(next) : "r"(a + i * 128 + 4) : "memory");
            w[i] = __byte_perm(w[i], next, 0x5432);
        }
    }
#pragma unroll
    for (int j = 0; j < BS_NV; j++) r[j] = make_uint4(w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
}

// A load's logits from n on (behind the row's end) become -inf in the ring (in registers the
// cut costs spills): the lane's own vectors, or, of a load that stands `shift` into the
// ring, by the whole warp.
template <int DT>
__device__ __forceinline__ void ring_low(uint32_t at)  // one logit
{
    if constexpr (DT == G4S_BF16) asm volatile("st.shared.u16 [%0], %1;" ::"r"(at), "h"((unsigned short)0xff80) : "memory");
    else asm volatile("st.shared.u32 [%0], %1;" ::"r"(at), "r"(0xff800000u) : "memory");
}
template <int DT>
__device__ __forceinline__ void ring_low16(uint32_t at)
{
    asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(at), "r"(DT == G4S_BF16 ? 0xff80ff80u : 0xff800000u) : "memory");
}
template <int DT>
__device__ __forceinline__ void ring_cut(uint32_t at, int lane, int n)
{
    using T = DtypeTraits<DT>;
#pragma unroll 1
    for (int left = n - lane * T::VW, j = 0; j < BS_NV; j++, left -= 32 * T::VW, at += 512) {
        if (left <= 0) ring_low16<DT>(at);
        else
            for (int i = left; i < T::VW; i++) ring_low<DT>(at + i * T::ESIZE);
    }
}
template <int DT>
__device__ __forceinline__ void ring_cut_shifted(uint32_t from, uint32_t shift, int lane, int n)
{
    using T = DtypeTraits<DT>;
    const uint32_t end = shift + n * T::ESIZE, up = (end + 15) & ~15u;
    if (lane < (int)(up - end) / T::ESIZE) ring_low<DT>(from + end + lane * T::ESIZE);
#pragma unroll 1
    for (uint32_t b = up + lane * 16; b < BS_NV * 512 + LINE; b += 512) ring_low16<DT>(from + b);
}

// A beam that continues: a score that is not -inf (nor NaN), and not ended.
__device__ __forceinline__ bool beam_live(const BeamArgs &a, int row)
{
    const float score = a.scores[row];  // (both loads under way at once)
    const uint8_t done = a.done ? a.done[row] : 0;
    return score > -__uint_as_float(0x7f800000u) && !done;
}

// Long-lived warps over the live rows' items; each lane copies its own vectors of the two
// loads ahead into the warp's ring (cp.async: no registers, no barrier).  Rows that are not
// 16-byte aligned are copied by the lines that hold them (bytes before the row's first
// logit in the same line, behind its last in the same 16 bytes) and read from the ring at
// their offset, so that a row's sums are grouped alike wherever it starts: equal beams
// score equal.  (256 rows of 262143 logits: bf16 46 us, aligned 42; fp32 56 for 54, or 5 more
// where the copies start at 16 bytes.)  A row's ragged end is filled with masked
// logits in the ring: element by element it took the whole kernel 2 to 10 us longer.  The
// ways through a load:
//   0  no logit above cap / 2: the polynomial of 5 coefficients (7 packed operations a
//      pair).  Below -cap / 2 it falls faster than tanh, to -inf for masked logits (its
//      last coefficient is positive); with the load's maximum at or above 0 and cap >=
//      28 T what is lost there is under 1e-7 of the load's sum (2047 other logits where
//      it is worst, at -0.92 cap), so the smallest logit is not looked for; else it has
//      to be at or above -cap / 2
//   1  |l| <= cap: the polynomial of 8 coefficients
//   2  the same with masked logits
//   3  element by element: |l| > cap, a NaN
// CAP_FAR has 0 (up to 512 T, its linear part apart) and 3, by differences; vectors without
// a term (beam_nothing) are passed over there.
// Without softcap way 0 takes all but NaNs: 2^-inf is 0.  PARTS: several items of a
// load (kept apart: the vectors that live on to the end cost the other kind 3 us of 43).
template <int DT, bool VEC, int CAP, bool PARTS>
__global__ void __launch_bounds__(BS_THREADS, BS_CTAS) beam_stream_kernel(const __grid_constant__ BeamArgs a)
{
    using T = DtypeTraits<DT>;
    constexpr int LOAD = 32 * BS_NV * T::VW;  // logits of a load
    const float NEG_INF = -__uint_as_float(0x7f800000u);
    constexpr int STAGE = BS_NV * 512 + (VEC ? 0 : LINE);  // bytes
    __shared__ uint4 s_ring[BS_THREADS / 32 * BS_STAGES * STAGE / 16];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int lane = threadIdx.x & 31;
    const uint32_t ring = (uint32_t)__cvta_generic_to_shared(s_ring) + (threadIdx.x >> 5) * (BS_STAGES * STAGE) + lane * 16;
    const int nw = (int)gridDim.x * (BS_THREADS / 32), w0 = (int)blockIdx.x * (BS_THREADS / 32) + (threadIdx.x >> 5);
    const int step_row = nw / a.rpr, step_run = nw % a.rpr;
    struct Load {
        int row, run, left;  // left: logits from its start to the run's end
        const char *p;
    };
    auto find = [&](int row, int run) {  // the first live run from here on in the warp's steps
        for (;; row += step_row, run += step_run) {
            if (run >= a.rpr) {
                run -= a.rpr;
                row++;
            }
            if (row >= a.rows) return Load{row, run, 0, nullptr};
            if (beam_live(a, row)) break;
        }
        const int e0 = run * a.run_len;
        return Load{row, run, min(a.vocab - e0, a.run_len),
                    (const char *)a.logits + ((int64_t)row * a.row_stride + e0) * T::ESIZE + (VEC ? lane * 16 : 0)};
    };
    auto after = [&](const Load &u) {
        if (u.left > LOAD) return Load{u.row, u.run, u.left - LOAD, u.p + LOAD * T::ESIZE};
        return u.row < a.rows ? find(u.row + step_row, u.run + step_run) : u;
    };
    auto fetch = [&](const Load &u, uint32_t to) {
        const int shift = VEC ? 0 : (int)((uintptr_t)u.p & (LINE - 1));
        const char *p = u.p - shift + (VEC ? 0 : lane * 16);
        if (u.left >= LOAD) {
            ring_copy<0>(to, p);
            if (!VEC && lane * 16 < shift) cp_async16s(to + BS_NV * 512, p + BS_NV * 512);
        } else {
            const int end = shift + u.left * T::ESIZE;
            for (int b = lane * 16; b < end; b += 512, p += 512, to += 512) cp_async16s(to, p);
        }
        cp_async_commit();
    };
    uint64_t h1[BEAM_H1], k2 = two(a.k);
#pragma unroll
    for (int i = 0; i < BEAM_H1; i++) h1[i] = CAP ? two(a.h1[i]) : 0;
    touch_params(a);
    const int row0 = w0 / a.rpr, run0 = w0 % a.rpr;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    Load cur = find(row0, run0), nx = after(cur);
    float m = NEG_INF, ref = 0.0f;
    uint64_t s0 = 0, s1 = 0;
    uint32_t at = ring;
    float4 old = make_float4(0.0f, 0.0f, 0.0f, 0.0f);  // the item before, its sum still to be added up
    int old_at = -1;
    fetch(cur, ring);
    fetch(nx, ring + STAGE);
    while (cur.row < a.rows) {
        uint4 r[BS_NV];
        const bool last = cur.left <= LOAD;
        cp_async_wait<1>();
        if constexpr (VEC) {
            if (cur.left < LOAD) ring_cut<DT>(at, lane, cur.left);
            ring_read<0>(at, r);
        } else {
            const uint32_t from = at - lane * 16, shift = (uint32_t)(uintptr_t)cur.p & (LINE - 1);
            __syncwarp();  // (the lanes read one another's copies)
            if (cur.left < LOAD) {
                ring_cut_shifted<DT>(from, shift, lane, cur.left);
                __syncwarp();
            }
            ring_read_shifted<DT>(from, shift, lane, r);
        }
        if constexpr (!PARTS) {  // beside this load's own work: at the item's end it cost 0.8 us of 43
#pragma unroll
            for (int d = 16; d > 0; d >>= 1) old.z += __shfl_xor_sync(FULLMASK, old.z, d);
            if (lane == 0 && old_at >= 0) a.istat[old_at] = old;
            old_at = -1;
        }
        float mx = lane_max<DT>(r);  // (with the vote, every lane's reads of the ring are done: it can be refilled)
        int way = __all_sync(FULLMASK, CAP != CAP_NONE ? mx <= a.lim1 : mx <= beam_max<DT>()) ? 0 : 1;  // a NaN fails
        const Load n2 = after(nx);
        fetch(n2, at);
        if (way == 1 && CAP == CAP_NONE) {
            way = 3;
        } else if (CAP != CAP_NONE && (way == 1 || !(a.skip_min && __any_sync(FULLMASK, mx >= 0.0f)))) {
            float mn = lane_min<DT>(r);
            if (way == 1 || !__all_sync(FULLMASK, mn >= -a.lim1)) {
                way = CAP == CAP_FOLD && __all_sync(FULLMASK, mx <= a.lim2 && mn >= -a.lim2) ? 1 : 3;
                if (way == 3) {
                    lane_extremes_open<DT>(r, mx, mn);
                    if (CAP == CAP_FOLD && __all_sync(FULLMASK, mx <= a.lim2 && mn >= -a.lim2)) way = 2;
                    mx = fminf(mx, beam_max<DT>());
                }
            }
        }
        if (CAP == CAP_FAR && m > a.lim1) way = 3;  // the item's sum stands against a maximum beyond the polynomial
        const char *p = cur.p - (VEC ? lane * 16 : 0);
        const int n = min(cur.left, LOAD);
        if (way == 3 && CAP == CAP_NONE) {
            mx = NEG_INF;
#pragma unroll 4
            for (int i = lane; i < n; i += 32) mx = fmaxf(mx, beam_raw<DT>(T::load1(p, i)));
        }
        mx = warp_max_redux(mx);
        if (mx > -1e30f) {
            // a new maximum moves the reference (any number near s(m) k, so long as the sums
            // are taken against the same)
            if (mx > m) {
                float to = mx, f = 0.0f;
                if constexpr (CAP == CAP_FOLD) to = beam_value<CAP>(a, mx, 0.0f);
                if constexpr (CAP == CAP_FAR) to = beam_off(a, mx, 0.0f);
                if (m > NEG_INF) {
                    f = CAP == CAP_NONE ? (ref - to) * a.k : ref - to;
                    if (CAP == CAP_FAR && !(fabsf(m) <= a.lim1 && fabsf(mx) <= a.lim1))
                        f = beam_off(a, mx, to) - beam_off(a, m, ref) - beam_below(a, mx, m);
                    f = ex2_approx(f);
                }
                s0 = mul2(s0, two(f, f));
                s1 = mul2(s1, two(f, f));
                m = mx;
                ref = to;
            }
            if (way == 0) {
                load_sum<DT, CAP ? BEAM_H1 : 0, false, CAP == CAP_FAR>(r, h1, k2, ref, s0, s1);
            } else if (CAP == CAP_FOLD && way < 3) {
                uint64_t h2[BEAM_H2];
#pragma unroll
                for (int i = 0; i < BEAM_H2; i++) h2[i] = two(a.h2[i]);
                if (way == 1) load_sum<DT, CAP ? BEAM_H2 : 0, false>(r, h2, k2, ref, s0, s1);
                else load_sum<DT, CAP ? BEAM_H2 : 0, true>(r, h2, k2, ref, s0, s1);
            } else if (CAP == CAP_FAR) {
                float s = 0.0f;
                const float off = beam_off(a, m, ref), none = beam_nothing(a, m);
                uint32_t near = 0;  // the lane's vectors that hold a term
#pragma unroll
                for (int j = 0; j < BS_NV; j++) {
                    float x[T::VW], most = NEG_INF;
                    T::unpack(r[j], x);
#pragma unroll
                    for (int i = 0; i < T::VW; i++) most = fmaxf(most, x[i]);
                    near |= most >= none && most > -1e30f ? 1u << j : 0u;
                }
                near = __reduce_or_sync(FULLMASK, near);
                for (; near; near &= near - 1) {
                    const int j = __ffs(near) - 1;
#pragma unroll 4
                    for (int i = 0; i < T::VW; i++) {
                        // vector j's element i, of aligned rows and of others (whose lanes take every 32nd word)
                        constexpr int WL = 4 / T::ESIZE;
                        const int at = VEC ? (j * 32 + lane) * T::VW + i : ((j * 4 + i / WL) * 32 + lane) * WL + i % WL;
                        const float v = at < n ? beam_raw<DT>(T::load1(p, at)) : NEG_INF;
                        const float e = ex2_approx(off - beam_below(a, m, v));
                        s += v == NEG_INF ? 0.0f : e;
                    }
                }
                s0 = add2(s0, two(s, 0.0f));
            } else {
                float s = 0.0f;
#pragma unroll 4
                for (int i = lane; i < n; i += 32) {
                    const float v = beam_raw<DT>(T::load1(p, i));
                    const float e = ex2_approx(CAP ? __fmaf_rn(beam_soft(v, a), a.k, -ref) : (v - ref) * a.k);
                    s += v == NEG_INF ? 0.0f : e;
                }
                s0 = add2(s0, two(s, 0.0f));
            }
        }
        if (last) {
            const float2 x = halves(add2(s0, s1));
            float S = x.x + x.y;
            if constexpr (!PARTS) {
                old = make_float4(m, ref, S, 0.0f);
                old_at = cur.row * a.ipr + cur.run;
            } else {
#pragma unroll
                for (int d = 16; d > 0; d >>= 1) S += __shfl_xor_sync(FULLMASK, S, d);
                // lane k: the largest of the load's k-th part, S with the first that is m
                float mine = NEG_INF;
#pragma unroll
                for (int j = 0; j < BS_NV; j++) {
                    float x = NEG_INF;
                    if (way < 3) {
                        float v[T::VW];
                        T::unpack(r[j], v);
#pragma unroll
                        for (int i = 0; i < T::VW; i++) x = fmaxf(x, v[i]);
                    } else {
                        for (int i = j * (LOAD / BS_NV) + lane; i < min(n, (j + 1) * (LOAD / BS_NV)); i += 32)
                            x = fmaxf(x, beam_raw<DT>(T::load1(p, i)));
                    }
                    x = warp_max_redux(x);
                    if (lane == j * a.subs / BS_NV) mine = fmaxf(mine, x);
                }
                const unsigned top = __ballot_sync(FULLMASK, lane < a.subs && mine == m);
                const int item = cur.run * a.subs + lane;
                if (lane < a.subs && item < a.ipr)
                    a.istat[cur.row * a.ipr + item] = make_float4(mine, ref, lane == __ffs(top) - 1 ? S : 0.0f, 0.0f);
            }
            m = NEG_INF;
            ref = 0.0f;
            s0 = s1 = 0;
        }
        cur = nx;
        nx = n2;
        at = at == ring ? ring + STAGE : ring;
    }
    cp_async_wait<0>();
    if constexpr (!PARTS) {
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) old.z += __shfl_xor_sync(FULLMASK, old.z, d);
        if (lane == 0 && old_at >= 0) a.istat[old_at] = old;
    }
}

// ---------------------------------------------------------------------------
// combine
// ---------------------------------------------------------------------------
// What is needed to more than 32 bits (the beams' scores meet here) is a sum of two fp32
// numbers, high + low: the error-free sums of Knuth (pair_sum) and Dekker (pair_norm) and the
// product's error by a fused multiply-add (pair_mul).  Measured on this GPU, one dependent
// 64-bit operation takes about 48 cycles and 128 scores in 64 bits 9000; the routines below
// are exact to 3e-11 of their result (checked against 80 bits over their ranges).
struct Pair {
    float h, l;
};
__device__ __forceinline__ Pair pair_sum(float a, float b)  // a + b, exactly
{
    const float s = __fadd_rn(a, b), bb = __fsub_rn(s, a);
    return {s, __fadd_rn(__fsub_rn(a, __fsub_rn(s, bb)), __fsub_rn(b, bb))};
}
__device__ __forceinline__ Pair pair_norm(float a, float b)  // a + b, exactly, for |a| >= |b|
{
    const float s = __fadd_rn(a, b);
    return {s, __fsub_rn(b, __fsub_rn(s, a))};
}
__device__ __forceinline__ Pair pair_add(Pair a, Pair b)
{
    const Pair s = pair_sum(a.h, b.h);
    return pair_norm(s.h, __fadd_rn(s.l, __fadd_rn(a.l, b.l)));
}
__device__ __forceinline__ Pair pair_mul(Pair a, Pair b)
{
    const float p = __fmul_rn(a.h, b.h);
    return pair_norm(p, __fmaf_rn(a.h, b.l, __fmaf_rn(a.l, b.h, __fmaf_rn(a.h, b.h, -p))));
}

// e^z for -180 <= z <= 80, as v 2^e with 1/2 < v < 2: z = n ln2 / 4 + f, |f| <= ln2 / 8, the
// Taylor series to f^6 (its first terms as pairs), times 2^(n / 4).
struct Scaled {
    Pair v;
    int e;
};
static __device__ __noinline__ Scaled pair_exp_scaled(Pair z)
{
    const float t = rintf(__fmul_rn(z.h, 5.770780087f));
    const int n = (int)t;
    // ln2 / 4 in 15 bits, so that the first difference is exact, and the rest
    const Pair f = pair_sum(__fmaf_rn(t, -0.17328643798828125f, z.h), __fmaf_rn(t, -3.571516913e-07f, z.l));
    const float g = __fmul_rn(f.h, f.h), gl = __fmaf_rn(f.h, f.h, -g);
    float c = __fmaf_rn(f.h, 1.0f / 720.0f, 1.0f / 120.0f);
    c = __fmaf_rn(f.h, c, 1.0f / 24.0f);
    c = __fmaf_rn(f.h, c, 1.0f / 6.0f);
    const float cubic = __fmul_rn(__fmul_rn(f.h, g), c);
    Pair s = pair_sum(f.h, 0.5f * g);
    s = pair_norm(s.h, __fadd_rn(__fadd_rn(s.l, f.l), __fadd_rn(__fmaf_rn(0.5f, gl, __fmul_rn(f.h, f.l)), cubic)));
    const Pair o = pair_sum(1.0f, s.h);
    const Pair e = pair_norm(o.h, __fadd_rn(o.l, s.l));
    const int q = n & 3;
    const Pair root = q < 2 ? (q ? Pair{1.189207077f, 3.797635273e-08f} : Pair{1.0f, 0.0f})
                            : (q == 2 ? Pair{1.414213538f, 2.420323497e-08f} : Pair{1.681792855f, -2.475532668e-08f});
    return {pair_mul(e, root), n >> 2};
}
__device__ __forceinline__ Pair pair_exp(Pair z)  // |z| <= 80
{
    const Scaled x = pair_exp_scaled(z);
    const float scale = pow2i(x.e);
    return {x.v.h * scale, x.v.l * scale};
}

// log s for 2^-60 <= s <= 2^60: a first value by the hardware, then ln(s e^-y) from its
// difference to 1.
__device__ __forceinline__ Pair pair_log(Pair s)
{
    float y;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(s.h));
    y *= 0.693147181f;
    const Pair u = pair_mul(s, pair_exp(Pair{-y, 0.0f}));
    const float d = __fadd_rn(__fsub_rn(u.h, 1.0f), u.l);
    return pair_norm(y, __fmaf_rn(-0.5f * d, d, d));
}

enum { BEAM_DEAD = 0, BEAM_LIVE = 1, BEAM_DONE = 2 };
struct BeamRow {
    Pair base;   // score less log of the row's sum (with the softcap less x of its largest logit too)
    Scaled inv;  // 1 / max(length, 1)^alpha (to 2^-248: alpha 8, 2^31 tokens)
    float score, ref;
    int len, kind;
};
__device__ __forceinline__ Scaled beam_length_power(int length, Pair alpha)
{
    const Pair ln = pair_log(pair_sum((float)(length & 0xffff), (float)(length & 0x7fff0000)));
    return pair_exp_scaled(pair_mul(ln, Pair{-alpha.h, -alpha.l}));
}

// What a logit adds to its row's base: cap tanh(l / cap) / T, tanh(q) = 1 - 2 / (e^2q + 1)
// (its cancellation for small q costs 3e-11 of the cap), or (l - ref) / T.
__device__ __forceinline__ Pair beam_x(const BeamArgs &a, float ref, uint32_t key)
{
    const float l = key2f(key);
    if (a.softcap > 0.0f) {
        const float b = 2.0f * fminf(fabsf(l), 20.0f * a.softcap);  // beyond, tanh is 1 to 2^-57
        Pair z;
        z.h = __fmul_rn(b, a.invcap2[0]);
        z.l = __fmaf_rn(b, a.invcap2[1], __fmaf_rn(b, a.invcap2[0], -z.h));
        const Pair e = pair_exp(z);
        Pair d = pair_sum(e.h, 1.0f);
        d.l = __fadd_rn(d.l, e.l);
        const float w = __frcp_rn(d.h), off = __fsub_rn(__fmaf_rn(-d.h, w, 1.0f), __fmul_rn(d.l, w));
        const Pair th = pair_sum(1.0f, -2.0f * w);
        const Pair x = pair_mul(pair_norm(th.h, __fsub_rn(th.l, 2.0f * w * off)), Pair{a.scale2[0], a.scale2[1]});
        return l < 0.0f ? Pair{-x.h, -x.l} : x;
    }
    const Pair d = pair_sum(l, -ref);
    const float x = __fmul_rn(d.h, a.scale2[0]);
    // far below any other, perhaps -inf
    return fabsf(d.h) < 1e30f && fabsf(x) < 1e30f ? pair_mul(d, Pair{a.scale2[0], a.scale2[1]}) : Pair{x, 0.0f};
}

// A continuation's score from its x (which a beam's score of 1e30 or more, or +inf, swallows).
__device__ __forceinline__ Pair beam_score(const BeamRow &r, Pair x)
{
    if (r.kind == BEAM_DONE || !(fabsf(r.score) < 1e30f)) return {r.score, 0.0f};
    return fabsf(x.h) < 1e30f ? pair_add(r.base, x) : x;
}

// A pair as a whole number that orders as it does, and its bits.  With a length power,
// whose exponent may leave fp32's range: sign, 10 bits of exponent, h's mantissa, and l in
// 2^-30 of h's last place.
__device__ __forceinline__ uint64_t beam_rank(const BeamRow &r, Pair score, bool scaled)
{
    if (!scaled) return ((uint64_t)f2key(score.h + 0.0f) << 32) | f2key(score.l + 0.0f);
    int e = 0;
    if (fabsf(score.h) < 1e30f) {
        score = pair_mul(score, r.inv.v);
        e = r.inv.e;
    }
    const uint32_t b = __float_as_uint(fabsf(score.h));
    const int eh = (int)(b >> 23);
    const float l = (score.h < 0.0f ? -score.l : score.l) * pow2i(127 - min(eh, 253));  // |l| <= 2^-24
    uint64_t m = ((uint64_t)(eh + e + 512) << 53 | (uint64_t)(b & 0x7fffffu) << 30) + (int64_t)rintf(l * 0x1p53f);
    if (b == 0) m = 0;
    return score.h < 0.0f ? ~(m | 1ull << 63) : m | 1ull << 63;
}
__device__ __forceinline__ uint64_t pair_bits(Pair x) { return ((uint64_t)__float_as_uint(x.h) << 32) | __float_as_uint(x.l); }
__device__ __forceinline__ Pair bits_pair(uint64_t b) { return {__uint_as_float((uint32_t)(b >> 32)), __uint_as_float((uint32_t)b)}; }

// Order of two continuations: rank, then the lower beam, the larger raw logit, the lower
// id (item): the latter three in one number, larger first.
__device__ __forceinline__ uint64_t beam_tie(int w, uint32_t key, uint32_t id)
{
    return ((uint64_t)(255 - w) << 56) | ((uint64_t)key << 24) | (0xffffffu - id);
}
__device__ __forceinline__ int tie_beam(uint64_t t) { return 255 - (int)(t >> 56); }
__device__ __forceinline__ uint32_t tie_key(uint64_t t) { return (uint32_t)(t >> 24); }
__device__ __forceinline__ uint32_t tie_id(uint64_t t) { return 0xffffffu - (uint32_t)(t & 0xffffffu); }

__device__ __forceinline__ bool beam_before(const ulonglong2 &x, const ulonglong2 &y)
{
    return (x.x > y.x) | ((x.x == y.x) & (x.y > y.y));  // (no branch)
}

// E entries from e0 on of n (rank, tie): each one's place by the entries before it.
template <int E, class Put, class Rest>
__device__ __forceinline__ void beam_places(const ulonglong2 *v, int e0, int n, int N, Put &put, Rest &rest)
{
    const int lane = threadIdx.x & 31;
    ulonglong2 x[E];
    int before[E] = {};
#pragma unroll
    for (int k = 0; k < E; k++) x[k] = v[e0 + k];  // (zeros from n on)
    for (int i0 = 0; i0 < n; i0 += 32) {
        const ulonglong2 y = v[min(i0 + lane, n)];
#pragma unroll
        for (int k = 0; k < E; k++) before[k] += __popc(__ballot_sync(FULLMASK, beam_before(y, x[k])));
    }
#pragma unroll
    for (int k = 0; k < E; k++) {
        if (lane == k && x[k].y) {
            if (before[k] < N) put(before[k], x[k]);
            else rest(x[k].y);
        }
    }
}

// The first N of n entries (rank, tie) in shared memory, in order: put(place, entry) for
// each of them, rest(tie) for each of the others.  Up to 512 entries every one counts those
// before it, a warp one entry at a time, or four (over 64 entries the loads from shared
// memory bound it); more are sorted in place (padded with zeros to P, a power of two).
// Pairs closer than 64 places stay within a warp's 32 exchanges, so only the wider steps
// need the CTA.
template <class Put, class Rest>
__device__ __forceinline__ void beam_first(ulonglong2 *v, int n, int P, int N, Put put, Rest rest)
{
    const int tid = threadIdx.x;
    if (n <= 64) {
        for (int e = tid / 32; e < n; e += BC_WARPS) beam_places<1>(v, e, n, N, put, rest);
    } else if (n <= 512) {
        for (int e = tid / 32 * 4; e < n; e += BC_WARPS * 4) beam_places<4>(v, e, n, N, put, rest);
    } else {
        for (int k = 2; k <= P; k <<= 1) {
            for (int j = k >> 1; j > 0; j >>= 1) {
                for (int t = tid; t < P / 2; t += BC_THREADS) {
                    const int i = 2 * t - (t & (j - 1)), o = i + j;
                    const ulonglong2 x = v[i], y = v[o];
                    if (beam_before(y, x) == ((i & k) == 0)) {
                        v[i] = y;
                        v[o] = x;
                    }
                }
                const int jn = j > 1 ? j >> 1 : k;  // the next step's distance
                if (j > 32 || jn > 32) __syncthreads();
                else __syncwarp();
            }
        }
        __syncthreads();
        for (int e = tid; e < n; e += BC_THREADS) {
            if (v[e].y == 0) continue;
            if (e < N) put(e, v[e]);
            else rest(v[e].y);
        }
    }
    __syncthreads();
}

// The smallest logit of the type with at least this key (NaN, which no logit reaches, above
// the largest finite one's, which +inf has too).
template <int DT>
__device__ __forceinline__ float beam_floor(uint32_t key)
{
    if (key > f2key(beam_max<DT>())) return __uint_as_float(0x7fc00000u);
    if (DT == G4S_BF16) {  // keys of bf16 numbers end in 0000 (from +0 on) or ffff
        const uint32_t low = key & 0x80000000u ? 0u : 0xffffu;
        if ((key & 0xffffu) != low) key = key & 0x80000000u ? (key | 0xffffu) + 1u : key | 0xffffu;
    }
    return key2f(key);
}
constexpr uint32_t BEAM_KEY_MIN = 0xeb60d36u;  // the key after -1e30's

// The unit position of bit `bit` of a lane's mask: logit (j, k) at j * 4 + k (bf16: the words'
// lower halves, then the upper); of rows that no vector load fits, every 32nd logit.
template <int DT, bool VEC>
__device__ __forceinline__ int mask_place(int bit, int lane)
{
    if (!VEC) return bit * 32 + lane;
    if (DT == G4S_F32) return ((bit >> 2) * 32 + lane) * 4 + (bit & 3);
    return (((bit & 15) >> 2) * 32 + lane) * 8 + (bit & 3) * 2 + (bit >> 4);
}

// Which of the lane's logits of a unit (n left) are at or above x.
template <int DT, bool VEC>
__device__ __forceinline__ uint32_t unit_mask(const char *p, int n, int lane, float x)
{
    using T = DtypeTraits<DT>;
    uint32_t m = 0;
    if (VEC && n % T::VW == 0) {
        uint4 r[BNV];  // (past the end: NaN)
#pragma unroll
        for (int j = 0; j < BNV; j++)
            r[j] = (j * 32 + lane) * T::VW < n ? __ldg((const uint4 *)p + j * 32 + lane) : make_uint4(~0u, ~0u, ~0u, ~0u);
#pragma unroll
        for (int j = 0; j < BNV; j++) {
            const uint32_t w[4] = {r[j].x, r[j].y, r[j].z, r[j].w};
#pragma unroll
            for (int k = 0; k < 4; k++) {
                uint32_t ge;
                if constexpr (DT == G4S_BF16) {  // both halves at once; x is a bf16 (or NaN) here
                    const uint32_t x2 = __byte_perm(__float_as_uint(x), 0u, 0x3232);
                    asm("set.ge.u32.bf16x2 %0, %1, %2;" : "=r"(ge) : "r"(w[k]), "r"(x2));
                    m |= ge & (0x00010001u << (j * 4 + k));
                } else {
                    asm("set.ge.u32.f32 %0, %1, %2;" : "=r"(ge) : "f"(__uint_as_float(w[k])), "f"(x));
                    m |= ge & (1u << (j * 4 + k));
                }
            }
        }
    } else {
        float v[BeamGeo<DT>::EPL];
#pragma unroll
        for (int i = 0; i < BeamGeo<DT>::EPL; i++) v[i] = T::load1(p, min(mask_place<DT, VEC>(i, lane), n - 1));
#pragma unroll
        for (int i = 0; i < BeamGeo<DT>::EPL; i++)
            m |= (mask_place<DT, VEC>(i, lane) < n && v[i] >= x ? 1u : 0u) << i;
    }
    return m;
}

// CAP_FAR: an item's sum counts this much in the row's of maximum `top` (apart from the
// combine, which waits for its instructions as it is).
static __device__ __noinline__ float beam_weight(const BeamArgs &a, float top, float4 q)
{
    return q.z > 0.0f ? ex2_approx(-beam_below(a, top, q.x) - beam_off(a, q.x, q.y)) : 0.0f;
}

// (64 registers at 1024 threads; the bf16 variant of unaligned rows spills 96 bytes, in its
// units' masks.)
template <int DT, bool VEC>
__global__ void __launch_bounds__(BC_THREADS, 1) beam_combine_kernel(const __grid_constant__ BeamArgs a)
{
    using T = DtypeTraits<DT>;
    constexpr int UNIT = BeamGeo<DT>::UNIT, SH = DT == G4S_BF16 ? 16 : 0;
    const float NEG_INF = -__uint_as_float(0x7f800000u);
    extern __shared__ ulonglong2 s_mem[];
    ulonglong2 *ent = s_mem;                         // [pe] the beams' items: (rank, tie), rank 0: none
    ulonglong2 *list = ent + a.pe;                   // [pe] those that can be among the first
    ulonglong2 *cand = list + a.pe;                  // [pc] collected tokens
    ulonglong2 *first = cand + a.pc;                 // [n_out] the first in order
    __shared__ BeamRow s_row[G4S_BEAM_MAX];
    __shared__ int s_sel[G4S_BEAM_MAX];      // items of the row among the first
    __shared__ uint32_t s_least[G4S_BEAM_MAX];  // the least key of its tokens wanted
    __shared__ int s_m, s_items, s_n;
    __shared__ uint32_t s_bound;             // upper half of a rank that N items reach
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int W = a.beams, N = a.n_out, row0 = (int)blockIdx.x * W;

    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    for (int e = tid; e < 2 * a.pe + a.pc + N; e += BC_THREADS) s_mem[e] = make_ulonglong2(0, 0);
    if (tid < G4S_BEAM_MAX) {
        s_least[tid] = BEAM_KEY_MIN;
        s_sel[tid] = 0;
    }
    if (tid == 0) {
        s_m = s_items = s_n = 0;
        s_bound = 0;
    }
    touch_params(a);
    __syncthreads();
    asm volatile("griddepcontrol.wait;" ::: "memory");

    // 1. two warps a beam (one from 16 beams on): one sums the row, the other takes its
    // n_out largest items and then ranks them
    const bool pairs = W < 16, scaled = a.alpha2[0] != 0.0f;
    if (warp < (pairs ? 2 * W : W)) {
        const bool sums = !pairs || warp < W, takes = !pairs || warp >= W;
        const int w = warp < W ? warp : warp - W, row = row0 + w;
        const float4 *st = a.istat + (int64_t)row * a.ipr;
        float4 q[BIPL];  // (a dead row's are what an earlier call left, and are not used)
#pragma unroll
        for (int j = 0; j < BIPL; j++)
            q[j] = j * 32 + lane < a.ipr ? __ldcg(st + j * 32 + lane) : make_float4(NEG_INF, NEG_INF, 0.0f, 0.0f);
        const float score = a.scores[row];
        const int len = a.lens ? a.lens[row] : 0;
        const int kind = !(score > NEG_INF) ? BEAM_DEAD : (a.done && a.done[row]) ? BEAM_DONE : BEAM_LIVE;
        uint32_t key[BIPL], kmax = 0;  // (bf16 keys: the upper half tells them apart)
#pragma unroll
        for (int j = 0; j < BIPL; j++) {
            key[j] = beam_key<DT>(q[j].x) >> SH;
            kmax = max(kmax, key[j]);
        }
        const uint32_t best = __reduce_max_sync(FULLMASK, kmax);
        const bool live = kind == BEAM_LIVE && best;
        auto full = [](uint32_t k) { return SH ? (k << SH) | (k & 0x8000u ? 0u : 0xffffu) : k; };
        if (sums) {
            BeamRow r{{0.0f, 0.0f}, {{1.0f, 0.0f}, 0}, score, 0.0f, len, kind};
            if (live) {
                float f[BIPL], off = 0.0f;
                if (a.kind == CAP_FAR) {
#pragma unroll
                    for (int j = 0; j < BIPL; j++) f[j] = beam_weight(a, key2f(full(best)), q[j]);
                } else {
                    float ref = NEG_INF;
#pragma unroll
                    for (int j = 0; j < BIPL; j++)
                        if (key[j]) ref = fmaxf(ref, q[j].y);
                    r.ref = warp_max_redux(ref);
                    if (a.kind == CAP_FOLD) off = beam_value<CAP_FOLD>(a, key2f(full(best)), r.ref);
#pragma unroll
                    for (int j = 0; j < BIPL; j++) f[j] = ex2_approx((q[j].y - r.ref) * a.ref32);
                }
                Pair sum{0.0f, 0.0f};
#pragma unroll
                for (int j = 0; j < BIPL; j++) {
                    const Pair s = pair_sum(sum.h, key[j] ? q[j].z * f[j] : 0.0f);
                    sum = {s.h, sum.l + s.l};
                }
#pragma unroll
                for (int d = 16; d > 0; d >>= 1) {
                    const Pair s = pair_sum(sum.h, __shfl_xor_sync(FULLMASK, sum.h, d));
                    sum = {s.h, s.l + (sum.l + __shfl_xor_sync(FULLMASK, sum.l, d))};
                }
                const Pair ln = pair_log(pair_norm(sum.h, sum.l));
                r.base = pair_add(Pair{score, 0.0f}, Pair{-ln.h, __fmaf_rn(off, 0.693147182f, -ln.l)});
            }
            if (a.alpha2[0] != 0.0f)
                r.inv = beam_length_power(max(kind == BEAM_LIVE ? len + 1 : len, 1), Pair{a.alpha2[0], a.alpha2[1]});
            if (lane == 0) s_row[w] = r;
            __syncwarp();
            if (pairs) asm volatile("bar.arrive %0, 64;" ::"r"(1 + w) : "memory");
        }
        int cnt = 0;
        Pair top{0.0f, 0.0f};  // x of the row's largest logit
        if (takes && kind == BEAM_DONE) {
            if (lane == 0) ent[w * N].y = beam_tie(w, 0u, 0u);
            cnt = 1;
        } else if (takes && live) {
            int nv = 0;
#pragma unroll
            for (int j = 0; j < BIPL; j++) nv += __popc(__ballot_sync(FULLMASK, key[j] != 0));
            // the largest `above` with at least N items at or above it, between the least of
            // the lanes' largest (for N <= 32) and the largest; out early at N exactly
            cnt = min(N, nv);
            uint32_t above = 0;  // keys over it are taken, then those equal to it
            if (nv > N) {
                uint32_t lo = max(N <= 32 ? __reduce_min_sync(FULLMASK, kmax) : 0u, 1u), hi = best;
                for (above = lo; lo < hi;) {
                    const uint32_t mid = lo + (hi - lo + 1) / 2;
                    int n = 0;
#pragma unroll
                    for (int j = 0; j < BIPL; j++) n += __popc(__ballot_sync(FULLMASK, key[j] >= mid));
                    if (n == N) {
                        above = mid - 1;
                        break;
                    }
                    if (n > N) lo = mid;
                    else hi = mid - 1;
                    above = lo;
                }
            }
            const unsigned below = (1u << lane) - 1;
            int o = w * N;
#pragma unroll
            for (int j = 0; j < BIPL; j++) {
                const unsigned b = __ballot_sync(FULLMASK, key[j] > above);
                if (key[j] > above) ent[o + __popc(b & below)].y = beam_tie(w, full(key[j]), (uint32_t)(j * 32 + lane));
                o += __popc(b);
            }
            if (o < w * N + cnt) {  // equals, the lowest first
#pragma unroll
                for (int j = 0; j < BIPL; j++) {
                    const unsigned b = __ballot_sync(FULLMASK, key[j] == above);
                    const int at = o + __popc(b & below);
                    if (key[j] == above && at < w * N + cnt) ent[at].y = beam_tie(w, full(above), (uint32_t)(j * 32 + lane));
                    o += __popc(b);
                }
            }
            __syncwarp();
            const float ref = key2f(full(best));
            bool have = false;
            for (int i = lane; i < cnt; i += 32) {
                const uint32_t k = tie_key(ent[w * N + i].y);
                const Pair x = beam_x(a, ref, k);
                ent[w * N + i].x = pair_bits(x);
                if (k == full(best)) top = x, have = true;
            }
            const int from = __ffs(__ballot_sync(FULLMASK, have)) - 1;  // (the largest is among them)
            top.h = __shfl_sync(FULLMASK, top.h, from);
            top.l = __shfl_sync(FULLMASK, top.l, from);
        }
        if (takes) {
            if (pairs) asm volatile("bar.sync %0, 64;" ::"r"(1 + w) : "memory");
            else __syncwarp();
            BeamRow r = s_row[w];
            if (live && a.softcap > 0.0f) {  // the sum stands against it
                r.base = pair_add(r.base, Pair{-top.h, -top.l});
                __syncwarp();
                if (lane == 0) s_row[w].base = r.base;
            }
            uint32_t low = 0xffffffffu;
            for (int i = lane; i < cnt; i += 32) {
                const uint64_t rank = beam_rank(r, beam_score(r, bits_pair(ent[w * N + i].x)), scaled);
                ent[w * N + i].x = rank;
                low = min(low, (uint32_t)(rank >> 32));
            }
            low = __reduce_min_sync(FULLMASK, low);
            if (lane == 0) {
                atomicAdd(&s_items, cnt);
                if (cnt == N) atomicMax(&s_bound, low);
            }
        }
    }
    __syncthreads();

    // 2. the items by their best token; below the best beam's last one they are out at once
    auto out = [&](uint64_t tie) { atomicMax(&s_least[tie_beam(tie)], tie_key(tie)); };
    for (int e = tid; e < W * N; e += BC_THREADS) {
        const ulonglong2 x = ent[e];
        if (x.y == 0) continue;
        if ((uint32_t)(x.x >> 32) >= s_bound) list[atomicAdd(&s_n, 1)] = x;
        else out(x.y);
    }
    __syncthreads();
    beam_first(
        list, s_n, a.pe, N,
        [&](int at, const ulonglong2 &x) {
            first[at] = x;
            atomicAdd(&s_sel[tie_beam(x.y)], 1);
        },
        out);
    const int nsel = min(N, s_items);
    // a beam's tokens count from its best item left out; where all of its N items are
    // in, from the last of them; where it has no more, all
    auto least = [&](int w) { return s_sel[w] == N ? max(tie_key(first[N - 1].y), BEAM_KEY_MIN) : s_least[w]; };

    // 3. their tokens, a warp a unit.  Where they are more than fit (equal logits, a small
    // vocabulary), again item by item: only n_out - j of the item in place j can count (the
    // j items before it hold a better token each).
    auto push = [&](int w, uint32_t key, int64_t id) {
        const int o = atomicAdd(&s_m, 1);
        if (o < a.pc) cand[o] = make_ulonglong2(0, beam_tie(w, key, (uint32_t)id));
    };
    const int tasks = (a.item_len + UNIT - 1) / UNIT;  // of an item
    for (int task = warp; task < nsel * tasks; task += BC_WARPS) {
        const int j = task / tasks, u = (task - j * tasks) * UNIT;
        const uint64_t t = first[j].y;
        const int w = tie_beam(t);
        if (s_row[w].kind == BEAM_DONE) {
            if (lane == 0 && u == 0) push(w, 0u, 0);
            continue;
        }
        const int64_t e0 = (int64_t)tie_id(t) * a.item_len + u;
        const int n = (int)min((int64_t)min(UNIT, a.item_len - u), a.vocab - e0);
        if (n <= 0) continue;
        const char *p = (const char *)a.logits + ((int64_t)(row0 + w) * a.row_stride + e0) * T::ESIZE;
        const uint32_t key0 = least(w);
        uint32_t m = unit_mask<DT, VEC>(p, n, lane, beam_floor<DT>(key0));
        if (key0 == BEAM_KEY_MIN && N - j <= 32) {
            // nothing bounds this beam's tokens: the N - j largest are at or above the
            // (N - j)-th largest of the lanes' maxima
            uint32_t k = 0;
            for (uint32_t q = m; q; q &= q - 1)
                k = max(k, beam_key<DT>(T::load1(p, mask_place<DT, VEC>(__ffs(q) - 1, lane))));
            k = __shfl_sync(FULLMASK, warp_sort_desc_u32(k), N - j - 1);
            if (k) m = unit_mask<DT, VEC>(p, n, lane, beam_floor<DT>(k));
        }
        for (; m; m &= m - 1) {
            const int e = mask_place<DT, VEC>(__ffs(m) - 1, lane);
            push(w, beam_key<DT>(T::load1(p, e)), e0 + e);
        }
    }
    __syncthreads();
    int m = s_m;
    if (m > a.pc) {
        __syncthreads();
        for (int e = tid; e < a.pc; e += BC_THREADS) cand[e] = make_ulonglong2(0, 0);
        if (tid == 0) s_m = 0;
        __syncthreads();
        for (int j = warp; j < nsel; j += BC_WARPS) {
            const uint64_t t = first[j].y;
            const int w = tie_beam(t), quota = N - j;
            if (s_row[w].kind == BEAM_DONE) {
                if (lane == 0) push(w, 0u, 0);
                continue;
            }
            const int64_t e0 = (int64_t)tie_id(t) * a.item_len;
            const int n = (int)min((int64_t)a.item_len, a.vocab - e0);
            const char *p = (const char *)a.logits + ((int64_t)(row0 + w) * a.row_stride + e0) * T::ESIZE;
            auto count = [&](uint32_t key, uint32_t but, int upto) {  // of keys key .. but - 1, at places up to `upto`
                int c = 0;
#pragma unroll 1
                for (int u = 0; u < n; u += UNIT) {
                    const char *pu = p + (int64_t)u * T::ESIZE;
                    uint32_t m = unit_mask<DT, VEC>(pu, min(n - u, UNIT), lane, beam_floor<DT>(key));
                    if (but) m &= ~unit_mask<DT, VEC>(pu, min(n - u, UNIT), lane, beam_floor<DT>(but));
                    for (; upto < n && m; m &= m - 1) c += u + mask_place<DT, VEC>(__ffs(m) - 1, lane) <= upto;
                    c += __popc(m);
                }
                return (int)__reduce_add_sync(FULLMASK, c);
            };
            // the quota-th largest key, and the place up to which its equals are taken
            uint32_t lo = least(w), hi = tie_key(t);
            int last = n;
            if (count(lo, 0u, n) > quota) {
                while (lo < hi) {
                    const uint32_t mid = lo + (hi - lo) / 2 + 1;
                    if (count(mid, 0u, n) >= quota) lo = mid;
                    else hi = mid - 1;
                }
                const int need = quota - count(lo + 1, 0u, n);
                int p0 = 0;
                last = n - 1;
                while (p0 < last) {
                    const int mid = (p0 + last) / 2;
                    if (count(lo, lo + 1, mid) >= need) last = mid;
                    else p0 = mid + 1;
                }
            }
            for (int u = 0; u < n; u += UNIT) {
                const char *pu = p + (int64_t)u * T::ESIZE;
                for (uint32_t m = unit_mask<DT, VEC>(pu, min(n - u, UNIT), lane, beam_floor<DT>(lo)); m; m &= m - 1) {
                    const int e = mask_place<DT, VEC>(__ffs(m) - 1, lane);
                    const uint32_t key = beam_key<DT>(T::load1(pu, e));
                    if (key > lo || u + e <= last) push(w, key, e0 + u + e);
                }
            }
        }
        __syncthreads();
        m = min(s_m, a.pc);  // (never more, unless the logits changed since the streaming pass)
    }
    for (int e = tid; e < m; e += BC_THREADS) {
        const uint64_t t = cand[e].y;
        const BeamRow &r = s_row[tie_beam(t)];
        cand[e].x = beam_rank(r, beam_score(r, beam_x(a, r.ref, tie_key(t))), scaled);
    }
    __syncthreads();
    beam_first(
        cand, m, a.pc, N, [&](int at, const ulonglong2 &x) { first[at] = x; }, [](uint64_t) {});
    if (tid < N) {
        const int64_t o = (int64_t)blockIdx.x * N + tid;
        float score = NEG_INF;
        int parent = -1, token = -1, len = 0, done = 0;
        if (tid < m) {
            const uint64_t t = first[tid].y;
            const int w = tie_beam(t);
            const BeamRow &r = s_row[w];
            score = scaled ? beam_score(r, beam_x(a, r.ref, tie_key(t))).h : key2f((uint32_t)(first[tid].x >> 32));
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

template <int DT, bool VEC, int CAP, bool PARTS>
static cudaError_t launch_stream(const BeamArgs &a, int sms, cudaStream_t s)
{
    static int bps[MAX_DEVICES] = {};
    const int dev = current_device();
    if (dev < 0 || dev >= MAX_DEVICES) return cudaErrorInvalidDevice;
    if (bps[dev] == 0) {
        const cudaError_t e =
            cudaOccupancyMaxActiveBlocksPerMultiprocessor(&bps[dev], beam_stream_kernel<DT, VEC, CAP, PARTS>, BS_THREADS, 0);
        if (e != cudaSuccess) return e;
    }
    // as many times the CTAs that fit as leave four loads each, so that they end together: 256
    // bf16 rows of 128 loads 42.5 us with 1, 41.6 with 2, 42.5 with 3, 42.2 with 4; 205 live
    // fp32 rows of 256 loads 47.0, 45.7, 45.0, 44.1; but 248 fp32 rows of 30 loads 16.4 with
    // 1, 18.2 with 4.  (CTAs of four warps: 4 rows 9.7 us for 9.15, 30 rows of 32003 logits
    // 10.2 for 9.8.)
    static_assert(BS_THREADS == 32, "a CTA takes one run at a time");
    const int64_t blocks = (int64_t)a.rows * a.rpr, fit = (int64_t)bps[dev] * sms;
    const int64_t loads = blocks * (a.run_len / (32 * BS_NV * DtypeTraits<DT>::VW));
    int64_t most = fit;
    for (int m = 2; m <= 4 && loads >= 4 * fit * m; m++) most = fit * m;
    return launch_dependent(beam_stream_kernel<DT, VEC, CAP, PARTS>, blocks < most ? blocks : most, BS_THREADS, 0, s, a);
}

template <int DT, bool VEC, int CAP>
static cudaError_t launch_beam_t(BeamArgs &a, int sms, cudaStream_t s)
{
    static bool ready[MAX_DEVICES] = {};
    const int dev = current_device();
    if (dev < 0 || dev >= MAX_DEVICES) return cudaErrorInvalidDevice;
    cudaError_t e;
    if (!ready[dev]) {
        e = cudaFuncSetAttribute(beam_combine_kernel<DT, VEC>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 BEAM_COMBINE_SMEM_MAX);
        if (e != cudaSuccess) return e;
        ready[dev] = true;
    }
    // up to BEAM_MAX_ITEMS items a row: of several loads where there are more, of parts of
    // one where there are few (an item has to hold few of the best tokens: 28 bf16 rows of
    // 2520 logits 124 us with whole loads, 15 with parts), to BEAM_PART_ITEMS at most (the
    // parts' maxima cost the streaming pass: 180 bf16 rows of 54 loads 27.2 us in halves,
    // 24.5 whole; 28 rows of 10 loads 11.5 with 4 parts a load, 12.4 with 2)
    const int load = 32 * BS_NV * DtypeTraits<DT>::VW, loads = (a.vocab + load - 1) / load;
    a.run_len = (loads + BEAM_MAX_ITEMS - 1) / BEAM_MAX_ITEMS * load;
    a.rpr = (a.vocab + a.run_len - 1) / a.run_len;
    for (a.subs = BS_NV; a.subs > 1 && loads * a.subs > BEAM_PART_ITEMS;) a.subs /= 2;
    a.item_len = a.run_len / a.subs;
    a.ipr = (a.vocab + a.item_len - 1) / a.item_len;
    e = a.subs > 1 ? launch_stream<DT, VEC, CAP, true>(a, sms, s) : launch_stream<DT, VEC, CAP, false>(a, sms, s);
    if (e != cudaSuccess) return e;
    return launch_dependent(beam_combine_kernel<DT, VEC>, a.rows / a.beams, BC_THREADS,
                            (size_t)(2 * a.pe + a.pc + a.n_out) * 16, s, a);
}

// tanh(q) / q = 1 + q^2 P(q^2) on |q| <= 1/2, P of degree 3 fitted for the least largest
// relative error (1.5e-8)
static const double BEAM_TH[4] = {-0.3333314389543194, 0.13325878934833307, -0.05304549251234199, 0.017241487414783898};

// Largest cap / T of CAP_FOLD and of CAP_FAR's polynomial, 256 rows of 262144 logits, cap 30:
//   CAP_FOLD / CAP_FAR's polynomial, bf16: 41.8 / 43.5 us; scores off by at most (10 kinds of rows)
//   at cap / T = 30 1.1e-6 / 1.6e-7, 60 2.3e-6 / 1.6e-7, 100 4.1e-6 / 1.1e-7, 400 2.0e-5 / 1.6e-7
//   polynomial / differences: 300 44.0 / 180 us, 500 43.9 / 178; at 1000 the polynomial is off by
//   5.7e-7, at 3000 by 3.2e-6 (43.9 / 89 us), differences by 1e-7
constexpr double BEAM_FOLD = 64.0, BEAM_FAR = 512.0;

template <int DT>
static cudaError_t launch_beam_dt(BeamArgs &a, bool vec, int sms, cudaStream_t s)
{
    if (a.kind == CAP_FOLD)
        return vec ? launch_beam_t<DT, true, CAP_FOLD>(a, sms, s) : launch_beam_t<DT, false, CAP_FOLD>(a, sms, s);
    if (a.kind == CAP_FAR) return vec ? launch_beam_t<DT, true, CAP_FAR>(a, sms, s) : launch_beam_t<DT, false, CAP_FAR>(a, sms, s);
    return vec ? launch_beam_t<DT, true, CAP_NONE>(a, sms, s) : launch_beam_t<DT, false, CAP_NONE>(a, sms, s);
}

cudaError_t launch_beam_select(BeamArgs &a, int dtype, bool vec, int sms, cudaStream_t s)
{
    a.k = (float)a.k64;
    a.ref32 = a.softcap > 0.0f ? 1.0f : a.k;
    const double invcap = a.softcap > 0.0f ? 1.0 / (double)a.softcap : 0.0, invt = a.k64 * 0.69314718055994530942;
    auto pair = [](double v, float (&o)[2]) {
        o[0] = (float)v;
        o[1] = (float)(v - (double)o[0]);
    };
    pair(invcap, a.invcap2);
    pair(a.softcap > 0.0f ? a.softcap * invt : invt, a.scale2);
    pair(a.alpha, a.alpha2);
    a.invcap = (float)invcap;
    // the folded coefficients stay normal numbers for caps of this range only
    const bool fold = a.softcap >= 1e-2f && a.softcap <= 1e3f;
    const double most = (double)a.softcap * invt;
    a.kind = a.softcap > 0.0f ? (most <= BEAM_FOLD ? CAP_FOLD : CAP_FAR) : CAP_NONE;
    a.lim1 = fold && most <= BEAM_FAR ? 0.5f * a.softcap : -1.0f;
    a.lim2 = fold && a.kind == CAP_FOLD ? a.softcap : -1.0f;
    a.skip_min = a.lim1 > 0.0f && most >= 28.0;
    pair(2.0 * 1.4426950408889634074 * invcap, a.two2);
    a.capk2 = (float)(2.0 * a.softcap * a.k64);
    a.sat = 64.0f * a.softcap;
    static const double th[BEAM_H2 - 1] = {G4_TH0, G4_TH1, G4_TH2, G4_TH3, G4_TH4, G4_TH5, G4_TH6};
    a.h1[0] = a.h2[0] = a.k;
    double c = a.k64;
    for (int i = 1; i < BEAM_H2; i++) {
        c *= invcap * invcap;
        a.h2[i] = (float)(c * th[i - 1]);
        if (i < BEAM_H1) a.h1[i] = (float)(c * BEAM_TH[i - 1]);
    }
    return dtype == G4S_F32 ? launch_beam_dt<G4S_F32>(a, vec, sms, s) : launch_beam_dt<G4S_BF16>(a, vec, sms, s);
}

// ---------------------------------------------------------------------------
// reordering of dense states
// ---------------------------------------------------------------------------
// A thread moves one column (sizeof(V) bytes at one place of a segment) of all of a
// group's rows: every row that is wanted is read before any is written, so that source
// and destination may be the same memory without a copy or a barrier, and a parent of
// several rows is read once.  Bound by memory: 801 MB read and written in 122 us, 6.5 TB/s,
// the bandwidth of a copy; one prompt's 1.6 MB take 4.3 us, latency.  With more beams the
// columns' registers leave fewer threads on an SM to hide it (60 registers to 8 beams, 100 to
// 16, 230 to 32): the same bytes in groups of 4, 8, 16 and 32 rows 123, 122, 130 and 150 us,
// in place (a row that stays is not moved) 98, 115, 127 and 150.
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
__global__ void __launch_bounds__(REORDER_THREADS) beam_reorder_kernel(const __grid_constant__ ReorderArgs a)
{
    __shared__ uint32_t s_child[WMAX];  // rows of the group that take row p's state
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int W = a.beams;
    int i = 0;
    while (i + 1 < a.n && (int64_t)blockIdx.x >= a.first[i + 1]) i++;
    const ReorderTensor &t = a.t[i];
    const int64_t b = (int64_t)blockIdx.x - a.first[i];
    const int row0 = (int)(b / t.blocks) * W;
    asm volatile("griddepcontrol.wait;" ::: "memory");
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
    if (a.beams <= 4) return launch_dependent(beam_reorder_kernel<4>, blocks, REORDER_THREADS, 0, s, a);
    if (a.beams <= 8) return launch_dependent(beam_reorder_kernel<8>, blocks, REORDER_THREADS, 0, s, a);
    if (a.beams <= 16) return launch_dependent(beam_reorder_kernel<16>, blocks, REORDER_THREADS, 0, s, a);
    return launch_dependent(beam_reorder_kernel<32>, blocks, REORDER_THREADS, 0, s, a);
}

}  // namespace g4s
