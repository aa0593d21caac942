// Attention over packed documents: what its kernels share.
//
// Tokens of many documents lie one behind another; document n holds the queries q_off[n] .. q_off[n+1] and the keys
// k_off[n] .. k_off[n+1].  Query i of document n sits at the key position c = i + (k_end - q_end) (aligned at the documents'
// ends: appended queries) or i + (k_begin - q_begin), and sees
//     the keys j of its document, with `causal` only those with j <= c or j < k_begin + prefix[n]:
// always an interval [lo, hi), and that is all the kernels know of masks.  Then
//     t = scale q.k;  t = cap tanh(t / cap) if cap > 0;  x = (t - slope[head] |c - j|) log2 e;  p = 2^(x - lse)
// A query that sees nothing, or belongs to no document, gives a row of zeros and lse = -inf.
// Query heads share key heads in groups of G = Hq / Hkv: a kernel's "row" is R = token * G + (query head in its group), so the
// rows of a key head are one list, K and V are read once for a group, and a group's gradients meet in one accumulator.
//
// Offsets come from the device and are not trusted: intervals are clamped to the tensors, whatever they hold.
#pragma once
#include "common.h"

struct DocArgs {
    const bf16_t *q, *k, *v, *o, *dout;
    bf16_t *out, *dq, *dk, *dv;
    float *lse, *delta;             // [Hq][Tq]
    int4* rows;                     // [Tq] {lo, hi, c, 0}: written by the dQ pass for the dK / dV pass
    const int *q_off, *k_off, *prefix;
    const float* slopes;
    long long ldq, ldk, ldv, ldo, lddo, lddq, lddk, lddv;
    int docs, Tq, Tk, Hq, Hkv, G, D;
    int causal, align_start;
    float scale, cap, rcap;         // rcap = 1 / cap
    unsigned drop_thresh, seed;     // an entry is dropped when its hash < drop_thresh
    float drop_scale;
    float* part;                    // partial results of `splits` runs (of keys: forward; of rows: dK and dV); 1: none
    int splits;
    int wave_rows;                  // rows of a wave that takes runs of keys by itself
    float* part_q;                  // the dQ pass's, over `splits_q` runs of keys
    int splits_q;
};

#define LOG2E 1.4426950408889634f

struct RowSpan { int lo, hi, c; };

// largest n < docs with off[n] <= i (0 if there is none)
__device__ __forceinline__ int doc_of(const int* __restrict__ off, int docs, int i) {
    int a = 0, b = docs;                         // off[a] <= i is assumed, off[b] > i
    while (b - a > 1) {
        const int mid = (a + b) >> 1;
        if (off[mid] <= i) a = mid; else b = mid;
    }
    return a;
}

// A document's queries [qb, qe) and its number; qb > qe: none
struct Doc { int n, b, e; };

// The document of token i by itself.
__device__ __forceinline__ Doc doc_at(const int* __restrict__ off, int docs, int i) {
    const int n = doc_of(off, docs, i);
    return {n, off[n], off[n + 1]};
}

// The same for the tokens i of a wave (every lane active, ascending from i0 to i1), out of `total`.  A lane's own binary search is a
// chain of loads, a third of a caption tile's time; here the 64 offsets around the place where documents of equal length would
// have this one are loaded at once and usually hold it - if not, a search that probes 64 places a step says where they are -
// and the lanes take their documents from those registers.
// (At most 2^30 documents: the estimate in fp32 is then some hundred places past the last offset at most, and no index passes 32 bits.)
// Loads return in order: the window is asked for before the rows' own operands, behind which it would wait (OffWindow).
struct OffWindow { int w, val; };        // first offset; the lane's
__device__ __forceinline__ OffWindow off_window(const int* __restrict__ off, int docs, int total, int i0) {
    const int w = max(0, (int)((float)i0 * (float)docs / (float)total) - 24), at = w + (int)(threadIdx.x & 63);
    return {w, off[min(at, docs)]};
}
__device__ __forceinline__ Doc doc_of_wave(const int* __restrict__ off, int docs, const OffWindow& window, int i0, int i1, int i) {
    const int lane = threadIdx.x & 63;
    int w = window.w;
    int val = w + lane <= docs ? window.val : 0x7fffffff;
    int k = __popcll(__ballot(val <= i0));                                      // offsets of the window up to i0
    if ((k == 0 && w > 0) || k == 64) {
        int a = 0, b = docs;
        while (b - a > 1) {
            const int step = (b - a + 63) / 64, at = a + 1 + lane * step;
            const int count = __popcll(__ballot(at < b && off[min(at, docs)] <= i0));
            if (count == 0) break;
            a += 1 + (count - 1) * step;
            b = min(b, a + step);
        }
        w = a;
        val = w + lane <= docs ? off[w + lane] : 0x7fffffff;
        k = __popcll(__ballot(val <= i0));
    }
    Doc d = {w + max(k - 1, 0), __builtin_amdgcn_readlane(val, max(k - 1, 0)), __builtin_amdgcn_readlane(val, max(min(k, 63), 1))};
    for (; k < 64; ++k) {                                                       // documents that begin behind i0
        const int b = __builtin_amdgcn_readlane(val, k);
        if (b > i1) break;
        const int e = __builtin_amdgcn_readlane(val, min(k + 1, 63));
        if (b <= i) d = {w + k, b, e};
    }
    if (d.n - w >= 63 && d.n < docs) return doc_at(off, docs, i);               // past the window: many tiny documents
    if (d.n >= docs) d = {docs - 1, 1, 0};
    return d;
}

__device__ __forceinline__ RowSpan row_span_in(const DocArgs& p, int i, const Doc& q) {
    int kb = q.b, ke = q.e;
    if (p.k_off != p.q_off) { kb = p.k_off[q.n]; ke = p.k_off[q.n + 1]; }
    kb = max(kb, 0);
    ke = min(ke, p.Tk);
    RowSpan s = {0, 0, 0};
    if (i < q.b || i >= q.e || kb >= ke) return s;
    s.c = (int)((long long)i + (p.align_start ? (long long)kb - q.b : (long long)ke - q.e));
    s.lo = kb;
    s.hi = ke;
    if (p.causal) {
        int seen = s.c < kb ? kb : s.c >= ke ? ke : s.c + 1;
        if (p.prefix) seen = max(seen, kb + min(max(p.prefix[q.n], 0), ke - kb));
        s.hi = seen;
    }
    return s;
}

// tokens whose rows may see key j of document k: [first, last)
__device__ __forceinline__ int2 key_span_in(const DocArgs& p, int j, const Doc& k) {
    const int kb = max(k.b, 0), ke = min(k.e, p.Tk);
    int qb = k.b, qe = k.e;
    if (p.k_off != p.q_off) { qb = p.q_off[k.n]; qe = p.q_off[k.n + 1]; }
    if (j < kb || j >= ke || qb >= qe) return make_int2(0, 0);
    long long first = qb;
    if (p.causal && !(p.prefix && j < kb + min(max(p.prefix[k.n], 0), ke - kb))) {
        const long long at = (long long)j - (p.align_start ? (long long)kb - qb : (long long)ke - qe);   // c >= j
        if (at > first) first = at;
    }
    const int last = min(qe, p.Tq);
    const int f = (int)(first < 0 ? 0 : first > last ? last : first);
    return make_int2(f, last);
}
__device__ __forceinline__ int2 key_span(const DocArgs& p, int j) { return key_span_in(p, j, doc_at(p.k_off, p.docs, j)); }

__device__ __forceinline__ float tanh_f(float x) {
    return 1.f - 2.f * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(x * (2.f * LOG2E)));
}

// Dropout of the probability of (query token i, key j, query head): a hash, regenerated in the backward pass.
__device__ __forceinline__ unsigned drop_row(const DocArgs& p, int i, int head) {
    unsigned x = (unsigned)i * 0x9E3779B1u + (unsigned)head * 0x85EBCA6Bu + p.seed;
    x ^= x >> 15; x *= 0x2C1B3C6Du; x ^= x >> 12;
    return x;
}
__device__ __forceinline__ bool drop_keep(const DocArgs& p, unsigned row, int j) {
    unsigned x = row + (unsigned)j * 0xC2B2AE35u;
    x ^= x >> 16; x *= 0x7FEB352Du; x ^= x >> 15; x *= 0x846CA68Bu; x ^= x >> 16;
    return x >= p.drop_thresh;
}

// -------------------------------------------------------------------------------------------------------------------
// One row, or one key, by one wave, without matrix instructions.  This is the definition the tiled kernels fall back on: a
// tile multiplies keys that a row does not see by probabilities of exactly 0, which is only right while those keys are
// finite.  A tiled kernel whose result is not finite hands those rows (keys) to these routines, which touch nothing but what
// the interval holds; on finite data they never run.
// -------------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ float dot_rows(const bf16_t* a, const bf16_t* b, int D) {
    float t = 0.f;
    for (int c = 0; c < D; c += 8) {
        const bf16x8 x = *(const bf16x8*)(a + c), y = *(const bf16x8*)(b + c);
#pragma unroll
        for (int e = 0; e < 8; ++e) t = fmaf((float)x[e], (float)y[e], t);
    }
    return t;
}

// score in log2 units; slope_c = 1 - tanh^2 (1 without a cap)
__device__ __forceinline__ float score2(const DocArgs& p, float dot, int c, int j, float slope, float& bend) {
    float t = dot * p.scale;
    bend = 1.f;
    if (p.cap > 0.f) {
        const float h = tanh_f(t * p.rcap);
        bend = 1.f - h * h;
        t = p.cap * h;
    }
    return (t - slope * fabsf((float)(c - j))) * LOG2E;
}

__device__ __forceinline__ const bf16_t* q_row(const DocArgs& p, int i, int head) { return p.q + (size_t)i * p.ldq + (size_t)head * p.D; }
__device__ __forceinline__ const bf16_t* k_row(const DocArgs& p, int j, int hk) { return p.k + (size_t)j * p.ldk + (size_t)hk * p.D; }
__device__ __forceinline__ const bf16_t* v_row(const DocArgs& p, int j, int hk) { return p.v + (size_t)j * p.ldv + (size_t)hk * p.D; }

// Keys [lo, hi) for one row: maximum m, sum l and the unnormalised output of the lane's columns lane and lane + 64.
__device__ inline void plain_row(const DocArgs& p, int i, int head, int lo, int hi, int c, float& m, float& l, float (&o)[2]) {
    const int lane = threadIdx.x & 63, hk = head / p.G;
    const bf16_t* q = q_row(p, i, head);
    const float slope = p.slopes ? p.slopes[head] : 0.f;
    const unsigned dr = drop_row(p, i, head);
    float bend;
    m = -INFINITY;
    bool nan = false;
    for (int j = lo + lane; j < hi; j += 64) {
        const float x = score2(p, dot_rows(q, k_row(p, j, hk), p.D), c, j, slope, bend);
        nan |= x != x;
        m = fmaxf(m, x);
    }
    m = wave_max(m);
    if (__ballot(nan) != 0) m = NAN;
    l = 0.f;
    o[0] = o[1] = 0.f;
    if (m == -INFINITY) return;
    for (int j0 = lo; j0 < hi; j0 += 64) {
        const int j = j0 + lane;
        float e = 0.f, keep = 0.f;
        if (j < hi) {
            e = __builtin_amdgcn_exp2f(score2(p, dot_rows(q, k_row(p, j, hk), p.D), c, j, slope, bend) - m);
            keep = p.drop_thresh == 0 ? e : drop_keep(p, dr, j) ? e * p.drop_scale : 0.f;
        }
        l += e;
        const int count = min(64, hi - j0);
        for (int t = 0; t < count; ++t) {
            const float w = __shfl(keep, t, 64);
            const bf16_t* v = v_row(p, j0 + t, hk);
#pragma unroll
            for (int u = 0; u < 2; ++u) if (lane + 64 * u < p.D) o[u] = fmaf(w, (float)v[lane + 64 * u], o[u]);
        }
    }
    l = wave_sum(l);
}

// the same, written to out and lse
__device__ inline void plain_row_out(const DocArgs& p, int i, int head, const RowSpan& s) {
    const int lane = threadIdx.x & 63;
    float m, l, o[2];
    plain_row(p, i, head, s.lo, s.hi, s.c, m, l, o);
    const float inv = l == 0.f ? 0.f : 1.f / l;
    bf16_t* out = p.out + (size_t)i * p.ldo + (size_t)head * p.D;
#pragma unroll
    for (int u = 0; u < 2; ++u) if (lane + 64 * u < p.D) out[lane + 64 * u] = (bf16_t)(o[u] * inv);
    if (lane == 0) p.lse[(size_t)head * p.Tq + i] = l == 0.f ? -INFINITY : m + log2f(l);
}

// p(row, key) and dS / scale of one entry; dp = dO.v already scaled for dropout by the caller
__device__ __forceinline__ void plain_entry(const DocArgs& p, int i, int head, int j, int c, float slope, unsigned dr, float lse, float delta,
                                            float& pd, float& ds) {
    const int hk = head / p.G;
    float bend;
    const float x = score2(p, dot_rows(q_row(p, i, head), k_row(p, j, hk), p.D), c, j, slope, bend);
    const float e = lse == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(x - lse);
    float dp = dot_rows(p.dout + (size_t)i * p.lddo + (size_t)head * p.D, v_row(p, j, hk), p.D);
    pd = e;
    if (p.drop_thresh != 0) {
        const bool keep = drop_keep(p, dr, j);
        pd = keep ? e * p.drop_scale : 0.f;
        dp = keep ? dp * p.drop_scale : 0.f;
    }
    ds = e * (dp - delta) * bend;
}

__device__ inline void plain_dq_row(const DocArgs& p, int i, int head, const RowSpan& s, float lse, float delta) {
    const int lane = threadIdx.x & 63, hk = head / p.G;
    const float slope = p.slopes ? p.slopes[head] : 0.f;
    const unsigned dr = drop_row(p, i, head);
    float acc[2] = {0.f, 0.f};
    for (int j0 = s.lo; j0 < s.hi; j0 += 64) {
        float pd = 0.f, ds = 0.f;
        if (j0 + lane < s.hi) plain_entry(p, i, head, j0 + lane, s.c, slope, dr, lse, delta, pd, ds);
        const int count = min(64, s.hi - j0);
        for (int t = 0; t < count; ++t) {
            const float w = __shfl(ds, t, 64);
            const bf16_t* k = k_row(p, j0 + t, hk);
#pragma unroll
            for (int u = 0; u < 2; ++u) if (lane + 64 * u < p.D) acc[u] = fmaf(w, (float)k[lane + 64 * u], acc[u]);
        }
    }
    bf16_t* dq = p.dq + (size_t)i * p.lddq + (size_t)head * p.D;
#pragma unroll
    for (int u = 0; u < 2; ++u) if (lane + 64 * u < p.D) dq[lane + 64 * u] = (bf16_t)(acc[u] * p.scale);
}

// dK and dV of one key of one key head, every query head of its group
__device__ inline void plain_dkdv_key(const DocArgs& p, int j, int hk) {
    const int lane = threadIdx.x & 63;
    const int2 span = key_span(p, j);
    float ak[2] = {0.f, 0.f}, av[2] = {0.f, 0.f};
    for (int g = 0; g < p.G; ++g) {
        const int head = hk * p.G + g;
        const float slope = p.slopes ? p.slopes[head] : 0.f;
        for (int i0 = span.x; i0 < span.y; i0 += 64) {
            const int i = i0 + lane;
            float pd = 0.f, ds = 0.f;
            bool sees = false;
            if (i < span.y) {
                const int4 r = p.rows[i];
                sees = j >= r.x && j < r.y;
                if (sees) {
                    const size_t at = (size_t)head * p.Tq + i;
                    plain_entry(p, i, head, j, r.z, slope, drop_row(p, i, head), p.lse[at], p.delta[at], pd, ds);
                }
            }
            unsigned long long who = __ballot(sees);
            while (who) {
                const int t = __builtin_ctzll(who);
                who &= who - 1;
                const float wp = __shfl(pd, t, 64), wd = __shfl(ds, t, 64);
                const bf16_t *q = q_row(p, i0 + t, head), *g_ = p.dout + (size_t)(i0 + t) * p.lddo + (size_t)head * p.D;
#pragma unroll
                for (int u = 0; u < 2; ++u)
                    if (lane + 64 * u < p.D) {
                        ak[u] = fmaf(wd, (float)q[lane + 64 * u], ak[u]);
                        av[u] = fmaf(wp, (float)g_[lane + 64 * u], av[u]);
                    }
            }
        }
    }
    bf16_t *dk = p.dk + (size_t)j * p.lddk + (size_t)hk * p.D, *dv = p.dv + (size_t)j * p.lddv + (size_t)hk * p.D;
#pragma unroll
    for (int u = 0; u < 2; ++u)
        if (lane + 64 * u < p.D) {
            dk[lane + 64 * u] = (bf16_t)(ak[u] * p.scale);
            dv[lane + 64 * u] = (bf16_t)av[u];
        }
}
