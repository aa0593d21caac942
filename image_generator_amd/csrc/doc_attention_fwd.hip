// Document attention, forward, on the matrix units.
//
// A wave owns 32 rows (a lane its row: S^T = K Q^T leaves a row's scores in two lanes, so the softmax statistics are lane-local
// plus one exchange), a workgroup four waves that share staged tiles of 64 keys.  One pass over the keys with the running
// sum, the maximum only where it is needed; scores never leave registers.  The key loop runs over the union of the rows'
// intervals, a wave skips the tiles that none of its rows sees and masks only those that some row sees in part.
//
// Probabilities are rounded to bf16, the matrix units' type, the sum is of the fp32 values: 0.24 % instead of 0.17 % in the 2-norm
// of a result that is itself rounded to bf16.
//
// Measured, with what bounds it: 58 255 caption tokens, 8 heads of 96 (358 MB): 87 us, 4.1 TB/s against 5.2 for a copy, the rest is
// the chain of a short workgroup (offsets, rows, keys, store).  Four documents of 4001 .. 8191 tokens, 8 heads on 2 of 64, causal
// with prefix, cap and bias (149 GFLOP): 349 us, 427 TFLOP/s, bound by vector issue (81 % of the cycles, a score's tanh, bias,
// exp2, sum and conversion against two products).  32768 image rows over 210 keys, 8 heads of 40: 21 us.
#include "doc_tiles.h"
#include <mutex>
#include <type_traits>

namespace {

template <int ND, int NO>
struct Rows {                        // a wave's 32 rows
    bf16x8 qf[ND];
    f32x16 o[NO];
    float m, l;
    int token, head;
    bool live;                       // the row exists
    RowSpan span;
    float slope2;
    unsigned drop;
    int lo, hi;                      // union of the intervals (wave-uniform)
    int in_lo, in_hi;                // their intersection
    int c_min;                       // first key position of a row

    // R0: the wave's first row, `rows` the end of its rows (32 at most)
    __device__ __forceinline__ void init(const DocArgs& p, unsigned R0, unsigned rows, int hk) {
        const unsigned R = R0 + (threadIdx.x & 31);
        live = R < rows;
        row_of(p, live ? R : rows - 1, hk, token, head);
        const int first = __builtin_amdgcn_readfirstlane(token);
        const OffWindow window = off_window(p.q_off, p.docs, p.Tq, first);
        load_row(qf, q_row(p, token, head), p.D);     // on its way while the intervals are looked up
        span = row_span_in(p, token, doc_of_wave(p.q_off, p.docs, window, first, __builtin_amdgcn_readlane(token, 31), token));
        if (!live) span.lo = span.hi = 0;
        const bool sees = span.hi > span.lo;
        lo = wave_min_i(sees ? span.lo : 0x7fffffff);
        hi = wave_max_i(sees ? span.hi : 0);
        // a row without keys asks for no mask: its result is replaced by zeros at the end
        in_lo = wave_max_i(sees ? span.lo : 0);
        in_hi = wave_min_i(sees ? span.hi : 0x7fffffff);
        if (lo > hi) lo = hi = 0;
        c_min = wave_min_i(sees ? span.c : 0x7fffffff);
        slope2 = p.slopes ? p.slopes[head] * LOG2E : 0.f;
        drop = drop_row(p, token, head);
    }
    // the rest of it, which waits for the rows: once the first keys are on their way
    __device__ __forceinline__ void settle(const DocArgs& p) { keep_row(qf, span.hi > span.lo, p.D); }

    // One staged tile of keys k0 .. k0 + 63.  FAST: no running maximum, p = 2^x against the fixed reference 0.  Floating point
    // does not mind the common factor while nothing leaves the normal range, and bf16 probabilities have fp32's exponents; a
    // row whose sum (`fits`) is not within 2^-60 .. 2^100 - scores all below some -40 nats or one beyond 70, or a distance bias
    // on every key it sees - sends its workgroup through the loop again with the maximum.  (Below, the products with values
    // would meet the end of the normal range sooner: values above 2^-66 keep theirs.)
    template <int KIND, bool FAST>
    __device__ __forceinline__ void tile(const DocArgs& p, const Bend& bend, const Reads<ND, NO>& at, const char* Ks, const char* Vs, int k0) {
        const int hh = (threadIdx.x & 63) >> 5;
        f32x16 s[2];
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int r = 0; r < 16; ++r) s[kb][r] = 0.f;
#pragma unroll
        for (int ks = 0; ks < ND; ++ks)
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) s[kb] = mfma(at.frag(Ks, ks, kb), qf[ks], s[kb]);
        float sl2 = bend.scale2;
        if constexpr (KIND != PLAIN) {
            const bool before = k0 + 63 <= c_min;
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) {
                f32x16 y = {};
                if (bend.biased) y = bias16(slope2, (float)(span.c - k0 - kb * 32 - 4 * hh), 0.f, before);
                bend.score16(s[kb], y);
            }
            sl2 = 1.f;
        }
        if (k0 < in_lo || k0 + 64 > in_hi) {
            const unsigned rel = (unsigned)(k0 + 4 * hh - span.lo), len = (unsigned)(span.hi - span.lo);
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if (rel + (unsigned)(kb * 32 + reg_row(r)) >= len) s[kb][r] = -INFINITY;
        }
        float ref = 0.f;
        if constexpr (!FAST) {
            float mx = -INFINITY;
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[kb][r]);
            mx = fmaxf(mx, __shfl_xor(mx, 32, 64)) * sl2;
            const float m_new = fmaxf(m, mx);
            ref = m_new == -INFINITY ? 0.f : m_new;
            const float alpha = EXP2(m - ref);
            l *= alpha;
            if (__ballot(m_new != m) != 0) {
#pragma unroll
                for (int i = 0; i < NO; ++i)
#pragma unroll
                    for (int r = 0; r < 16; ++r) o[i][r] *= alpha;
            }
            m = m_new;
        }
        bf16x8 pf[2][2];
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                float e;
                if constexpr (FAST) e = EXP2(KIND == PLAIN ? s[kb][r] * sl2 : s[kb][r]);
                else e = EXP2(fmaf(s[kb][r], sl2, -ref));
                l += e;
                if constexpr (KIND == DROPPED) e = drop_keep(p, drop, k0 + kb * 32 + reg_row(r) + 4 * hh) ? e * p.drop_scale : 0.f;
                pf[kb][r >> 3][r & 7] = (bf16_t)e;
            }
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int st = 0; st < 2; ++st)
#pragma unroll
                for (int db = 0; db < NO; ++db) o[db] = mfma(at.frag_t(Vs, db, kb * 2 + st), pf[kb][st], o[db]);
    }
    __device__ __forceinline__ void reset(float reference) {
#pragma unroll
        for (int i = 0; i < NO; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) o[i][r] = 0.f;
        m = reference;
        l = 0.f;
    }
    // the two lanes of a row hold the sums of the keys whose scores they hold
    __device__ __forceinline__ void join() { l += __shfl_xor(l, 32, 64); }
    // the row sees keys of the run [from, to)
    __device__ __forceinline__ bool some(int from, int to) const { return max(span.lo, from) < min(span.hi, to); }
    __device__ __forceinline__ bool fits(int from, int to) const { return !some(from, to) || (l > 0x1p-60f && l < 0x1p100f); }
    // rows whose result is not finite
    __device__ __forceinline__ unsigned bad() const {
        const float z = not_finite(o) + l * 0.f;
        return bad_rows(span.hi > span.lo && !(z == 0.f));
    }
    // The unnormalised result of the run [from, to), for the join; R0: the wave's first row of `rows`.  m = -inf: no key of the run is
    // seen, the values stay unwritten and unread.
    __device__ __forceinline__ void leave(const DocArgs& p, unsigned rows, unsigned R0, int hk, int split, int from, int to) const {
        const int lane = threadIdx.x & 63, hh = lane >> 5;
        const size_t row = ((size_t)hk * rows + R0 + (lane & 31)) * p.splits + split;
        float2* ml = (float2*)p.part;
        float* parts = p.part + (size_t)p.Hkv * rows * p.splits * 2;
        const bool any = live && some(from, to) && !(l == 0.f);
        if (live && hh == 0) ml[row] = make_float2(any ? m : -INFINITY, any ? l : 0.f);
#pragma unroll
        for (int db = 0; db < NO; ++db)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int d = db * 32 + 8 * g + 4 * hh;
                if (any && d < p.D) *(f32x4*)(parts + row * p.D + d) = f32x4{o[db][4 * g], o[db][4 * g + 1], o[db][4 * g + 2], o[db][4 * g + 3]};
            }
        for (unsigned bads = from < to ? bad() : 0u; bads; bads &= bads - 1) {
            const int t = __builtin_ctz(bads);
            float pm, pl, po[2];
            plain_row(p, __shfl(token, t, 64), __shfl(head, t, 64), max(__shfl(span.lo, t, 64), from), min(__shfl(span.hi, t, 64), to), __shfl(span.c, t, 64), pm, pl, po);
            const size_t at = ((size_t)hk * rows + R0 + t) * p.splits + split;
            if (lane == 0) ml[at] = make_float2(pm, pl);
#pragma unroll
            for (int u = 0; u < 2; ++u) if (lane + 64 * u < p.D) parts[at * p.D + lane + 64 * u] = po[u];
        }
    }
};

template <int ND, int NO, int KIND>
__global__ __launch_bounds__(256, NO <= 2 && KIND == PLAIN ? 3 : 2) void doc_fwd_kernel(const DocArgs p, int tiles) {
    __shared__ __attribute__((aligned(16))) char even[2 * TILE_BYTES<NO>], odd[2 * TILE_BYTES<NO>];      // K and V, twice
    __shared__ int range[4][2];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, hh = lane >> 5;
    int unit, hk;
    if (!unit_of(tiles * p.splits, p.Hkv, unit, hk)) return;
    const int split = unit / tiles;
    int tile = unit - split * tiles;
    if (p.causal) tile = tiles - 1 - tile;       // the last rows of a document see most: the longest work first
    Rows<ND, NO> w;
    w.init(p, tile * 128u + wave * 32, (unsigned)p.Tq * (unsigned)p.G, hk);
    if (lane == 0) { range[wave][0] = w.hi > w.lo ? w.lo : 0x7fffffff; range[wave][1] = w.hi; }
    __syncthreads();
    const int klo = min(min(range[0][0], range[1][0]), min(range[2][0], range[3][0]));
    const int khi = max(max(range[0][1], range[1][1]), max(range[2][1], range[3][1]));
    int from, to;
    run_of(klo, khi, p.splits, split, from, to);
    const Bend bend(p);
    const bf16_t *kbase = p.k + (size_t)hk * p.D, *vbase = p.v + (size_t)hk * p.D;
    const Reads<ND, NO> at;
    Fetch<NO, 4> kf, vf;
    kf.init(p.ldk, p.D);
    vf.init(p.ldv, p.D);
    auto request = [&](char* to, int k0) __attribute__((always_inline)) {
        kf.dma(to, kbase, p.ldk, p.D, k0, khi - k0);
        vf.dma(to + TILE_BYTES<NO>, vbase, p.ldv, p.D, k0, khi - k0);
    };
    auto pass = [&](auto fast) __attribute__((always_inline)) {
        auto visit = [&](const char* Ks, int k0) __attribute__((always_inline)) {
            if (k0 < w.hi && k0 + 64 > w.lo) w.template tile<KIND, decltype(fast)::value>(p, bend, at, Ks, Ks + TILE_BYTES<NO>, k0);
        };
        w.reset(decltype(fast)::value ? 0.f : -INFINITY);
        if (from < to) request(even, from);
        w.settle(p);
        for (int k0 = from; k0 < to; k0 += 128) {
            tiles_landed();                        // ... and every wave has left the tile before
            if (k0 + 64 < to) request(odd, k0 + 64);
            visit(even, k0);
            if (k0 + 64 >= to) break;
            tiles_landed();
            if (k0 + 128 < to) request(even, k0 + 128);
            visit(odd, k0 + 64);
        }
        w.join();
    };
    // far runs under a distance bias have nothing but tiny sums
    bool shifted = p.splits > 1 && bend.biased;
    if (!shifted) {
        pass(std::true_type{});
        shifted = __syncthreads_or(!w.fits(from, to));             // (the loop has barriers: the workgroup decides as one)
    }
    if (shifted) {
        pass(std::false_type{});
        __syncthreads();
    }
    if (p.splits > 1) {
        w.leave(p, tiles * 128u, tile * 128u + wave * 32, hk, split, from, to);
        return;
    }
    const bool none = w.span.hi <= w.span.lo;
    put_rows<NO>(even + wave * 32 * TILE_LD<NO>, w.o, w.l > 0.f ? 1.f / w.l : 0.f, none,
                 w.live ? p.out + (size_t)w.token * p.ldo + (size_t)w.head * p.D : nullptr, p.D);
    if (w.live && hh == 0) p.lse[(size_t)w.head * p.Tq + w.token] = none ? -INFINITY : w.m + log2f(w.l);
    for (unsigned bad = w.bad(); bad; bad &= bad - 1) {
        const int t = __builtin_ctz(bad);
        const RowSpan s = {__shfl(w.span.lo, t, 64), __shfl(w.span.hi, t, 64), __shfl(w.span.c, t, 64)};
        plain_row_out(p, __shfl(w.token, t, 64), __shfl(w.head, t, 64), s);
    }
}

// Few rows over many keys (single queries over what their documents hold): a wave takes 32 rows and one run of their keys,
// alone - its own staged tiles, no barrier with the others - and leaves an unnormalised result; the join weighs the runs of a
// row against each other.  The rows of a tile may belong to many documents, whose keys lie one behind another: a run is read
// once and only the rows that see a tile take part, so what is bound here is reading K and V: 48 queries over 339 602 keys, 8
// heads on 2 of 96 (261 MB), 74 us, 3.5 TB/s, and 5.5 us for the join.
template <int ND, int NO, int KIND>
__global__ __launch_bounds__(256, 1) void doc_fwd_split_kernel(const DocArgs p) {
    extern __shared__ __attribute__((aligned(16))) char smem_all[];
    const int wave = threadIdx.x >> 6;
    char *Ks = smem_all + wave * 2 * TILE_BYTES<NO>, *Vs = Ks + TILE_BYTES<NO>;
    const int hk = blockIdx.y, split = blockIdx.z * 4 + wave;
    const unsigned R0 = blockIdx.x * (unsigned)p.wave_rows;
    Rows<ND, NO> w;
    w.init(p, R0, min((unsigned)p.Tq * (unsigned)p.G, R0 + p.wave_rows), hk);
    int from, to;
    {
        const int tiles = (w.hi - w.lo + 63) / 64, each = (tiles + p.splits - 1) / p.splits;
        from = w.lo + min(tiles, each * split) * 64;
        to = min(w.hi, w.lo + min(tiles, each * (split + 1)) * 64);
    }
    const Bend bend(p);
    const bf16_t *kbase = p.k + (size_t)hk * p.D, *vbase = p.v + (size_t)hk * p.D;
    const Reads<ND, NO> at;
    Fetch<NO, 1> kf, vf;
    bf16x8 kreg[kf.N], vreg[vf.N];
    kf.init(p.ldk, p.D);
    vf.init(p.ldv, p.D);
    w.reset(-INFINITY);
    w.settle(p);
    {   // (with the running maximum: what bounds this loop is memory, and a distance bias makes far runs tiny)
        if (from < to) {
            kf.load(kreg, kbase, p.ldk, p.D, from, to - from);
            vf.load(vreg, vbase, p.ldv, p.D, from, to - from);
        }
        for (int k0 = from; k0 < to; k0 += 64) {
            // one wave: its LDS operations complete in order, the fences only keep the compiler from reordering them
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            kf.put(kreg, Ks);
            vf.put(vreg, Vs);
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            if (k0 + 64 < to) {
                kf.load(kreg, kbase, p.ldk, p.D, k0 + 64, to - k0 - 64);
                vf.load(vreg, vbase, p.ldv, p.D, k0 + 64, to - k0 - 64);
            }
            // a run ends with whole tiles, or where the last of the rows' intervals does
            w.template tile<KIND, false>(p, bend, at, Ks, Vs, k0);
        }
        w.join();
    }
    w.leave(p, gridDim.x * (unsigned)p.wave_rows, R0, hk, split, from, to);
}

// out = sum o_s 2^(m_s - M) / sum l_s 2^(m_s - M) over the runs of a row: a wave per row, at most 64 runs
__global__ __launch_bounds__(256) void doc_fwd_join_kernel(const DocArgs p, unsigned rows) {
    const int lane = threadIdx.x & 63;
    const unsigned R = blockIdx.x * 4 + (threadIdx.x >> 6);
    const int hk = blockIdx.y;
    if (R >= (unsigned)p.Tq * (unsigned)p.G) return;
    int token, head;
    row_of(p, R, hk, token, head);
    const size_t row = ((size_t)hk * rows + R) * p.splits;
    float2 ml = make_float2(-INFINITY, 0.f);
    if (lane < p.splits) ml = ((const float2*)p.part)[row + lane];
    const bool nan = __ballot(ml.x != ml.x) != 0;
    const float M = wave_max(ml.x);
    const float w = ml.x == -INFINITY ? 0.f : EXP2(ml.x - M);
    const float l = wave_sum(ml.y * w);
    const float* part = p.part + (size_t)p.Hkv * rows * p.splits * 2 + row * p.D;
    // runs with something to add, eight loads at a time (a run that adds nothing is not read: its values were not written)
    float o[2] = {0.f, 0.f};
    const int d0 = min(lane, p.D - 1), d1 = min(lane + 64, p.D - 1);
    unsigned long long who = __ballot(ml.x != -INFINITY);
    while (who) {
        float ws[8], v0[8], v1[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int s = who ? __builtin_ctzll(who) : -1;
            who &= who - 1;
            ws[e] = s < 0 ? 0.f : __shfl(w, s < 0 ? 0 : s, 64);
            v0[e] = v1[e] = 0.f;
            if (s >= 0) {                                  // (uniform)
                v0[e] = part[(size_t)s * p.D + d0];
                v1[e] = part[(size_t)s * p.D + d1];
            }
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            o[0] = fmaf(ws[e], v0[e], o[0]);
            o[1] = fmaf(ws[e], v1[e], o[1]);
        }
    }
    const float inv = nan ? NAN : l > 0.f || l != l ? 1.f / l : 0.f;
    bf16_t* out = p.out + (size_t)token * p.ldo + (size_t)head * p.D;
#pragma unroll
    for (int u = 0; u < 2; ++u) if (lane + 64 * u < p.D) out[lane + 64 * u] = (bf16_t)(o[u] * inv);
    if (lane == 0) p.lse[(size_t)head * p.Tq + token] = nan ? NAN : l == 0.f ? -INFINITY : M + log2f(l);
}

// Rows of a document that are few (single queries) share no tile worth its staging: waves take runs by themselves, about 2048 of them,
// one tile at least, at most 64 for a row.  Where 64 runs of 32 rows make less than 768, a wave takes fewer rows, down to a
// group's: a tile of keys is of use to its own document's rows alone, so nothing is read twice (30 queries of one head over 5000
// keys each: 112 -> 17 us; but the fewer documents a wave has, the less even the runs: 48 queries of two groups over 339 602
// keys, 82 us with 32 rows, 86 with 8).  Longer documents, and few keys (a tile or six, where a second launch costs more): key_runs().
struct Plan {
    bool waves;
    int splits, wave_rows;
    size_t rows;                     // of a key head, padded to whole tiles
};
static Plan plan(int Tq, long long Tk, int Hq, int Hkv, int docs) {
    const long long G = Hq / Hkv, rows = (long long)Tq * G, wgs = (rows + 127) / 128 * Hkv;
    const Plan tiled = {false, key_runs(Tq, (int)Tk, Hq, Hkv, docs), 0, (size_t)(rows + 127) / 128 * 128};
    if (rows == 0 || rows >= 64ll * docs || wgs >= 256 || Tk < 384) return tiled;
    int R = 32;
    while (R > 1 && R / 2 >= G && (rows + R - 1) / R * Hkv * 64 < 768 && Tk * R / rows > 64 * 64) R /= 2;
    const long long tiles = (rows + R - 1) / R;
    long long s = 2048 / (tiles * Hkv);
    const long long most = (Tk / tiles + 63) / 64;
    if (s > most) s = most;
    if (s > 64) s = 64;
    s = s < 4 ? 4 : s / 4 * 4;
    return {true, (int)s, R, (size_t)(tiles * R)};
}

template <int ND, int NO, int KIND>
int launch_split(const DocArgs& a, hipStream_t st) {
    constexpr int LDS = 4 * 2 * TILE_BYTES<NO>;
    static std::once_flag once;
    static hipError_t set;
    std::call_once(once, [] { set = hipFuncSetAttribute((const void*)doc_fwd_split_kernel<ND, NO, KIND>, hipFuncAttributeMaxDynamicSharedMemorySize, LDS); });
    if (set != hipSuccess) return mi355_fail(MI355_ERR_LAUNCH, "doc_attention: %s", hipGetErrorString(set));
    const unsigned tiles = (unsigned)(((long long)a.Tq * a.G + a.wave_rows - 1) / a.wave_rows);
    hipLaunchKernelGGL((doc_fwd_split_kernel<ND, NO, KIND>), dim3(tiles, a.Hkv, a.splits / 4), dim3(256), LDS, st, a);
    hipLaunchKernelGGL(doc_fwd_join_kernel, dim3((unsigned)(((long long)a.Tq * a.G + 3) / 4), a.Hkv), dim3(256), 0, st, a, tiles * a.wave_rows);
    return mi355_check_launch("doc_attention_fwd(split)");
}

template <int ND, int NO>
int launch(const DocArgs& a, const Plan& how, hipStream_t st) {
    const bool bent = a.cap > 0.f || a.slopes || !(a.scale > 0.f);
    if (how.waves)
        return a.drop_thresh ? launch_split<ND, NO, DROPPED>(a, st) : bent ? launch_split<ND, NO, BENT>(a, st) : launch_split<ND, NO, PLAIN>(a, st);
    const int tiles = (int)(how.rows / 128);
    const dim3 grid(unit_grid((long long)tiles * a.splits, a.Hkv));
    if (a.drop_thresh) hipLaunchKernelGGL((doc_fwd_kernel<ND, NO, DROPPED>), grid, dim3(256), 0, st, a, tiles);
    else if (bent) hipLaunchKernelGGL((doc_fwd_kernel<ND, NO, BENT>), grid, dim3(256), 0, st, a, tiles);
    else hipLaunchKernelGGL((doc_fwd_kernel<ND, NO, PLAIN>), grid, dim3(256), 0, st, a, tiles);
    if (a.splits > 1) hipLaunchKernelGGL(doc_fwd_join_kernel, dim3((unsigned)(((long long)a.Tq * a.G + 3) / 4), a.Hkv), dim3(256), 0, st, a, (unsigned)how.rows);
    return mi355_check_launch("doc_attention_fwd");
}

}  // namespace

int doc_fwd_tiles(const DocArgs& a, hipStream_t st) {
    const Plan how = plan(a.Tq, a.Tk, a.Hq, a.Hkv, a.docs);
    DocArgs b = a;
    b.splits = how.splits;
    b.wave_rows = how.wave_rows;
    return BY_WIDTH(a.D, launch, b, how, st);
}
size_t doc_fwd_workspace(int Tq, int Tk, int Hq, int Hkv, int D, int docs) {
    const Plan how = plan(Tq, Tk, Hq, Hkv, docs);
    return how.splits > 1 ? how.rows * Hkv * how.splits * (D + 2) * 4 : 0;
}
