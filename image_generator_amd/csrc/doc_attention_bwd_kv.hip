// Document attention, dK and dV, on the matrix units: a lane owns its key (S = Q K^T, dP = dO V^T), a wave 32 keys, and
// staged tiles of 64 rows - tokens times the query heads that share the key head - pass by: dV^T += dO^T P,
// dK^T += Q^T dS.  -lse and -delta of a row start the accumulators of its scores, so subtracting them costs nothing.
//
// P and dS are rounded to bf16 for their products, as in the other passes; sums over rows and heads are fp32.
//
// Measured, with what bounds it: 58 255 caption tokens, 8 heads of 96 (537 MB): 160 us, 3.4 TB/s, a chain per workgroup as in the
// dQ pass with four products instead of three.  Four documents of 4001 .. 8191 tokens, 8 heads on 2 of 64, causal with prefix, cap and
// bias (298 GFLOP): 673 us, 443 TFLOP/s: 229 registers leave two waves per SIMD, whose scores and products follow each other
// (vector issue 57 %, matrix units 25 % of the cycles), and 30 us for the join.  32768 image rows over 210 keys, 8 heads of 40:
// 33 us and 6 us for the join.
//
// Few keys under many rows (captions under image tokens) leave most of the chip idle: the rows of a key tile are then cut
// into `splits` runs whose fp32 partial gradients a second launch adds, in their order.  No atomics anywhere.
#include "doc_tiles.h"

namespace {

// 64-row tiles of Q and dO: rows are (token, head of the group)
template <int NO>
struct RowFetch {
    static constexpr int N = Fetch<NO, 4>::N;
    int vq[N], vg[N];
    __device__ __forceinline__ void init(const DocArgs& p, unsigned phase) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const unsigned x = phase + Fetch<NO, 4>::row_of_slot(i), c = Fetch<NO, 4>::col_of_slot(i);
            const unsigned t = p.G == 1 ? x : x / (unsigned)p.G, g = x - t * (unsigned)p.G;
            const bool in = (int)c * 8 < p.D;
            vq[i] = in ? (int)(t * p.ldq + g * p.D + c * 8) * 2 : NOWHERE;
            vg[i] = in ? (int)(t * p.lddo + g * p.D + c * 8) * 2 : NOWHERE;
        }
    }
    // rows from token t0 on, tokens below `end`
    __device__ __forceinline__ void dma(char* q, char* g, const DocArgs& p, int hk, int t0, int end) const {
#if defined(__HIP_DEVICE_COMPILE__)
        const int n = min(end - t0, 65);                // 64 rows lie in at most 64 tokens, one more if they begin inside one
        const size_t first = (size_t)hk * p.G * p.D;
        const __amdgpu_buffer_rsrc_t rq = __builtin_amdgcn_make_buffer_rsrc(
            (void*)(p.q + (size_t)t0 * p.ldq + first), 0, (unsigned)(((long long)(n - 1) * p.ldq + (long long)p.G * p.D) * 2), 0x00020000);
        const __amdgpu_buffer_rsrc_t rg = __builtin_amdgcn_make_buffer_rsrc(
            (void*)(p.dout + (size_t)t0 * p.lddo + first), 0, (unsigned)(((long long)(n - 1) * p.lddo + (long long)p.G * p.D) * 2), 0x00020000);
        const int piece = (int)__builtin_amdgcn_readfirstlane(threadIdx.x >> 6) * N * 1024;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rq, LDS_PTR(q + piece + i * 1024), 16, vq[i], 0, 0, 0);
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rg, LDS_PTR(g + piece + i * 1024), 16, vg[i], 0, 0, 0);
        }
#endif
    }
};

struct RowInfo {                     // of the 64 staged rows
    float lse[64], delta[64];        // -lse, PLAIN: -lse / (scale log2 e);  -delta (DROPPED: delta)
    int lo[64], count[64];
    float c[64], slope2[64];         // key position, from the workgroup's first key;  -slope log2 e
    float shift[64];                 // -lse - slope c log2 e
    unsigned drop[64];
};

template <int ND, int NO, int KIND>
__global__ __launch_bounds__(256, NO <= 2 || (NO == 3 && KIND == PLAIN) ? 2 : 1) void doc_dkdv_kernel(const DocArgs p, int tiles) {
    __shared__ __attribute__((aligned(16))) char even[2 * TILE_BYTES<NO>], odd[2 * TILE_BYTES<NO>];      // Q and dO, twice
    __shared__ __attribute__((aligned(16))) RowInfo infos[2];
    __shared__ int range[4][2];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l31 = lane & 31, hh = lane >> 5;
    int unit, hk;
    if (!unit_of(tiles * p.splits, p.Hkv, unit, hk)) return;
    const int split = unit / tiles, tile = unit - split * tiles;
    const int base = tile * 128, key0 = base + wave * 32, key = key0 + l31;
    bf16x8 kf[ND], vf[ND];
    const int mine = min(key, p.Tk - 1);
    const int first_key = __builtin_amdgcn_readfirstlane(mine);
    const OffWindow window = off_window(p.k_off, p.docs, p.Tk, first_key);
    load_row(kf, k_row(p, mine, hk), p.D);            // on their way while the keys' rows are looked up
    load_row(vf, v_row(p, mine, hk), p.D);
    const int2 span = key_span_in(p, mine, doc_of_wave(p.k_off, p.docs, window, first_key, __builtin_amdgcn_readlane(mine, 31), mine));
    const bool seen = key < p.Tk && span.y > span.x;
    int lo = seen ? span.x : 0x7fffffff, hi = seen ? span.y : 0;
    lo = wave_min_i(lo);
    hi = wave_max_i(hi);
    if (lane == 0) { range[wave][0] = lo; range[wave][1] = hi; }
    f32x16 dkT[NO], dvT[NO];
#pragma unroll
    for (int i = 0; i < NO; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) { dkT[i][r] = 0.f; dvT[i][r] = 0.f; }
    const Reads<ND, NO> rd;
    const Bend bend(p);
    __syncthreads();
    const int tlo = __builtin_amdgcn_readfirstlane(min(min(range[0][0], range[1][0]), min(range[2][0], range[3][0])));
    const int thi = __builtin_amdgcn_readfirstlane(max(max(range[0][1], range[1][1]), max(range[2][1], range[3][1])));
    const unsigned G = (unsigned)p.G;
    unsigned rlo = tlo < thi ? tlo * G : 0u, rhi = tlo < thi ? thi * G : 0u;
    if (p.splits > 1) {
        const unsigned n = (rhi - rlo + 63) / 64, each = (n + p.splits - 1) / p.splits;
        const unsigned from = rlo + min(n, each * split) * 64;
        rhi = min(rhi, rlo + min(n, each * (split + 1)) * 64);
        rlo = from;
    }
    const unsigned wlo = lo < hi ? lo * G : 0xffffffffu, whi = lo < hi ? hi * G : 0u;
    const int kmax = min(key0 + 32, p.Tk);       // the wave's keys: seen whole by a row with lo <= key0 and hi >= kmax
    const float rsl2 = KIND == PLAIN ? 1.f / bend.scale2 : 0.f;

    RowFetch<NO> f;
    f.init(p, 0);
    int4 ireg = {0, 0, 0, 0};
    float lreg = 0.f, dreg = 0.f, sreg = 0.f;
    unsigned hreg = 0;
    bool in = false;
    auto request = [&](char* to, unsigned r0) __attribute__((always_inline)) {
        const unsigned t0 = G == 1 ? r0 : r0 / G;
        if (64 % G != 0) f.init(p, r0 - t0 * G);
        f.dma(to, to + TILE_BYTES<NO>, p, hk, (int)t0, thi);
        if (threadIdx.x < 64) {
            const unsigned R = r0 + threadIdx.x;
            in = R < rhi;
            int token, head;
            row_of(p, in ? R : rhi - 1, hk, token, head);
            const size_t at = (size_t)head * p.Tq + token;
            ireg = p.rows[token];
            lreg = p.lse[at];
            dreg = p.delta[at];
            if (KIND != PLAIN && p.slopes) sreg = p.slopes[head];
            if (KIND == DROPPED) hreg = drop_row(p, token, head);
        }
    };
    auto note = [&](RowInfo& info) __attribute__((always_inline)) {      // what request() read of the rows, into the LDS
        if (threadIdx.x < 64) {
            const float ls = !in || lreg == -INFINITY ? INFINITY : lreg;         // rows that see nothing: probabilities of 0
            info.lse[threadIdx.x] = KIND == PLAIN ? -ls * rsl2 : -ls;
            info.delta[threadIdx.x] = KIND == DROPPED ? dreg : -dreg;
            info.lo[threadIdx.x] = ireg.x;
            info.count[threadIdx.x] = in ? ireg.y - ireg.x : 0;
            if (KIND != PLAIN) {
                const float c = (float)(ireg.z - base), slope2 = -sreg * LOG2E;
                info.c[threadIdx.x] = c;
                info.slope2[threadIdx.x] = slope2;
                info.shift[threadIdx.x] = fmaf(slope2, c, -ls);
            }
            if (KIND == DROPPED) info.drop[threadIdx.x] = hreg;
        }
    };
    auto visit = [&](const char* Qs, const RowInfo& info, unsigned r0) __attribute__((always_inline)) {
        if (r0 >= whi || r0 + 64 <= wlo) return;
        const char* Gs = Qs + TILE_BYTES<NO>;
        const int first = info.lo[lane], count = info.count[lane];
        const bool masked = __ballot(first > key0 || first + count < kmax) != 0;
        const bool before = KIND != PLAIN && __ballot(info.c[lane] < (float)(key0 + 31 - base)) == 0;
        const float keyf = (float)(key - base);
#pragma unroll
        for (int qs = 0; qs < 2; ++qs) {
            f32x16 s, dp;
            f32x4 ls[4], dl[4];
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                ls[g] = *(const f32x4*)&info.lse[qs * 32 + 8 * g + 4 * hh];
                dl[g] = *(const f32x4*)&info.delta[qs * 32 + 8 * g + 4 * hh];
            }
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                s[r] = KIND == PLAIN ? ls[r >> 2][r & 3] : 0.f;
                dp[r] = KIND == DROPPED ? 0.f : dl[r >> 2][r & 3];
            }
#pragma unroll
            for (int ks = 0; ks < ND; ++ks) {
                const bf16x8 aq = rd.frag(Qs, ks, qs), ag = rd.frag(Gs, ks, qs);
                s = mfma(aq, kf[ks], s);
                dp = mfma(ag, vf[ks], dp);
            }
            unsigned kept = 0;           // DROPPED: one bit for each register
            if constexpr (KIND == DROPPED) {
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const bool keep = drop_keep(p, info.drop[qs * 32 + reg_row(r) + 4 * hh], key);
                    kept |= keep ? 1u << r : 0u;
                    dp[r] = (keep ? dp[r] * p.drop_scale : 0.f) - dl[r >> 2][r & 3];
                }
            }
            if constexpr (KIND == PLAIN) {
#pragma unroll
                for (int r = 0; r < 16; ++r) s[r] = EXP2(s[r] * bend.scale2);
            } else {
                float gain = bend.scale2;
                if (bend.capped) {
                    bend.tanh16(s);
#pragma unroll
                    for (int r = 0; r < 16; ++r) dp[r] *= fmaf(-s[r], s[r], 1.f);
                    gain = bend.cap2;
                }
                if (!bend.biased) {
#pragma unroll
                    for (int r = 0; r < 16; ++r) s[r] = fmaf(s[r], gain, ls[r >> 2][r & 3]);
                } else if (before) {     // every key at or before every row's position: -slope (c - key) - lse = slope key + shift
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        const f32x4 shift = *(const f32x4*)&info.shift[qs * 32 + 8 * g + 4 * hh];
                        const f32x4 sl = *(const f32x4*)&info.slope2[qs * 32 + 8 * g + 4 * hh];
#pragma unroll
                        for (int e = 0; e < 4; ++e) s[4 * g + e] = fmaf(s[4 * g + e], gain, fmaf(-sl[e], keyf, shift[e]));
                    }
                } else {
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        const f32x4 c = *(const f32x4*)&info.c[qs * 32 + 8 * g + 4 * hh];
                        const f32x4 sl = *(const f32x4*)&info.slope2[qs * 32 + 8 * g + 4 * hh];
#pragma unroll
                        for (int e = 0; e < 4; ++e) s[4 * g + e] = fmaf(s[4 * g + e], gain, fmaf(sl[e], fabsf(c[e] - keyf), ls[g][e]));
                    }
                }
#pragma unroll
                for (int r = 0; r < 16; ++r) s[r] = EXP2(s[r]);
            }
#pragma unroll
            for (int r = 0; r < 16; ++r) dp[r] *= s[r];
            if (masked) {        // what a row does not see is 0, whatever its scores and gradients are
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const int4 a = *(const int4*)&info.lo[qs * 32 + 8 * g + 4 * hh], n = *(const int4*)&info.count[qs * 32 + 8 * g + 4 * hh];
                    const int lo4[4] = {a.x, a.y, a.z, a.w}, n4[4] = {n.x, n.y, n.z, n.w};
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if ((unsigned)(key - lo4[e]) >= (unsigned)n4[e]) {
                            s[4 * g + e] = 0.f;
                            dp[4 * g + e] = 0.f;
                        }
                }
            }
            bf16x8 pf[2], dsf[2];
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                pf[r >> 3][r & 7] = (bf16_t)(KIND != DROPPED ? s[r] : kept >> r & 1 ? s[r] * p.drop_scale : 0.f);
                dsf[r >> 3][r & 7] = (bf16_t)dp[r];
            }
#pragma unroll
            for (int st = 0; st < 2; ++st)
#pragma unroll
                for (int db = 0; db < NO; ++db) {
                    const bf16x8 ag = rd.frag_t(Gs, db, qs * 2 + st), aq = rd.frag_t(Qs, db, qs * 2 + st);
                    dvT[db] = mfma(ag, pf[st], dvT[db]);
                    dkT[db] = mfma(aq, dsf[st], dkT[db]);
                }
        }
    };
    if (rlo < rhi) {
        request(even, rlo);
        note(infos[0]);
    }
    keep_row(kf, seen, p.D);
    keep_row(vf, seen, p.D);
    for (unsigned r0 = rlo; r0 < rhi; r0 += 128) {
        tiles_landed();
        const bool second = r0 + 64 < rhi, more = r0 + 128 < rhi;
        if (second) request(odd, r0 + 64);
        visit(even, infos[0], r0);
        if (!second) break;
        note(infos[1]);
        tiles_landed();
        if (more) request(even, r0 + 128);
        visit(odd, infos[1], r0 + 64);
        if (more) note(infos[0]);
    }
    if (p.splits > 1) {
        if (key >= p.Tk) return;
        float* part = p.part + (((size_t)split * p.Tk + key) * p.Hkv + hk) * 2 * p.D;
#pragma unroll
        for (int db = 0; db < NO; ++db)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int d = db * 32 + 8 * g + 4 * hh;
                if (d >= p.D) continue;
                const f32x16 &a = dkT[db], &c = dvT[db];
                *(f32x4*)(part + d) = f32x4{a[4 * g], a[4 * g + 1], a[4 * g + 2], a[4 * g + 3]};
                *(f32x4*)(part + p.D + d) = f32x4{c[4 * g], c[4 * g + 1], c[4 * g + 2], c[4 * g + 3]};
            }
        return;
    }
    __syncthreads();
    put_rows<NO>(even + wave * 32 * TILE_LD<NO>, dkT, p.scale, !seen, key < p.Tk ? p.dk + (size_t)key * p.lddk + (size_t)hk * p.D : nullptr, p.D);
    put_rows<NO>(odd + wave * 32 * TILE_LD<NO>, dvT, 1.f, !seen, key < p.Tk ? p.dv + (size_t)key * p.lddv + (size_t)hk * p.D : nullptr, p.D);
    for (unsigned bad = bad_rows(seen && !(not_finite(dkT) + not_finite(dvT) == 0.f)); bad; bad &= bad - 1)
        plain_dkdv_key(p, key0 + __builtin_ctz(bad), hk);
}

// The partial gradients of a key, added in order: a wave per (key, key head).  A key that no row sees has sums of zeros, or, beside rows
// that are not finite, what plain_dkdv_key replaces by zeros.
__global__ __launch_bounds__(256) void doc_dkdv_join_kernel(const DocArgs p) {
    const int lane = threadIdx.x & 63;
    const size_t u = (size_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (u >= (size_t)p.Tk * p.Hkv) return;
    const int key = (int)(u / p.Hkv), hk = (int)(u % p.Hkv);
    const int n = 2 * p.D, at = min(lane * 4, n - 4);      // dK then dV: at most 256 values, four a lane
    const float* part = p.part + u * n + at;
    const size_t step = (size_t)p.Tk * p.Hkv * n;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    int z = 0;
    for (; z + 8 <= p.splits; z += 8) {
        f32x4 v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = *(const f32x4*)(part + (z + e) * step);
#pragma unroll
        for (int e = 0; e < 8; ++e) acc += v[e];
    }
    for (; z < p.splits; ++z) acc += *(const f32x4*)(part + z * step);
    bool bad = false;
#pragma unroll
    for (int e = 0; e < 4; ++e) bad |= !(acc[e] * 0.f == 0.f);
    if (lane * 4 < n) {
        const bool v = at >= p.D;
        bf16_t* to = v ? p.dv + (size_t)key * p.lddv + (size_t)hk * p.D + at - p.D : p.dk + (size_t)key * p.lddk + (size_t)hk * p.D + at;
        bf16x4 y;
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = (bf16_t)(v ? acc[e] : acc[e] * p.scale);
        *(bf16x4*)to = y;
    }
    if (__ballot(bad) != 0) plain_dkdv_key(p, key, hk);
}

template <int ND, int NO>
int launch(const DocArgs& a, hipStream_t st) {
    const int tiles = (int)(((long long)a.Tk + 127) / 128);
    const dim3 grid(unit_grid((long long)tiles * a.splits, a.Hkv));
    if (a.drop_thresh) hipLaunchKernelGGL((doc_dkdv_kernel<ND, NO, DROPPED>), grid, dim3(256), 0, st, a, tiles);
    else if (a.cap > 0.f || a.slopes || !(a.scale > 0.f)) hipLaunchKernelGGL((doc_dkdv_kernel<ND, NO, BENT>), grid, dim3(256), 0, st, a, tiles);
    else hipLaunchKernelGGL((doc_dkdv_kernel<ND, NO, PLAIN>), grid, dim3(256), 0, st, a, tiles);
    if (a.splits > 1) hipLaunchKernelGGL(doc_dkdv_join_kernel, dim3((unsigned)(((size_t)a.Tk * a.Hkv + 3) / 4)), dim3(256), 0, st, a);
    return mi355_check_launch("doc_attention_dkdv");
}

}  // namespace

// Workgroups without a split: one per 128 keys and key head, each passing about G * (the rows of one document, and of the others
// that its keys belong to).  Runs of at least three tiles; without a causal mask as many as are resident at once (two workgroups
// per CU: 8 x 4096 rows over 210 keys took 48 us with three times as many, 36 us with these), with one four times as many, which
// evens out that the first keys of a document are passed by all its rows and the last by few (twice as many were slower).
int doc_bwd_kv_splits(int Tq, int Tk, int Hq, int Hkv, int docs, int causal) {
    if (Tk < 1) return 1;
    const double wgs = (double)((Tk + 127) / 128) * Hkv, keys_per_doc = (double)Tk / docs;
    const double tiles = (double)Tq * (Hq / Hkv) / docs * (1.0 + 127.0 / (keys_per_doc < 1.0 ? 1.0 : keys_per_doc)) / 64.0;
    const double cap = (double)Tq * (Hq / Hkv) / 64.0;
    double s = (causal ? 2048.0 : 512.0) / wgs, most = (tiles < cap ? tiles : cap) / 3.0;
    if (s > most) s = most;
    return s < 2.0 ? 1 : s > 64.0 ? 64 : (int)s;
}

int doc_bwd_kv_tiles(const DocArgs& a, hipStream_t st) { return BY_WIDTH(a.D, launch, a, st); }
