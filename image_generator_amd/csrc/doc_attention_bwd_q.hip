// Document attention, dQ, on the matrix units: a lane owns its row as in the forward pass, S^T = K Q^T and dP^T = V dO^T give
// dS^T in the layout that dQ^T += K^T dS^T takes.  delta and the interval of a row are left for the dK / dV pass.
//
// dS is rounded to bf16 (the matrix units' type): half a step, 2^-8 of each entry at most, beside the result's own rounding, 0.24 %
// instead of 0.17 % in the 2-norm; -lse and -delta start the accumulators, in fp32.  Rows of many keys whose weight lies on a few
// (a steep distance bias: a slope of 0.5 leaves some four) also show the rounding of the result in delta, 0.16 % by itself: 0.28 %.
//
// Measured, with what bounds it: 58 255 caption tokens, 8 heads of 96 (537 MB): 147 us, 3.7 TB/s, bound by the chain of a short
// workgroup (offsets, rows, keys, three tiles, store) at two workgroups per CU.  Four documents of 4001 .. 8191 tokens, 8 heads on 2
// of 64, causal with prefix, cap and bias (223 GFLOP): 424 us, 526 TFLOP/s, bound by vector issue (80 % of the cycles: tanh, bias,
// exp2 and the conversions of a score against three products); at three waves per SIMD its registers spill, 430 us.  32768 image rows over 210 keys, 8 heads of 40: 34 us, 2.5 TB/s.
#include "doc_tiles.h"

namespace {

constexpr int FEW = 32;              // keys of a row whose delta is summed over them

template <int ND, int NO, int KIND>
__global__ __launch_bounds__(256, NO <= 2 && KIND == PLAIN ? 3 : 2) void doc_dq_kernel(const DocArgs p, int tiles) {
    // three: captions' tiles stay in place for both walks; of the widest heads they would leave one workgroup to a CU
    constexpr int BUFS = NO <= 3 && KIND == PLAIN ? 3 : 2;
    __shared__ __attribute__((aligned(16))) char ring0[2 * TILE_BYTES<NO>], ring1[2 * TILE_BYTES<NO>], ring2[BUFS == 3 ? 2 * TILE_BYTES<NO> : 16];
    __shared__ __attribute__((aligned(16))) int range[4][4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l31 = lane & 31, hh = lane >> 5;
    int unit, hk;
    if (!unit_of(tiles * p.splits_q, p.Hkv, unit, hk)) return;
    const int split = unit / tiles;
    int tile = unit - split * tiles;
    if (p.causal) tile = tiles - 1 - tile;       // the last rows of a document see most: the longest work first
    const unsigned rows = (unsigned)p.Tq * (unsigned)p.G, R = tile * 128u + wave * 32 + l31;
    const bool live = R < rows;
    int token, head;
    row_of(p, live ? R : rows - 1, hk, token, head);
    const int first = __builtin_amdgcn_readfirstlane(token);
    const OffWindow window = off_window(p.q_off, p.docs, p.Tq, first);
    const size_t at = (size_t)head * p.Tq + token;
    const float lse_at = p.lse[at], slope = p.slopes ? p.slopes[head] : 0.f;
    bf16x8 qf[ND], gf[ND];
    bf16x8 ov[ND];                               // on their way while the intervals are looked up
    load_row(gf, p.dout + (size_t)token * p.lddo + (size_t)head * p.D, p.D);
    load_row(ov, p.o + (size_t)token * p.ldo + (size_t)head * p.D, p.D);
    load_row(qf, q_row(p, token, head), p.D);
    RowSpan span = row_span_in(p, token, doc_of_wave(p.q_off, p.docs, window, first, __builtin_amdgcn_readlane(token, 31), token));
    if (live && hh == 0 && head == 0 && split == 0) p.rows[token] = make_int4(span.lo, span.hi, span.c, 0);
    if (!live) span.lo = span.hi = 0;
    const bool sees = span.hi > span.lo;
    const int lo = wave_min_i(sees ? span.lo : 0x7fffffff);
    const int hi = wave_max_i(sees ? span.hi : 0);
    const int in_lo = wave_max_i(sees ? span.lo : 0);
    const int in_hi = wave_min_i(sees ? span.hi : 0x7fffffff);
    const int c_min = wave_min_i(sees ? span.c : 0x7fffffff);
    const bool few = sees && span.hi - span.lo <= FEW;
    const int few_lo = wave_min_i(few ? span.lo : 0x7fffffff), few_hi = wave_max_i(few ? span.hi : 0);
    if (lane == 0) *(int4*)range[wave] = make_int4(lo, hi, few_lo, few_hi);
    __syncthreads();
    auto least = [&](int i) { return min(min(range[0][i], range[1][i]), min(range[2][i], range[3][i])); };
    auto most = [&](int i) { return max(max(range[0][i], range[1][i]), max(range[2][i], range[3][i])); };
    const int klo = least(0), khi = most(1), flo = least(2), fhi = most(3);
    const bf16_t *kbase = p.k + (size_t)hk * p.D, *vbase = p.v + (size_t)hk * p.D;
    Fetch<NO, 4> kf, vf;
    kf.init(p.ldk, p.D);
    vf.init(p.ldv, p.D);
    auto request = [&](char* to, int k0) __attribute__((always_inline)) {
        kf.dma(to, kbase, p.ldk, p.D, k0, khi - k0);
        vf.dma(to + TILE_BYTES<NO>, vbase, p.ldv, p.D, k0, khi - k0);
    };
    // up to BUFS tiles stay where they are; of more, all but one buffer are filled ahead
    int k_from, k_to;
    run_of(klo, khi, p.splits_q, split, k_from, k_to);
    const bool resident = p.splits_q == 1 && (klo >= khi || khi - klo <= BUFS * 64);
    auto start = [&](int from, int to) __attribute__((always_inline)) {
        if (from >= to) return;                  // (rows that see nothing leave `from` at the largest int)
        request(ring0, from);
        if ((BUFS == 3 || resident) && from + 64 < to) request(ring1, from + 64);
        if (BUFS == 3 && resident && from + 128 < to) request(ring2, from + 128);
    };
    start(k_from, k_to);
    keep_row(gf, sees, p.D);
    keep_row(ov, sees, p.D);
    float delta = 0.f;
#pragma unroll
    for (int ks = 0; ks < ND; ++ks)
#pragma unroll
        for (int e = 0; e < 8; ++e) delta = fmaf((float)ov[ks][e], (float)gf[ks][e], delta);
    delta += __shfl_xor(delta, 32, 64);
    keep_row(qf, sees, p.D);
    const float lse_raw = sees ? lse_at : -INFINITY;
    const float lse = lse_raw == -INFINITY ? INFINITY : lse_raw;      // nothing seen: probabilities of 0
    const float slope2 = slope * LOG2E;
    const unsigned drop = drop_row(p, token, head);
    const Bend bend(p);
    const float s0 = KIND == PLAIN ? -lse / bend.scale2 : 0.f;
    const Reads<ND, NO> rd;
    auto each_tile = [&](int from, int to, int wave_lo, int wave_hi, auto visit) __attribute__((always_inline)) {
        auto step = [&](const char* now, char* free, int k0) __attribute__((always_inline)) {
            if (!resident) {
                tile_landed<(BUFS - 2) * 2 * kf.N>(k0 + 64 < to);
                if (k0 + (BUFS - 1) * 64 < to) request(free, k0 + (BUFS - 1) * 64);
            }
            if (k0 < wave_hi && k0 + 64 > wave_lo) visit(now, k0);
        };
        for (int k0 = from; k0 < to; k0 += BUFS * 64) {
            step(ring0, BUFS == 3 ? ring2 : ring1, k0);
            if (k0 + 64 < to) step(ring1, ring0, k0 + 64);
            if constexpr (BUFS == 3) if (k0 + 128 < to) step(ring2, ring1, k0 + 128);
        }
    };
    // delta = sum dO o of the result as it was handed out carries its rounding, some 2^-9 of |dO| |o|.  Over many keys that is lost
    // in dP - delta; over few it is not (gradients 1.2 % off in the 2-norm with two keys, 0.25 % with 32, where the rounding of dS is
    // what counts), so rows of few keys take the sum over their keys instead, delta = sum P dP, in a walk of its own over the tiles
    // that such rows see: captions 128 -> 149 us, where the tiles are still in place, long documents nothing.
    if (resident) tiles_landed();
    if (flo < fhi) {
        float sum = 0.f;
        if (!resident) {
            tiles_landed();
            start(flo, fhi);
        }
        each_tile(resident ? klo : flo, resident ? khi : fhi, few_lo, few_hi, [&](const char* Ks, int k0) __attribute__((always_inline)) {
            const char* Vs = Ks + TILE_BYTES<NO>;
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) {
                f32x16 s, dp;
#pragma unroll
                for (int r = 0; r < 16; ++r) { s[r] = s0; dp[r] = 0.f; }
#pragma unroll
                for (int ks = 0; ks < ND; ++ks) {
                    s = mfma(rd.frag(Ks, ks, kb), qf[ks], s);
                    dp = mfma(rd.frag(Vs, ks, kb), gf[ks], dp);
                }
                const f32x16 y = KIND != PLAIN && bend.biased ? bias16(slope2, (float)(span.c - k0 - kb * 32 - 4 * hh), -lse, false) : f32x16{} - lse;
                if (KIND != PLAIN) bend.score16(s, y);
                const unsigned rel = (unsigned)(k0 + kb * 32 + 4 * hh - span.lo), len = (unsigned)(span.hi - span.lo);
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    float d = dp[r];
                    if constexpr (KIND == DROPPED) d = drop_keep(p, drop, k0 + kb * 32 + reg_row(r) + 4 * hh) ? d * p.drop_scale : 0.f;
                    const float w = EXP2(KIND == PLAIN ? s[r] * bend.scale2 : s[r]);
                    sum = rel + (unsigned)reg_row(r) < len ? fmaf(w, d, sum) : sum;
                }
            }
        });
        sum += __shfl_xor(sum, 32, 64);
        if (few) delta = sum;
        if (!resident) {
            __syncthreads();
            start(k_from, k_to);
        }
    }
    if (live && hh == 0 && split == 0) p.delta[at] = delta;
    f32x16 dqT[NO];
#pragma unroll
    for (int i = 0; i < NO; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) dqT[i][r] = 0.f;
    each_tile(k_from, k_to, lo, hi, [&](const char* Ks, int k0) __attribute__((always_inline)) {
        const char* Vs = Ks + TILE_BYTES<NO>;
        const bool masked = k0 < in_lo || k0 + 64 > in_hi;
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
            f32x16 s, dp;                 // started at -lse and -delta, which saves subtracting them
#pragma unroll
            for (int r = 0; r < 16; ++r) { s[r] = s0; dp[r] = KIND == DROPPED ? 0.f : -delta; }
#pragma unroll
            for (int ks = 0; ks < ND; ++ks) {
                s = mfma(rd.frag(Ks, ks, kb), qf[ks], s);
                dp = mfma(rd.frag(Vs, ks, kb), gf[ks], dp);
            }
            if constexpr (KIND == DROPPED) {
#pragma unroll
                for (int r = 0; r < 16; ++r) dp[r] = (drop_keep(p, drop, k0 + kb * 32 + reg_row(r) + 4 * hh) ? dp[r] * p.drop_scale : 0.f) - delta;
            }
            if constexpr (KIND == PLAIN) {
#pragma unroll
                for (int r = 0; r < 16; ++r) s[r] = EXP2(s[r] * bend.scale2) * dp[r];
            } else {
                float gain = bend.scale2;
                if (bend.capped) {
                    bend.tanh16(s);
#pragma unroll
                    for (int r = 0; r < 16; ++r) dp[r] *= fmaf(-s[r], s[r], 1.f);
                    gain = bend.cap2;
                }
                if (bend.biased) {
                    const f32x16 y = bias16(slope2, (float)(span.c - k0 - kb * 32 - 4 * hh), -lse, k0 + 63 <= c_min);
#pragma unroll
                    for (int r = 0; r < 16; ++r) s[r] = fmaf(s[r], gain, y[r]);
                } else {
#pragma unroll
                    for (int r = 0; r < 16; ++r) s[r] = fmaf(s[r], gain, -lse);
                }
#pragma unroll
                for (int r = 0; r < 16; ++r) s[r] = EXP2(s[r]) * dp[r];
            }
            bf16x8 dsf[2];
            if (masked) {
                const unsigned rel = (unsigned)(k0 + kb * 32 + 4 * hh - span.lo), len = (unsigned)(span.hi - span.lo);
#pragma unroll
                for (int r = 0; r < 16; ++r) if (rel + (unsigned)reg_row(r) >= len) s[r] = 0.f;
            }
#pragma unroll
            for (int r = 0; r < 16; ++r) dsf[r >> 3][r & 7] = (bf16_t)s[r];
#pragma unroll
            for (int st = 0; st < 2; ++st)
#pragma unroll
                for (int db = 0; db < NO; ++db) dqT[db] = mfma(rd.frag_t(Ks, db, kb * 2 + st), dsf[st], dqT[db]);
        }
    });
    if (p.splits_q > 1) {
        if (!live) return;
        float* part = p.part_q + (((size_t)split * p.Tq + token) * p.Hq + head) * p.D;
#pragma unroll
        for (int db = 0; db < NO; ++db)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int d = db * 32 + 8 * g + 4 * hh;
                if (d < p.D) *(f32x4*)(part + d) = f32x4{dqT[db][4 * g], dqT[db][4 * g + 1], dqT[db][4 * g + 2], dqT[db][4 * g + 3]};
            }
        return;
    }
    __syncthreads();
    put_rows<NO>(ring0 + wave * 32 * TILE_LD<NO>, dqT, p.scale, !sees, live ? p.dq + (size_t)token * p.lddq + (size_t)head * p.D : nullptr, p.D);
    for (unsigned bad = bad_rows(sees && !(not_finite(dqT) == 0.f)); bad; bad &= bad - 1) {
        const int t = __builtin_ctz(bad);
        const RowSpan s = {__shfl(span.lo, t, 64), __shfl(span.hi, t, 64), __shfl(span.c, t, 64)};
        plain_dq_row(p, __shfl(token, t, 64), __shfl(head, t, 64), s, __shfl(lse_raw, t, 64), __shfl(delta, t, 64));
    }
}

// the runs of a row, added in order: half a wave for a row
__global__ __launch_bounds__(256) void doc_dq_join_kernel(const DocArgs p) {
    const int lane = threadIdx.x & 63, half = lane >> 5;
    const size_t rows = (size_t)p.Tq * p.Hq, R0 = ((size_t)blockIdx.x * 4 + (threadIdx.x >> 6)) * 2;
    if (R0 >= rows) return;
    const size_t R = min(R0 + half, rows - 1);
    const int token = (int)(R / p.Hq), head = (int)(R - (size_t)token * p.Hq);
    const int4 span = p.rows[token];
    const bool sees = span.y > span.x;
    const int d = min((lane & 31) * 4, p.D - 4);
    const float* part = p.part_q + R * p.D + d;
    const size_t step = rows * p.D;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    for (int z = 0; z < p.splits_q; z += 4) {
        f32x4 v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = *(const f32x4*)(part + min(z + e, p.splits_q - 1) * step);
#pragma unroll
        for (int e = 0; e < 4; ++e) if (z + e < p.splits_q) acc += v[e];
    }
    bool bad = false;
    bf16x4 y;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        bad |= !(acc[e] * 0.f == 0.f);
        y[e] = sees ? (bf16_t)(acc[e] * p.scale) : (bf16_t)0.f;
    }
    if (R0 + half < rows && (lane & 31) * 4 < p.D) *(bf16x4*)(p.dq + (size_t)token * p.lddq + (size_t)head * p.D + d) = y;
    const unsigned long long bads = __ballot(sees && bad && R0 + half < rows);
#pragma unroll 1
    for (int h = 0; h < 2; ++h)
        if ((unsigned)(bads >> (32 * h))) {
            const int t = __shfl(token, 32 * h, 64), q = __shfl(head, 32 * h, 64);
            const RowSpan s = {__shfl(span.x, 32 * h, 64), __shfl(span.y, 32 * h, 64), __shfl(span.z, 32 * h, 64)};
            const size_t at = (size_t)q * p.Tq + t;
            plain_dq_row(p, t, q, s, p.lse[at], p.delta[at]);
        }
}

template <int ND, int NO>
int launch(const DocArgs& a, hipStream_t st) {
    const int tiles = (int)(((long long)a.Tq * a.G + 127) / 128);
    const dim3 grid(unit_grid((long long)tiles * a.splits_q, a.Hkv));
    if (a.drop_thresh) hipLaunchKernelGGL((doc_dq_kernel<ND, NO, DROPPED>), grid, dim3(256), 0, st, a, tiles);
    else if (a.cap > 0.f || a.slopes || !(a.scale > 0.f)) hipLaunchKernelGGL((doc_dq_kernel<ND, NO, BENT>), grid, dim3(256), 0, st, a, tiles);
    else hipLaunchKernelGGL((doc_dq_kernel<ND, NO, PLAIN>), grid, dim3(256), 0, st, a, tiles);
    if (a.splits_q > 1) hipLaunchKernelGGL(doc_dq_join_kernel, dim3((unsigned)(((size_t)a.Tq * a.Hq + 7) / 8)), dim3(256), 0, st, a);
    return mi355_check_launch("doc_attention_dq");
}

}  // namespace

int doc_bwd_q_tiles(const DocArgs& a, hipStream_t st) { return BY_WIDTH(a.D, launch, a, st); }
