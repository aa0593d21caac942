// Document attention, dK and dV, on the matrix units: a lane owns its key (S = Q K^T, dP = dO V^T), a wave 32 keys, a workgroup
// 128, and staged tiles of 64 rows - tokens times the query heads that share the key head - pass by: dV^T += dO^T P,
// dK^T += Q^T dS.  Nothing is added across workgroups, so there are no atomics and no order to choose.
#include "doc_tiles.h"

namespace {

template <int ND, int NO, int KIND>
__global__ __launch_bounds__(256) void doc_dkdv_kernel(const DocArgs p) {
    constexpr int LD = tr_ld(NO);
    constexpr int NCH = (64 * NO * 4 + 255) / 256;
    __shared__ __attribute__((aligned(16))) char smem[2 * 64 * LD];
    __shared__ float4 info[64];          // lse, delta, first key and number of keys of a row (as bits)
    __shared__ float2 place[64];         // its key position (as bits) and slope
    __shared__ unsigned drops[64];
    __shared__ int range[4][2];
    char *Qs = smem, *Gs = smem + 64 * LD;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l31 = lane & 31, hh = lane >> 5;
    const int hk = blockIdx.y;
    const int key = (int)blockIdx.x * 128 + wave * 32 + l31;
    const bool live = key < p.Tk;
    int2 span = live ? key_span(p, key) : make_int2(0, 0);
    const bool seen = span.y > span.x;
    const int lo = __builtin_amdgcn_readfirstlane(wave_min_i(seen ? span.x : 0x7fffffff));
    const int hi = __builtin_amdgcn_readfirstlane(wave_max_i(seen ? span.y : 0));
    if (lane == 0) { range[wave][0] = lo; range[wave][1] = hi; }
    const bf16x8 zero8 = {0, 0, 0, 0, 0, 0, 0, 0};
    bf16x8 kf[ND], vf[ND];
#pragma unroll
    for (int ks = 0; ks < ND; ++ks) {
        const int d = ks * 16 + 8 * hh;
        const bool ok = seen && d < p.D;
        kf[ks] = ok ? *(const bf16x8*)(k_row(p, key, hk) + d) : zero8;
        vf[ks] = ok ? *(const bf16x8*)(v_row(p, key, hk) + d) : zero8;
    }
    f32x16 dkT[NO], dvT[NO];
#pragma unroll
    for (int i = 0; i < NO; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) { dkT[i][r] = 0.f; dvT[i][r] = 0.f; }
    const int tr_row = 4 * hh + ((lane & 15) >> 2);
    int tr_c0, tr_c1;
    tr_cols_swz(lane, tr_c0, tr_c1);
    const Bend bend(p);
    __syncthreads();
    const int tlo = min(min(range[0][0], range[1][0]), min(range[2][0], range[3][0]));
    const int thi = max(max(range[0][1], range[1][1]), max(range[2][1], range[3][1]));
    const unsigned G = (unsigned)p.G;
    const unsigned rlo = tlo < thi ? tlo * G : 0u, rhi = tlo < thi ? thi * G : 0u;
    const unsigned wlo = lo < hi ? lo * G : 0xffffffffu, whi = lo < hi ? hi * G : 0u;
    const int kmin = (int)blockIdx.x * 128 + wave * 32;       // the wave's keys: all of them seen in full by a row with
    const int kmax = min(kmin + 32, p.Tk);                    // lo <= kmin and hi >= kmax

    bf16x8 qreg[NCH], greg[NCH];
    float4 ireg;
    float2 preg;
    unsigned dreg;
    auto load = [&](unsigned r0) {
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
            const int idx = threadIdx.x + 256 * i, r = idx / (NO * 4), c = idx % (NO * 4);
            const unsigned R = r0 + r;
            const bool ok = (64 * NO * 4 % 256 == 0 || idx < 64 * NO * 4) && R < rhi && c * 8 < p.D;
            qreg[i] = greg[i] = zero8;
            if (ok) {
                int token, head;
                row_of(p, R, hk, token, head);
                qreg[i] = *(const bf16x8*)(q_row(p, token, head) + c * 8);
                greg[i] = *(const bf16x8*)(p.dout + (size_t)token * p.lddo + (size_t)head * p.D + c * 8);
            }
        }
        if (threadIdx.x < 64) {
            const unsigned R = r0 + threadIdx.x;
            ireg = make_float4(INFINITY, 0.f, 0.f, 0.f);
            preg = make_float2(0.f, 0.f);
            dreg = 0;
            if (R < rhi) {
                int token, head;
                row_of(p, R, hk, token, head);
                const int4 s = p.rows[token];
                const size_t at = (size_t)head * p.Tq + token;
                const float ls = p.lse[at];
                ireg = make_float4(ls == -INFINITY ? INFINITY : ls, p.delta[at], __int_as_float(s.x), __int_as_float(s.y - s.x));
                preg = make_float2(__int_as_float(s.z), p.slopes ? p.slopes[head] * LOG2E : 0.f);
                dreg = drop_row(p, token, head);
            }
        }
    };
    if (rlo < rhi) load(rlo);
    for (unsigned r0 = rlo; r0 < rhi; r0 += 64) {
        __syncthreads();
        put_tile<NCH, NO * 4, true>(qreg, Qs, LD, threadIdx.x);
        put_tile<NCH, NO * 4, true>(greg, Gs, LD, threadIdx.x);
        if (threadIdx.x < 64) { info[threadIdx.x] = ireg; place[threadIdx.x] = preg; drops[threadIdx.x] = dreg; }
        __syncthreads();
        if (r0 + 64 < rhi) load(r0 + 64);
        if (r0 >= whi || r0 + 64 <= wlo) continue;
        bool masked;
        {
            const float4 f = info[lane];
            const int first = __float_as_int(f.z), count = __float_as_int(f.w);
            masked = __ballot(first > kmin || first + count < kmax) != 0;
        }
#pragma unroll
        for (int qs = 0; qs < 2; ++qs) {
            const char *Qt = Qs + qs * 32 * LD, *Gt = Gs + qs * 32 * LD;
            f32x16 s, dp;
#pragma unroll
            for (int r = 0; r < 16; ++r) { s[r] = 0.f; dp[r] = 0.f; }
#pragma unroll
            for (int ks = 0; ks < ND; ++ks) {
                const int off = l31 * LD + ((ks * 2 + hh) ^ ((l31 >> 2) & 3)) * 16;
                s = mfma(*(const bf16x8*)(Qt + off), kf[ks], s);
                dp = mfma(*(const bf16x8*)(Gt + off), vf[ks], dp);
            }
            bf16x8 pf[2], dsf[2];
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int row = qs * 32 + reg_row(r) + 4 * hh;
                const float4 f = info[row];
                float x = s[r] * bend.scale2, turn = 1.f;
                if constexpr (KIND != PLAIN) {
                    if (bend.capped) {
                        const float u = __builtin_amdgcn_rcpf(1.f + EXP2(s[r] * bend.in));
                        x = fmaf(-2.f * bend.cap2, u, bend.cap2);
                        turn = 4.f * fmaf(-u, u, u);
                    }
                    if (bend.biased) {
                        const float2 g = place[row];
                        x = fmaf(-g.y, fabsf((float)(__float_as_int(g.x) - key)), x);
                    }
                }
                float e = EXP2(x - f.x);
                if (masked && (unsigned)(key - __float_as_int(f.z)) >= (unsigned)__float_as_int(f.w)) e = 0.f;
                float pd = e, d = dp[r];
                if constexpr (KIND == DROPPED) {
                    const bool keep = drop_keep(p, drops[row], key);
                    pd = keep ? e * p.drop_scale : 0.f;
                    d = keep ? d * p.drop_scale : 0.f;
                }
                float ds = e * (d - f.y);
                if constexpr (KIND != PLAIN) ds *= turn;
                // a row that does not see the key: its dO may be anything
                if (masked && e == 0.f) ds = 0.f;
                pf[r >> 3][r & 7] = (bf16_t)pd;
                dsf[r >> 3][r & 7] = (bf16_t)ds;
            }
#pragma unroll
            for (int st = 0; st < 2; ++st)
#pragma unroll
                for (int db = 0; db < NO; ++db) {
                    const int off = (16 * st + tr_row) * LD + db * 64;
                    dvT[db] = mfma(cat4(LDS_TR(Gt + off + tr_c0), LDS_TR(Gt + off + 8 * LD + tr_c1)), pf[st], dvT[db]);
                    dkT[db] = mfma(cat4(LDS_TR(Qt + off + tr_c0), LDS_TR(Qt + off + 8 * LD + tr_c1)), dsf[st], dkT[db]);
                }
        }
    }
    if (live) {
        bf16_t *dk = p.dk + (size_t)key * p.lddk + (size_t)hk * p.D, *dv = p.dv + (size_t)key * p.lddv + (size_t)hk * p.D;
#pragma unroll
        for (int db = 0; db < NO; ++db)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int d = db * 32 + 8 * g + 4 * hh;
                if (d < p.D) {
                    bf16x4 a, c;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        a[e] = seen ? (bf16_t)(dkT[db][4 * g + e] * p.scale) : (bf16_t)0.f;
                        c[e] = seen ? (bf16_t)dvT[db][4 * g + e] : (bf16_t)0.f;
                    }
                    *(bf16x4*)(dk + d) = a;
                    *(bf16x4*)(dv + d) = c;
                }
            }
    }
    for (unsigned bad = bad_rows(seen && !(not_finite(dkT) + not_finite(dvT) == 0.f)); bad; bad &= bad - 1)
        plain_dkdv_key(p, __shfl(key, __builtin_ctz(bad), 64), hk);
}

template <int ND, int NO>
int launch(const DocArgs& a, hipStream_t st) {
    const dim3 grid((unsigned)(((long long)a.Tk + 127) / 128), a.Hkv);
    if (a.drop_thresh) hipLaunchKernelGGL((doc_dkdv_kernel<ND, NO, DROPPED>), grid, dim3(256), 0, st, a);
    else if (a.cap > 0.f || a.slopes) hipLaunchKernelGGL((doc_dkdv_kernel<ND, NO, BENT>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((doc_dkdv_kernel<ND, NO, PLAIN>), grid, dim3(256), 0, st, a);
    return mi355_check_launch("doc_attention_dkdv");
}

}  // namespace

int doc_bwd_kv_tiles(const DocArgs& a, hipStream_t st) { return BY_WIDTH(a.D, launch, a, st); }
