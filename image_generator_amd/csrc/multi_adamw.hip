// AdamW over many tensors in one launch, states in 32 or 8 bits, behind one launch for the global gradient norm.
//
//   g = c grad,  c = min(1, max_norm / (|grad| + 1e-6));   m = b1 m + (1 - b1) g;   v = b2 v + (1 - b2) g^2
//   p = p (1 - lr wd) - lr / bc1 * m / (sqrt(v) / sqrt(bc2) + eps)
//
// A tensor's elements are dealt out in blocks of 256.  States of 8 bits hold one fp32 scale s per block (the largest magnitude
// in it) and a code per element: m = s sgn(q) (q / 127)^2 and sqrt(v) = s (q / 255)^2.  The square gives small moments a finer
// step than large ones (the smallest non-zero one is 6e-5 and 1.5e-5 of the largest), and holding the ROOT of v halves the
// range that its code has to span; a root above zero keeps a code of at least 1, so no denominator falls to eps because its
// code did.  The largest magnitude of a block is held exactly, as its scale; the
// others move with it.
//
// Moments between reading and writing 8-bit codes are fp64 (vector fp64 runs at the rate of vector fp32 on this chip), so a code
// does not depend on the order in which a compiler rounds the steps before it.  States of 32 bits are stepped in fp32, by the expressions of
// the flat-buffer update, whose bits they reproduce.
#include "common.h"

namespace {

constexpr int BLK = 256;             // elements that share a scale; one wave
constexpr int WG_BLOCKS = 8;         // blocks per workgroup of four waves
constexpr int PARTS = 512;           // partial sums of the norm: two workgroups of eight waves per CU

// A code is the nearest whole number, the lower one of a tie: bf16 gradients from zero states do meet ties (a quarter of the
// largest magnitude, at 127 / 2), and the margin keeps the fp64 steps' own rounding from deciding them.
constexpr double HALF = 0.5 - 0x1p-30;

// record of a tensor: parameter (0: its gradient counts in the norm, nothing is stepped), bf16 copy (or 0), elements, first block
// in the flat moment arrays
struct Rec { long long p, p16, n, block0; };
// hyper: lr, beta1, beta2, eps, weight decay, bc1, bc2, max norm, 1 - lr wd, lr / bc1, 1 / sqrt(bc2), 1 - beta1, 1 - beta2
enum { H_LR, H_B1, H_B2, H_EPS, H_WD, H_BC1, H_BC2, H_MAX, H_DECAY, H_STEP, H_RBC2, H_OMB1, H_OMB2 };

// four gradients from element i of a tensor: fp32, or bf16 where the lowest bit of the address is set
__device__ __forceinline__ f32x4 load_grad(long long g, size_t i, size_t n) {
    f32x4 r = {0.f, 0.f, 0.f, 0.f};
    if (g & 1) {
        const bf16_t* s = (const bf16_t*)(g & ~1ll) + i;
        if (i + 4 <= n && ((uintptr_t)s & 7) == 0) {
            const bf16x4 t = __builtin_nontemporal_load((const bf16x4*)s);
            r = f32x4{(float)t[0], (float)t[1], (float)t[2], (float)t[3]};
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) if (i + e < n) r[e] = (float)s[e];
        }
    } else {
        const float* s = (const float*)g + i;
        if (i + 4 <= n && ((uintptr_t)s & 15) == 0) r = *(const f32x4*)s;
        else {
#pragma unroll
            for (int e = 0; e < 4; ++e) if (i + e < n) r[e] = s[e];
        }
    }
    return r;
}

// ---- norm: partial[b] = sum of the squares of a fixed share of the gradients, fp64, in a fixed order --------------------
// Bound by reading: 69.9 million fp32 gradients (280 MB) 91 us, 3.1 TB/s; 243 million of bf16 (485 MB) 126 us, 3.8 TB/s.  Two workgroups per
// CU with all loads of a run of eight blocks ahead of their use; more, smaller workgroups would only add partial sums that every
// workgroup of the update adds up again.
__global__ __launch_bounds__(512) void multi_sumsq_kernel(const Rec* __restrict__ recs, const long long* __restrict__ grads,
                                                           const int2* __restrict__ map, int n_wg, double* __restrict__ partial) {
    __shared__ double red[8];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    double acc = 0.0;
    const int e0 = __builtin_amdgcn_readfirstlane((int)blockIdx.x * 8 + wave);
    // addresses two entries ahead: place -> gradient -> values is a chain of three loads
    constexpr int STEP = PARTS * 8;
    int2 next = e0 < n_wg ? map[e0] : make_int2(0, 0), after = e0 + STEP < n_wg ? map[e0 + STEP] : make_int2(0, 0);
    long long g_next = e0 < n_wg ? grads[next.x] : 0, n_next = e0 < n_wg ? recs[next.x].n : 0;
    for (int e = e0; e < n_wg; e += STEP) {
        const int2 now = next;
        const long long g = g_next;
        const size_t n = (size_t)n_next, i0 = (size_t)now.y * BLK;
        next = after;
        if (e + STEP < n_wg) { g_next = grads[next.x]; n_next = recs[next.x].n; }
        if (e + 2 * STEP < n_wg) after = map[e + 2 * STEP];
        if (g == 0) continue;
        if (i0 + WG_BLOCKS * BLK <= n && (g & 15) == 0) {          // a whole run of fp32: every load issued before the first use
            const f32x4* src = (const f32x4*)g + i0 / 4 + lane;
            f32x4 v[WG_BLOCKS];
#pragma unroll
            for (int u = 0; u < WG_BLOCKS; ++u) v[u] = src[u * (BLK / 4)];
#pragma unroll
            for (int u = 0; u < WG_BLOCKS; ++u)
#pragma unroll
                for (int k = 0; k < 4; ++k) acc = fma((double)v[u][k], (double)v[u][k], acc);
        } else if (i0 + WG_BLOCKS * BLK <= n && (g & 15) == 1) {   // of bf16
            const bf16x8* src = (const bf16x8*)(g & ~1ll) + i0 / 8 + lane;
            bf16x8 v[WG_BLOCKS / 2];
#pragma unroll
            for (int u = 0; u < WG_BLOCKS / 2; ++u) v[u] = src[u * (BLK / 4)];
#pragma unroll
            for (int u = 0; u < WG_BLOCKS / 2; ++u)
#pragma unroll
                for (int k = 0; k < 8; ++k) acc = fma((double)(float)v[u][k], (double)(float)v[u][k], acc);
        } else {
            for (int u = 0; u < WG_BLOCKS; ++u) {
                const size_t i = i0 + u * BLK + lane * 4;
                if (i >= n) break;
                const f32x4 v = load_grad(g, i, n);
#pragma unroll
                for (int k = 0; k < 4; ++k) acc = fma((double)v[k], (double)v[k], acc);
            }
        }
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) acc += __shfl_xor(acc, o, 64);
    if (lane == 0) red[wave] = acc;
    __syncthreads();
    if (threadIdx.x == 0) {
        double t = 0.0;
        for (int w = 0; w < 8; ++w) t += red[w];
        partial[blockIdx.x] = t;
    }
}

// Reductions over a wave by DPP: within rows of 16 lanes, then across them; lane 63 holds the result.
template <int CTRL, int ROWS>
__device__ __forceinline__ int dpp(int old, int v) { return __builtin_amdgcn_update_dpp(old, v, CTRL, ROWS, 0xf, false); }
// the largest of whole numbers: 0, what lanes without a source get, changes none, which lets the move join the comparison
__device__ __forceinline__ unsigned wave_max_u(unsigned v) {
    v = max(v, (unsigned)dpp<0x111, 0xf>(0, (int)v));
    v = max(v, (unsigned)dpp<0x112, 0xf>(0, (int)v));
    v = max(v, (unsigned)dpp<0x114, 0xf>(0, (int)v));
    v = max(v, (unsigned)dpp<0x118, 0xf>(0, (int)v));
    v = max(v, (unsigned)dpp<0x142, 0xa>(0, (int)v));
    v = max(v, (unsigned)dpp<0x143, 0xc>(0, (int)v));
    return (unsigned)__builtin_amdgcn_readlane((int)v, 63);
}
// of values >= 0, whose bits order like whole numbers
__device__ __forceinline__ float wave_max_pos(float x) { return __uint_as_float(wave_max_u(__float_as_uint(x))); }
template <int CTRL, int ROWS>
__device__ __forceinline__ double dpp_d(double x) {               // lanes without a source get 0
    const long long b = __double_as_longlong(x);
    const unsigned lo = (unsigned)dpp<CTRL, ROWS>(0, (int)b), hi = (unsigned)dpp<CTRL, ROWS>(0, (int)(b >> 32));
    return __longlong_as_double(((long long)hi << 32) | lo);
}
__device__ __forceinline__ double lane63(double x) {
    const long long b = __double_as_longlong(x);
    const unsigned lo = (unsigned)__builtin_amdgcn_readlane((int)b, 63), hi = (unsigned)__builtin_amdgcn_readlane((int)(b >> 32), 63);
    return __longlong_as_double(((long long)hi << 32) | lo);
}
__device__ __forceinline__ double wave_max_pos(double x) {        // the same of doubles: the upper halves, then the lower ones of their lanes
    const unsigned long long b = (unsigned long long)__double_as_longlong(x);
    const unsigned hi = (unsigned)(b >> 32), top = wave_max_u(hi), low = wave_max_u(hi == top ? (unsigned)b : 0u);
    return __longlong_as_double((long long)((unsigned long long)top << 32 | low));
}
__device__ __forceinline__ double wave_sum_d(double x) {
    x += dpp_d<0x111, 0xf>(x);
    x += dpp_d<0x112, 0xf>(x);
    x += dpp_d<0x114, 0xf>(x);
    x += dpp_d<0x118, 0xf>(x);
    x += dpp_d<0x142, 0xa>(x);
    x += dpp_d<0x143, 0xc>(x);
    return lane63(x);
}

// every wave sums the partials in the same order
__device__ __forceinline__ double total_sumsq(const double* __restrict__ partial) {
    const int lane = threadIdx.x & 63;
    double t = 0.0;
#pragma unroll
    for (int k = 0; k < PARTS / 64; ++k) t += partial[k * 64 + lane];
    return wave_sum_d(t);
}

// sqrt(x) to about 2^-45, x >= 0
__device__ __forceinline__ double root(double x) {
    const double y = __builtin_amdgcn_rsq(x), h = x * y;
    const double r = fma(fma(-h, h, x), 0.5 * y, h);
    return x > 0.0 ? r : 0.0;
}
// 1 / s to about 2^-45; 0 for a scale of 0
__device__ __forceinline__ double inverse(float s) {
    const double d = (double)s, y = __builtin_amdgcn_rcp(d);
    return s > 0.f ? fma(fma(-d, y, 1.0), y, y) : 0.0;
}

__device__ __forceinline__ void store_param(const Rec& t, size_t i, f32x4 p) {
    float* d = (float*)t.p + i;
    bf16_t* d16 = (bf16_t*)t.p16 + i;
    if (i + 4 <= (size_t)t.n && ((uintptr_t)d & 15) == 0) *(f32x4*)d = p;
    else {
#pragma unroll
        for (int e = 0; e < 4; ++e) if (i + e < (size_t)t.n) d[e] = p[e];
    }
    if (t.p16) {
        if (i + 4 <= (size_t)t.n && ((uintptr_t)d16 & 7) == 0)
            *(bf16x4*)d16 = bf16x4{(bf16_t)p[0], (bf16_t)p[1], (bf16_t)p[2], (bf16_t)p[3]};
        else {
#pragma unroll
            for (int e = 0; e < 4; ++e) if (i + e < (size_t)t.n) d16[e] = (bf16_t)p[e];
        }
    }
}
__device__ __forceinline__ f32x4 load_param(const Rec& t, size_t i) {
    const float* s = (const float*)t.p + i;
    if (i + 4 <= (size_t)t.n && ((uintptr_t)s & 15) == 0) return *(const f32x4*)s;
    f32x4 r = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int e = 0; e < 4; ++e) if (i + e < (size_t)t.n) r[e] = s[e];
    return r;
}

// The norm, what it says about the step: false = skip it (state[1] counts).
__device__ __forceinline__ bool norm_of(const double* __restrict__ partial, float* __restrict__ state, double& norm) {
    const double sq = total_sumsq(partial);
    const bool fine = sq <= 3.4028234663852886e38;            // false for NaN; beyond fp32 is where the flat-buffer update skips
    norm = sqrt(sq);
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        state[0] = fine ? (float)norm : sq == sq ? INFINITY : NAN;
        if (!fine) state[1] += 1.f;
    }
    return fine;
}

// States of 32 bits.  Bound by bytes: 69.9 million parameters, 30 bytes each (2.1 GB), 369 us, 5.7 TB/s, what a copy reaches.
#pragma clang fp contract(off)
__global__ __launch_bounds__(256) void multi_adamw32_kernel(const Rec* __restrict__ recs, const long long* __restrict__ grads,
                                                            const int2* __restrict__ map, float* __restrict__ m, float* __restrict__ v,
                                                            const double* __restrict__ partial, const double* __restrict__ hyper,
                                                            float* __restrict__ state) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    double norm;
    if (!norm_of(partial, state, norm)) return;
    const int2 at = map[blockIdx.x];
    const Rec t = recs[at.x];
    const long long g = t.p ? grads[at.x] : 0;
    if (g == 0) return;
    const float lr = (float)hyper[H_LR], b1 = (float)hyper[H_B1], b2 = (float)hyper[H_B2], eps = (float)hyper[H_EPS];
    const float wd = (float)hyper[H_WD], bc1 = (float)hyper[H_BC1], bc2 = (float)hyper[H_BC2];
    float scale = 1.f;
    if (hyper[H_MAX] > 0.0) { const double c = hyper[H_MAX] / (norm + 1e-6); if (c < 1.0) scale = (float)c; }
    const float decay = fmaf(-lr, wd, 1.f), rbc2 = 1.f / sqrtf(bc2), step = lr / bc1;
    const float omb1 = (float)hyper[H_OMB1], omb2 = (float)hyper[H_OMB2];
#pragma unroll
    for (int u = 0; u < WG_BLOCKS / 4; ++u) {
        const size_t i = (size_t)(at.y + u * 4 + wave) * BLK + lane * 4;
        if (i >= (size_t)t.n) return;
        float* mp = m + (size_t)t.block0 * BLK + i;
        float* vp = v + (size_t)t.block0 * BLK + i;
        f32x4 pv = load_param(t, i), mv = *(const f32x4*)mp, vv = *(const f32x4*)vp;
        const f32x4 gv = load_grad(g, i, (size_t)t.n);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            // the roundings of the flat-buffer update, spelled out: which products fuse is otherwise the compiler's choice per kernel
            const float gg = gv[e] * scale;
            const float me = fmaf(omb1, gg, __fmul_rn(b1, mv[e]));
            const float ve = __fadd_rn(__fmul_rn(b2, vv[e]), __fmul_rn(__fmul_rn(omb2, gg), gg));
            const float denom = fmaf(sqrtf(ve), rbc2, eps);
            const float pe = fmaf(decay, pv[e], -__fmul_rn(step, me / denom));
            pv[e] = pe; mv[e] = me; vv[e] = ve;
        }
        *(f32x4*)mp = mv;
        *(f32x4*)vp = vv;
        store_param(t, i, pv);
    }
}

#pragma clang fp contract(fast)
__device__ __forceinline__ int sbyte(unsigned w, int e) { return (int)(w << (24 - 8 * e)) >> 24; }
__device__ __forceinline__ int ubyte(unsigned w, int e) { return (int)((w >> (8 * e)) & 255u); }

// States of 8 bits, 18 bytes a parameter.  A wave takes two blocks, every load of both ahead of the norm's sum; a scale needs the
// largest value of its block, hence one wave a block and DPP reductions.  69.9 million parameters (1.26 GB) 227 us, 5.6 TB/s; 243 million
// with bf16 gradients (3.9 GB) 855 us, 4.6 TB/s, at 87 % of the vector units' cycles: fp64 steps, conversions and roots, 80 instructions
// an element.
__global__ __launch_bounds__(256) void multi_adamw8_kernel(const Rec* __restrict__ recs, const long long* __restrict__ grads,
                                                           const int2* __restrict__ map, unsigned* __restrict__ m_codes,
                                                           float* __restrict__ m_scales, unsigned* __restrict__ u_codes,
                                                           float* __restrict__ u_scales, const double* __restrict__ partial,
                                                           const double* __restrict__ hyper, float* __restrict__ state) {
    constexpr int MINE = WG_BLOCKS / 4;                               // blocks of a wave, all of them on their way at once
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int2 at = map[blockIdx.x];
    const Rec t = recs[at.x];
    const long long g = t.p ? grads[at.x] : 0;
    f32x4 pvs[MINE], gvs[MINE];
    unsigned mcs[MINE], ucs[MINE];
    float mss[MINE], uss[MINE];
    // a run that lies inside the tensor, at aligned addresses: nothing to look at lane by lane
    const bool whole = (long long)(at.y + WG_BLOCKS) * BLK <= t.n && ((t.p | t.p16 * 2) & 15) == 0 && ((g & 1 ? (g & ~1ll) * 2 : g) & 15) == 0;
    if (whole && g != 0) {
#pragma unroll
        for (int u = 0; u < MINE; ++u) {
            const size_t tb = (size_t)(at.y + u * 4 + wave), i = tb * BLK + lane * 4, blk = (size_t)t.block0 + tb;
            pvs[u] = *(const f32x4*)((const float*)t.p + i);
            if (g & 1) {
                const bf16x4 v = __builtin_nontemporal_load((const bf16x4*)((const bf16_t*)(g & ~1ll) + i));
                gvs[u] = f32x4{(float)v[0], (float)v[1], (float)v[2], (float)v[3]};
            } else gvs[u] = *(const f32x4*)((const float*)g + i);
            mcs[u] = m_codes[blk * (BLK / 4) + lane];
            ucs[u] = u_codes[blk * (BLK / 4) + lane];
            mss[u] = m_scales[blk];
            uss[u] = u_scales[blk];
        }
    } else if (g != 0) {
#pragma unroll
        for (int u = 0; u < MINE; ++u) {
            const size_t tb = (size_t)(at.y + u * 4 + wave), i = tb * BLK + lane * 4;
            const size_t blk = (size_t)t.block0 + (tb * BLK < (size_t)t.n ? tb : 0);
            pvs[u] = gvs[u] = f32x4{0.f, 0.f, 0.f, 0.f};
            if (i < (size_t)t.n) { pvs[u] = load_param(t, i); gvs[u] = load_grad(g, i, (size_t)t.n); }
            mcs[u] = m_codes[blk * (BLK / 4) + lane];
            ucs[u] = u_codes[blk * (BLK / 4) + lane];
            mss[u] = m_scales[blk];
            uss[u] = u_scales[blk];
        }
    }
    // what the norm says, by one wave for the four (the sum, a root and a division in fp64 were an eighth of the instructions)
    __shared__ double said[2];
    if (wave == 0) {
        double norm, clip = 1.0;
        const bool fine = norm_of(partial, state, norm);
        if (hyper[H_MAX] > 0.0) { clip = hyper[H_MAX] / (norm + 1e-6); if (clip > 1.0) clip = 1.0; }
        if (lane == 0) { said[0] = clip; said[1] = fine ? 1.0 : 0.0; }
    }
    __syncthreads();
    if (said[1] == 0.0 || g == 0) return;
    const double c = said[0], b1 = hyper[H_B1], b2 = hyper[H_B2], omb1 = hyper[H_OMB1], omb2 = hyper[H_OMB2];
    const float eps = (float)hyper[H_EPS], decay = (float)hyper[H_DECAY], step = (float)hyper[H_STEP], rbc2 = (float)hyper[H_RBC2];
    const double omb1c = omb1 * c, omb2c = omb2 * c * c;
#pragma unroll
    for (int u = 0; u < MINE; ++u) {
        const size_t tb = (size_t)(at.y + u * 4 + wave);             // block within the tensor
        if (tb * BLK >= (size_t)t.n) return;
        const size_t i = tb * BLK + lane * 4, blk = (size_t)t.block0 + tb, w = blk * (BLK / 4) + lane;
        const bool in = i < (size_t)t.n;
        f32x4 pv = pvs[u];
        const f32x4 gv = gvs[u];
        const unsigned mc = mcs[u], uc = ucs[u];
        // m = b1 md q|q| + (1 - b1) c g;  v = b2 (ud q^2)^2 + (1 - b2) (c g)^2, with the factors of a block made once
        const double md = (double)mss[u] * (b1 / 16129.0), ud = (double)uss[u] * (1.0 / 65025.0), vd = b2 * ud * ud;
        typedef double f64x4 __attribute__((ext_vector_type(4)));
        f64x4 me, ve;
        double vmax = 0.0;
        float mf[4], mmax = 0.f;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const double gg = (double)gv[e];
            const float qm = (float)sbyte(mc, e), qu = (float)ubyte(uc, e);        // squares of codes are exact in fp32
            const double qu2 = (double)(qu * qu);
            me[e] = fma((double)(qm * fabsf(qm)), md, omb1c * gg);
            ve[e] = fma(qu2 * qu2, vd, omb2c * (gg * gg));
            mf[e] = (float)me[e];
            mmax = fmaxf(mmax, fabsf(mf[e]));
            vmax = fmax(vmax, ve[e]);
        }
        mmax = wave_max_pos(mmax);
        float umax = (float)root(wave_max_pos(vmax));
        // a scale below the normal range is held as 0, with its codes: nothing of that size moves a parameter
        mmax = mmax >= 0x1p-126f ? mmax : 0.f;
        umax = umax >= 0x1p-126f ? umax : 0.f;
        const double rm = inverse(mmax), ru = inverse(umax), ru2 = ru * ru;
        // Codes from fp32 roots, whose positions are good to 6.5e-5: a ratio rounded once, two roots of 1 ulp, a product, times 255 -
        // 255 ((2^-24 / 2 + 2^-23) / 2 + 2^-23 + 2^-24).  A lane with a position within 8e-5 of the border of two codes takes the
        // fp64 roots: one wave and block in twelve.
        constexpr float SURE = 0.5f - 8e-5f;
        f32x4 qm, qu, uf;                                            // codes as whole floats
        bool near = false;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float tm = 127.f * __builtin_amdgcn_sqrtf((float)(fabs(me[e]) * rm));
            const float ratio = __builtin_amdgcn_sqrtf((float)(ve[e] * ru2)), tu = 255.f * __builtin_amdgcn_sqrtf(ratio);
            const float fm = floorf(tm + 0.5f), fu = floorf(tu + 0.5f);
            near |= fabsf(tm - fm) > SURE || fabsf(tu - fu) > SURE;
            qm[e] = fm;
            qu[e] = fu;
            uf[e] = ratio * umax;
        }
        if (umax == 0.f) {                                           // (uniform) roots too small to be held still divide
#pragma unroll 1
            for (int e = 0; e < 4; ++e) uf[e] = (float)root(ve[e]);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) pv[e] = fmaf(pv[e], decay, -step * (mf[e] * __builtin_amdgcn_rcpf(fmaf(uf[e], rbc2, eps))));
        if (near) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                qm[e] = (float)(int)fma(127.0, root(fabs(me[e]) * rm), HALF);
                qu[e] = (float)(int)fma(255.0, root(root(ve[e] * ru2)), HALF);
            }
        }
        if (whole) {
            *(f32x4*)((float*)t.p + i) = pv;
            if (t.p16) *(bf16x4*)((bf16_t*)t.p16 + i) = bf16x4{(bf16_t)pv[0], (bf16_t)pv[1], (bf16_t)pv[2], (bf16_t)pv[3]};
        } else if (in) store_param(t, i, pv);
        unsigned mo = 0, uo = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            // (no ratio is above 1 + 2^-24, no code above 127 and 255)
            const float sq = mf[e] < 0.f ? -qm[e] : qm[e];
            mo = __builtin_amdgcn_cvt_pk_u8_f32(sq < 0.f ? sq + 256.f : sq, e, mo);
            uo = __builtin_amdgcn_cvt_pk_u8_f32(ve[e] > 0.0 && umax > 0.f ? fmaxf(qu[e], 1.f) : qu[e], e, uo);
        }
        m_codes[w] = mo;
        u_codes[w] = uo;
        if (lane == 0) { m_scales[blk] = mmax; u_scales[blk] = umax; }
    }
}

// the values that 8-bit states stand for, fp32, laid out like the codes: 69.9 million of each in 112 us, 6.3 TB/s
__global__ __launch_bounds__(256) void moments_kernel(const unsigned* __restrict__ m_codes, const float* __restrict__ m_scales,
                                                      const unsigned* __restrict__ u_codes, const float* __restrict__ u_scales,
                                                      size_t words, float* __restrict__ m, float* __restrict__ v) {
    const size_t w = (size_t)blockIdx.x * 256 + threadIdx.x;
    if (w >= words) return;
    const unsigned mc = m_codes[w], uc = u_codes[w];
    const double md = (double)m_scales[w / (BLK / 4)] * (1.0 / 16129.0), ud = (double)u_scales[w / (BLK / 4)] * (1.0 / 65025.0);
    f32x4 mo, vo;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const int qm = sbyte(mc, e), qu = ubyte(uc, e);
        const double u = (double)(qu * qu) * ud;
        mo[e] = (float)((double)(qm * abs(qm)) * md);
        vo[e] = (float)(u * u);
    }
    *(f32x4*)(m + w * 4) = mo;
    *(f32x4*)(v + w * 4) = vo;
}

static bool off16(const void* a) { return ((uintptr_t)a & 15) != 0; }

}  // namespace

extern "C" {

int mi355_multi_adamw_parts(void) { return PARTS; }

int mi355_multi_adamw_step(const long long* recs, const long long* grads, const int* map, int n_wg, int bits, void* m, float* m_scales,
                           void* v, float* u_scales, double* partial, const double* hyper, float* state, double elements, void* stream) {
    if (bits != 8 && bits != 32) return mi355_fail(MI355_ERR_ARG, "multi_adamw: states of 8 or 32 bits, not %d", bits);
    if (n_wg < 0) return mi355_fail(MI355_ERR_ARG, "multi_adamw: negative workgroup count");
    if (!partial || !hyper || !state || (n_wg > 0 && (!recs || !grads || !map || !m || !v || (bits == 8 && (!m_scales || !u_scales)))))
        return mi355_fail(MI355_ERR_ARG, "multi_adamw: null pointer");
    if (off16(m) || off16(v)) return mi355_fail(MI355_ERR_ARG, "multi_adamw: moments not 16-byte aligned");
    if (n_wg == 0) return MI355_OK;
    const hipStream_t st = (hipStream_t)stream;
    ProfScope prof(FAM_ELEM, st, elements * (bits == 8 ? 22.0 : 34.0));
    hipLaunchKernelGGL(multi_sumsq_kernel, dim3(PARTS), dim3(512), 0, st, (const Rec*)recs, grads, (const int2*)map, n_wg, partial);
    if (bits == 32)
        hipLaunchKernelGGL(multi_adamw32_kernel, dim3(n_wg), dim3(256), 0, st, (const Rec*)recs, grads, (const int2*)map, (float*)m,
                           (float*)v, partial, hyper, state);
    else
        hipLaunchKernelGGL(multi_adamw8_kernel, dim3(n_wg), dim3(256), 0, st, (const Rec*)recs, grads, (const int2*)map, (unsigned*)m,
                           m_scales, (unsigned*)v, u_scales, partial, hyper, state);
    return mi355_check_launch("multi_adamw");
}

int mi355_adamw_moments(const void* m_codes, const float* m_scales, const void* u_codes, const float* u_scales, long long blocks, float* m,
                        float* v, void* stream) {
    if (blocks < 0) return mi355_fail(MI355_ERR_ARG, "adamw_moments: negative block count");
    if (blocks == 0) return MI355_OK;
    if (!m_codes || !m_scales || !u_codes || !u_scales || !m || !v) return mi355_fail(MI355_ERR_ARG, "adamw_moments: null pointer");
    if (off16(m) || off16(v)) return mi355_fail(MI355_ERR_ARG, "adamw_moments: outputs not 16-byte aligned");
    if (blocks > (1ll << 25)) return mi355_fail(MI355_ERR_ARG, "adamw_moments: more than 2^25 blocks");
    const size_t words = (size_t)blocks * (BLK / 4);
    hipLaunchKernelGGL(moments_kernel, dim3((unsigned)((words + 255) / 256)), dim3(256), 0, (hipStream_t)stream, (const unsigned*)m_codes,
                       m_scales, (const unsigned*)u_codes, u_scales, words, m, v);
    return mi355_check_launch("adamw_moments");
}

}  // extern "C"
