// Tiles of the document attention kernels: global -> registers -> LDS, matrix fragments, score modifiers.
//
// Products are v_mfma_f32_32x32x16_bf16.  Register r of a 32 x 32 result holds row (r & 3) + 8 (r >> 2) + 4 (lane >> 5) of
// column lane & 31, which makes the registers of a transposed score tile directly the right operand of the product that
// contracts over its rows.
#pragma once
#include "doc_attention.h"

typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));

#define EXP2(x) __builtin_amdgcn_exp2f(x)
#define LDS_TR(ptr) __builtin_amdgcn_ds_read_tr16_b64_v4bf16((__attribute__((address_space(3))) bf16x4*)(ptr))
__device__ __forceinline__ bf16x8 cat4(bf16x4 a, bf16x4 b) { return bf16x8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]}; }
__device__ __forceinline__ f32x16 mfma(bf16x8 a, bf16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }

// A staged tile: 64 rows of NO * 4 chunks of 16 bytes, without padding (the LDS-DMA writes a wave's 64 chunks one behind
// another), chunk c of row r at place c ^ swz(r).  Read by rows, 16 consecutive rows at one c cover all 16 bank slots of the
// 256-byte bank row; read by ds_read_b64_tr_b16, the four rows of a 16-lane group lie in four different 64-byte blocks of it.
template <int NO>
__host__ __device__ constexpr int swz(int r) {
    return NO == 2 ? ((r >> 1) & 1) << 2 | ((r >> 2) & 1) << 1 | ((r >> 3) & 1)
         : NO == 4 ? (r & 3) << 2 | ((r >> 2) & 3) : (r >> 2) & 3;
}
template <int NO> constexpr int TILE_LD = NO * 64;
template <int NO> constexpr int TILE_BYTES = 64 * NO * 64;

// offsets of a lane's reads inside a tile
template <int ND, int NO>
struct Reads {
    int row[ND];                     // chunk of contraction step ks in row lane & 31 (rows 32 apart: + 32 * TILE_LD)
    int tr[NO][2];                   // transposing reads of column block db: rows 0 .. 7 and 8 .. 15 of a 16-row block
    __device__ __forceinline__ Reads() {
        const int lane = threadIdx.x & 63, l31 = lane & 31, hh = lane >> 5;
#pragma unroll
        for (int ks = 0; ks < ND; ++ks) row[ks] = l31 * TILE_LD<NO> + ((ks * 2 + hh) ^ swz<NO>(l31)) * 16;
        const int r = 4 * hh + ((lane & 15) >> 2), c = ((lane >> 4) & 1) * 2 + ((lane & 3) >> 1);
#pragma unroll
        for (int db = 0; db < NO; ++db)
#pragma unroll
            for (int h = 0; h < 2; ++h) tr[db][h] = (r + 8 * h) * TILE_LD<NO> + ((db * 4 + c) ^ swz<NO>(r + 8 * h)) * 16 + (lane & 1) * 8;
    }
    __device__ __forceinline__ bf16x8 frag(const char* tile, int ks, int block32) const {
        return *(const bf16x8*)(tile + row[ks] + block32 * 32 * TILE_LD<NO>);
    }
    __device__ __forceinline__ bf16x8 frag_t(const char* tile, int db, int block16) const {
        const char* t = tile + block16 * 16 * TILE_LD<NO>;
        return cat4(LDS_TR(t + tr[db][0]), LDS_TR(t + tr[db][1]));
    }
};

// A lane's row as the right operand of ND steps: 16-byte pieces at columns 16 ks + 8 (lane >> 5), zeros past D.  One tensor at a time
// and without branches: the pieces of a 128-byte line are asked for in a row, while it is in the first-level cache.  (Three tensors
// taken in turn were four times the requests to the second-level cache.)
template <int ND>
__device__ __forceinline__ void load_row(bf16x8 (&f)[ND], const bf16_t* row, int D) {
    const int hh = (threadIdx.x & 63) >> 5;
#pragma unroll
    for (int ks = 0; ks < ND; ++ks) {
        const int d = ks * 16 + 8 * hh;
        f[ks] = *(const bf16x8*)(row + (d < D ? d : 0));
    }
}
template <int ND>
__device__ __forceinline__ void keep_row(bf16x8 (&f)[ND], bool keep, int D) {
    const int hh = (threadIdx.x & 63) >> 5;
    const bf16x8 zero8 = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
    for (int ks = 0; ks < ND; ++ks) f[ks] = keep && ks * 16 + 8 * hh < D ? f[ks] : zero8;
}

// the row of a result register
__device__ __forceinline__ constexpr int reg_row(int r) { return (r & 3) + 8 * (r >> 2); }

// kinds of score
enum { PLAIN = 0, BENT = 1, DROPPED = 2 };      // scale alone; cap / bias; cap / bias / dropout

#define LDS_PTR(p) ((__attribute__((address_space(3))) void*)(p))
constexpr int NOWHERE = (int)0x80000000;        // a buffer offset that reads as zeros

// The part of a 64-row tile that one of WAVES waves brings: chunks per lane, and where they come from.  A lane's chunks are the
// same places of every tile; a tile has a descriptor of its own (a 64-bit base, made from scalars), so no row offset passes 32
// bits, and its bound turns the rows past `valid` and the columns past D into zeros.
template <int NO, int WAVES>
struct Fetch {
    static constexpr int N = NO * 4 / WAVES;
    int voff[N];
    __device__ __forceinline__ static int slot(int i) { return (((int)(threadIdx.x >> 6) % WAVES) * N + i) * 64 + (int)(threadIdx.x & 63); }
    __device__ __forceinline__ static int row_of_slot(int i) { return slot(i) / (NO * 4); }
    __device__ __forceinline__ static int col_of_slot(int i) { const int s = slot(i), r = s / (NO * 4); return (s - r * (NO * 4)) ^ swz<NO>(r); }
    __device__ __forceinline__ void init(long long ld, int D) {
#pragma unroll
        for (int i = 0; i < N; ++i) voff[i] = col_of_slot(i) * 8 < D ? (int)(row_of_slot(i) * ld + col_of_slot(i) * 8) * 2 : NOWHERE;
    }
#if defined(__HIP_DEVICE_COMPILE__)
    __device__ __forceinline__ static __amdgpu_buffer_rsrc_t rsrc(const bf16_t* base, long long ld, int D, int row0, int valid) {
        valid = min(valid, 64);
        const unsigned bytes = valid > 0 ? (unsigned)(((long long)(valid - 1) * ld + D) * 2) : 0u;
        return __builtin_amdgcn_make_buffer_rsrc((void*)(base + (size_t)row0 * ld), 0, bytes, 0x00020000);
    }
#endif
    // rows row0 .. row0 + 63 of base straight into the LDS; whoever reads them waits (tiles_landed) and meets at a barrier first
    __device__ __forceinline__ void dma(char* tile, const bf16_t* base, long long ld, int D, int row0, int valid) const {
#if defined(__HIP_DEVICE_COMPILE__)
        const __amdgpu_buffer_rsrc_t rs = rsrc(base, ld, D, row0, valid);
        char* to = tile + (int)__builtin_amdgcn_readfirstlane((threadIdx.x >> 6) % WAVES) * N * 1024;
#pragma unroll
        for (int i = 0; i < N; ++i) __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, LDS_PTR(to + i * 1024), 16, voff[i], 0, 0, 0);
#endif
    }
    // ... or by way of registers
    __device__ __forceinline__ void load(bf16x8 (&reg)[N], const bf16_t* base, long long ld, int D, int row0, int valid) const {
#if defined(__HIP_DEVICE_COMPILE__)
        const __amdgpu_buffer_rsrc_t rs = rsrc(base, ld, D, row0, valid);
#pragma unroll
        for (int i = 0; i < N; ++i) reg[i] = __builtin_bit_cast(bf16x8, __builtin_amdgcn_raw_buffer_load_b128(rs, voff[i], 0, 0));
#endif
    }
    __device__ __forceinline__ static void put(const bf16x8 (&reg)[N], char* tile) {
#pragma unroll
        for (int i = 0; i < N; ++i) *(bf16x8*)(tile + slot(i) * 16) = reg[i];
    }
};
// Every request of this wave has landed, and every wave is here.
// The buffers that take turns are LDS variables of their own, in code unrolled over them: the compiler, which keeps reads of the
// LDS behind DMA writes that may alias, then sees that they do not.  With one array and an offset it waited for the next tile's
// arrival before it read the present one (captions 434 -> 406 us, long documents 1440 -> 1333 us).
__device__ __forceinline__ void tiles_landed() {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
}

// the same for all but the last N requests, if there are any behind the one waited for
template <int N>
__device__ __forceinline__ void tile_landed(bool more) {
    if (N > 0 && more) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
    else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
}

// Reductions over a wave by DPP: within rows of 16 lanes, then across them; lane 63 holds the result.  (By way of the LDS, as
// __shfl_xor goes, the five of a tile were a chain of 3000 cycles.)
template <int CTRL, int ROWS>
__device__ __forceinline__ int dpp(int none, int v) { return __builtin_amdgcn_update_dpp(none, v, CTRL, ROWS, 0xf, false); }   // `none`: lanes without a source
__device__ __forceinline__ int wave_min_i(int v) {
    constexpr int N = 0x7fffffff;
    v = min(v, dpp<0x111, 0xf>(N, v)); v = min(v, dpp<0x112, 0xf>(N, v)); v = min(v, dpp<0x114, 0xf>(N, v)); v = min(v, dpp<0x118, 0xf>(N, v));
    v = min(v, dpp<0x142, 0xa>(N, v)); v = min(v, dpp<0x143, 0xc>(N, v));
    return __builtin_amdgcn_readlane(v, 63);
}
__device__ __forceinline__ int wave_max_i(int v) {
    constexpr int N = (int)0x80000000;
    v = max(v, dpp<0x111, 0xf>(N, v)); v = max(v, dpp<0x112, 0xf>(N, v)); v = max(v, dpp<0x114, 0xf>(N, v)); v = max(v, dpp<0x118, 0xf>(N, v));
    v = max(v, dpp<0x142, 0xa>(N, v)); v = max(v, dpp<0x143, 0xc>(N, v));
    return __builtin_amdgcn_readlane(v, 63);
}

// q.k -> score in log2 units (cap and bias decided at run time, uniformly).
//
// The cap's tanh costs an exponential and a reciprocal beside a probability's own exponential, and what bounds these kernels
// is vector issue.  Scores are mostly small against their cap, and for |z| <= 0.625 tanh z = z P(z^2) with P of degree 4
// (fitted to the largest error of z P on that range: 8e-8, less than the 2.4e-7 of the other form): in s = q.k, with the
// scale folded into the coefficients, five multiply-adds and two products.  A block of scores that are all that small - one
// wave-uniform test of its largest magnitude - uses it.
struct Bend {
    float scale2, cap2;              // scale log2 e;  cap log2 e
    float in, small;                 // 2 scale log2 e / cap;  |s| below which |z| <= 0.625
    float c0, c1, c2, c3, c4;        // tanh(s scale / cap) = s (c0 + c1 s^2 + ...)
    bool capped, biased;
    __device__ __forceinline__ Bend(const DocArgs& p)
        : scale2(p.scale * LOG2E), cap2(p.cap * LOG2E), in(p.scale * (2.f * LOG2E) * p.rcap), small(0.625f * p.cap / fabsf(p.scale)),
          capped(p.cap > 0.f), biased(p.slopes != nullptr) {
        const float z = p.scale * p.rcap, zz = z * z;
        c0 = z * 0.999999463558197f;
        c1 = z * zz * -0.33330482244491577f;
        c2 = z * zz * zz * 0.13291031122207642f;
        c3 = z * zz * zz * zz * -0.051362864673137665f;
        c4 = z * zz * zz * zz * zz * 0.014530063606798649f;
    }
    __device__ __forceinline__ bool all_small(const f32x16& s) const {
        float top = fabsf(s[0]);
#pragma unroll
        for (int r = 1; r < 16; ++r) top = fmaxf(top, fabsf(s[r]));
        return __ballot(!(top <= small)) == 0;
    }
    __device__ __forceinline__ float poly(float s) const {           // tanh(s scale / cap) / s
        const float w = s * s;
        return fmaf(w, fmaf(w, fmaf(w, fmaf(w, c4, c3), c2), c1), c0);
    }
    __device__ __forceinline__ float any(float s) const { return fmaf(-2.f, __builtin_amdgcn_rcpf(1.f + EXP2(s * in)), 1.f); }
    // s -> tanh(s scale / cap)
    __device__ __forceinline__ void tanh16(f32x16& s) const {
        if (all_small(s)) {
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] *= poly(s[r]);
        } else {
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] = any(s[r]);
        }
    }
    // s -> score + y, in log2 units
    __device__ __forceinline__ void score16(f32x16& s, const f32x16& y) const {
        if (!capped) {
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] = fmaf(s[r], scale2, y[r]);
            return;
        }
        tanh16(s);
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = fmaf(s[r], cap2, y[r]);
    }
};
// -slope |c - key| + rest over the registers of a block whose first key lies cf keys before c.  `before`: every key is at or
// before c, which leaves one multiply-add for each.
__device__ __forceinline__ f32x16 bias16(float slope2, float cf, float rest, bool before) {
    f32x16 y;
    if (before) {
        const float first = fmaf(-slope2, cf, rest);
#pragma unroll
        for (int r = 0; r < 16; ++r) y[r] = fmaf(slope2, (float)reg_row(r), first);
    } else {
#pragma unroll
        for (int r = 0; r < 16; ++r) y[r] = fmaf(-slope2, fabsf(cf - (float)reg_row(r)), rest);
    }
    return y;
}

// A wave's 32 rows of a result, a lane its row, out by way of the LDS (`own`: 32 * TILE_LD bytes of this wave's, that nobody
// reads any more): 16-byte pieces, a row's side by side.  Straight from the registers a store would touch 16 bytes in each of
// 32 rows, eight times the requests.  `to`: where the lane's row goes, nullptr: nowhere; `zero`: as zeros.
template <int NO>
__device__ __forceinline__ void put_rows(char* own, const f32x16 (&a)[NO], float scale, bool zero, bf16_t* to, int D) {
    const int lane = threadIdx.x & 63, l31 = lane & 31, hh = lane >> 5;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
    for (int db = 0; db < NO; ++db)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            bf16x4 v;
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = zero ? (bf16_t)0.f : (bf16_t)(a[db][4 * g + e] * scale);
            *(bf16x4*)(own + l31 * TILE_LD<NO> + ((db * 4 + g) ^ swz<NO>(l31)) * 16 + hh * 8) = v;
        }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");       // one wave: its LDS operations complete in order
    const unsigned lo = (unsigned)(uintptr_t)to, hi = (unsigned)((uintptr_t)to >> 32);
#pragma unroll
    for (int i = 0; i < 2 * NO; ++i) {
        const int s = i * 64 + lane, r = s / (NO * 4), c = s - r * (NO * 4);
        const bf16x8 v = *(const bf16x8*)(own + r * TILE_LD<NO> + (c ^ swz<NO>(r)) * 16);
        bf16_t* row = (bf16_t*)((uintptr_t)(unsigned)__shfl((int)hi, r, 64) << 32 | (unsigned)__shfl((int)lo, r, 64));
        if (row && c * 8 < D) *(bf16x8*)(row + c * 8) = v;
    }
}

// NaN if any register is not finite, else 0
template <int NO>
__device__ __forceinline__ float not_finite(const f32x16 (&a)[NO]) {
    float z = 0.f;
#pragma unroll
    for (int i = 0; i < NO; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) z = fmaf(a[i][r], 0.f, z);
    return z;
}

// rows of the wave (as bits) of which a lane says `bad`
__device__ __forceinline__ unsigned bad_rows(bool bad) {
    const unsigned long long b = __ballot(bad);
    return (unsigned)b | (unsigned)(b >> 32);
}

// row R of a key head -> token and query head
__device__ __forceinline__ void row_of(const DocArgs& p, unsigned R, int hk, int& token, int& head) {
    if (p.G == 1) { token = (int)R; head = hk; return; }
    const unsigned t = R / (unsigned)p.G;
    token = (int)t;
    head = hk * p.G + (int)(R - t * (unsigned)p.G);
}

// Workgroup -> (unit, key head), a unit being a tile (and one of its runs).  Ids go to the 8 XCDs in turn: the heads of a unit
// follow each other on one XCD, so the lines and pages that neighbouring heads share (a head's columns are a piece of each
// row) are fetched once, and neighbouring tiles, whose work grows alike along a causal document, spread over all XCDs.
// Fewer units than fill the XCDs evenly: heads spread too.
__device__ __forceinline__ bool unit_of(int units, int heads, int& unit, int& head) {
    if (units < 64) {
        unit = (int)blockIdx.x / heads;
        head = (int)blockIdx.x - unit * heads;
        return true;
    }
    const int slot = (int)(blockIdx.x >> 3), group = slot / heads;
    head = slot - group * heads;
    unit = group * 8 + (int)(blockIdx.x & 7);
    return unit < units;
}
inline unsigned unit_grid(long long units, int heads) { return (unsigned)(units < 64 ? units * heads : (units + 7) / 8 * 8 * heads); }

int doc_fwd_tiles(const DocArgs& a, hipStream_t st);
int doc_bwd_q_tiles(const DocArgs& a, hipStream_t st);
int doc_bwd_kv_tiles(const DocArgs& a, hipStream_t st);
int doc_bwd_kv_splits(int Tq, int Tk, int Hq, int Hkv, int docs, int causal);
size_t doc_fwd_workspace(int Tq, int Tk, int Hq, int Hkv, int D, int docs);

// Runs of keys for each tile of 128 rows, where the tiles alone leave much of the chip idle (few heads, few long documents): as many as
// make 768 workgroups, three to a CU, each run of at least RUN_TILES tiles (some 5 us, what a second launch that adds the runs up
// costs); 1: none.  Three documents of up to 5012 tokens, 2 heads of 24, forward and backward: 317 us without, 189 with.
constexpr int RUN_TILES = 3;
inline int key_runs(int Tq, int Tk, int Hq, int Hkv, int docs) {
    const long long wgs = ((long long)Tq * (Hq / Hkv) + 127) / 128 * Hkv;
    long long s = wgs >= 384 || wgs == 0 ? 1 : 768 / wgs;
    const long long most = (long long)Tk / docs / (64 * RUN_TILES);
    if (s > most) s = most;
    return s < 2 ? 1 : s > 32 ? 32 : (int)s;
}
// the run `split` of [lo, hi), cut at whole tiles
__device__ __forceinline__ void run_of(int lo, int hi, int splits, int split, int& from, int& to) {
    from = lo;
    to = hi;
    if (splits > 1 && lo < hi) {
        const int n = (hi - lo + 63) / 64, each = (n + splits - 1) / splits;
        from = lo + min(n, each * split) * 64;
        to = min(hi, lo + min(n, each * (split + 1)) * 64);
    }
}

// FN<ND, NO>(args...) for the head width: ND 16-wide steps of a contraction over it, NO 32-wide blocks of it
#define BY_WIDTH(D, FN, ...)                              \
    ((D) <= 32 ? FN<2, 1>(__VA_ARGS__) : (D) <= 48 ? FN<3, 2>(__VA_ARGS__) : (D) <= 64 ? FN<4, 2>(__VA_ARGS__) \
     : (D) <= 80 ? FN<5, 3>(__VA_ARGS__) : (D) <= 96 ? FN<6, 3>(__VA_ARGS__) : FN<8, 4>(__VA_ARGS__))
