// Embedding rows and the gradient of their table.
//
//   out[i][:]    = scale * table[id_i][:]
//   dtable[v][:] = scale * sum over i with id_i = v of dy[i][:]
//
// The gradient groups the positions by id with a stable sort instead of adding with atomics, so every row of the table is
// written once, by one wave, in an order that depends on the ids alone: the same call returns the same bits.  Sums are fp32,
// rounded once if the table is bf16.  An id outside [0, rows) reads as a NaN row and contributes to no gradient (ids live on
// the device; nothing here waits for the host).
#include "common.h"

namespace {

constexpr int RANKED = 8192;         // ids sorted by counting, for each, those below it
constexpr int SHARES = 16;           // lanes that count for one id
constexpr int TILE = 2048;           // ids per workgroup of a radix pass: four waves with 512 consecutive ids each
constexpr int MAXBINS = 256;
constexpr int CHUNK = 32;            // sorted positions of one id that are summed ahead when they fill an aligned chunk ...
constexpr int SUPER = 32;            // ... and aligned runs of so many such chunks,
constexpr int SUPERS_FROM = 4096;    // from so many positions on

template <typename T> __device__ __forceinline__ float ldf(const T* p) { return (float)*p; }
template <typename T> struct Vec4;
template <> struct Vec4<float> { typedef f32x4 t; };
template <> struct Vec4<bf16_t> { typedef bf16x4 t; };
template <typename T, int VEC> struct Raw { typedef typename Vec4<T>::t t; };
template <typename T> struct Raw<T, 1> { typedef T t; };
template <typename T> __device__ __forceinline__ f32x4 ld4(const T* p) {
    const typename Vec4<T>::t v = *(const typename Vec4<T>::t*)p;
    return f32x4{(float)v[0], (float)v[1], (float)v[2], (float)v[3]};
}
template <typename T> __device__ __forceinline__ void st4(T* p, f32x4 v) {
    typename Vec4<T>::t o;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = (T)v[e];
    *(typename Vec4<T>::t*)p = o;
}

__device__ __forceinline__ long long load_id(const void* ids, int ids64, size_t i) {
    return ids64 ? ((const long long*)ids)[i] : (long long)((const int*)ids)[i];
}

// ---- rows -------------------------------------------------------------------------------------------------------
// One thread per 8 (or, for odd widths and unaligned tensors, 1) elements of the output.  Bound by moving bytes: 262143 rows of
// 768 bf16 out of an fp32 table of 16384 rows are 805 MB read - 50 MB of them distinct, the rest from the last-level cache -
// and 403 MB written, 129 us, 9.4 TB/s (four pieces per thread with their loads together: the same 129 us).
// An output beyond half of the 256 MB last-level cache is stored past it (PAST): whoever reads it next finds its beginning
// evicted anyway, and what the caches hold survives (that call with the gradient behind it 316 -> 290 us; at 2.5 MB there is
// nothing to win, 31 us either way).
template <typename TI, typename TO, int VEC, bool PAST>
__global__ __launch_bounds__(256) void embed_rows_kernel(const void* __restrict__ ids, int ids64, const TI* __restrict__ table,
                                                         TO* __restrict__ out, unsigned total, unsigned per_row, long long rows,
                                                         int width, float scale) {
    const unsigned idx = blockIdx.x * 256u + threadIdx.x;
    if (idx >= total) return;
    const unsigned row = idx / per_row, c = (idx - row * per_row) * VEC;
    const long long id = load_id(ids, ids64, row);
    const bool ok = id >= 0 && id < rows;
    const TI* src = table + (size_t)(ok ? id : 0) * width + c;
    TO* dst = out + (size_t)row * width + c;
    if constexpr (VEC == 8) {
        const float f = ok ? scale : NAN;
        f32x4 a = ld4(src), b = ld4(src + 4);
        a = ok ? a * f : f32x4{NAN, NAN, NAN, NAN};
        b = ok ? b * f : f32x4{NAN, NAN, NAN, NAN};
        if constexpr (sizeof(TO) == 2) {
            const bf16x8 r = {(bf16_t)a[0], (bf16_t)a[1], (bf16_t)a[2], (bf16_t)a[3], (bf16_t)b[0], (bf16_t)b[1], (bf16_t)b[2], (bf16_t)b[3]};
            if constexpr (PAST) __builtin_nontemporal_store(r, (bf16x8*)dst);
            else *(bf16x8*)dst = r;
        }
        else if constexpr (PAST) {
            __builtin_nontemporal_store(a, (f32x4*)dst);
            __builtin_nontemporal_store(b, (f32x4*)(dst + 4));
        } else { st4(dst, a); st4(dst + 4, b); }
    } else {
        *dst = ok ? (TO)(ldf(src) * scale) : (TO)NAN;
    }
}

// ---- sort: up to RANKED ids ---------------------------------------------------------------------------------------
// The place of an id in the sorted list is the number of (id, position) pairs below its own: ids up to its own in front of it,
// ids below it behind.  That is n^2 comparisons, but spread over the chip (16 lanes for each id, every workgroup with the whole
// list in LDS, four ids a read) they beat the passes below, whose six launches wait for each other: 17.6 against 32 us of
// kernels at 8192 ids, 5.2 us at 2048 (two trips to memory and a launch).
__global__ __launch_bounds__(256) void rank_sort_kernel(const void* __restrict__ ids, int ids64, int n, unsigned rows,
                                                        unsigned* __restrict__ keys, unsigned* __restrict__ pos) {
    extern __shared__ __attribute__((aligned(16))) unsigned list[];
    const int padded = (n + 4 * SHARES - 1) / (4 * SHARES) * (4 * SHARES);       // (the padding is above every id)
    for (int i0 = threadIdx.x; i0 < padded; i0 += 8 * 256) {
        long long id[8];                         // eight loads under way at a time
#pragma unroll
        for (int u = 0; u < 8; ++u) id[u] = load_id(ids, ids64, min(i0 + u * 256, n - 1));
#pragma unroll
        for (int u = 0; u < 8; ++u)
            if (i0 + u * 256 < padded) list[i0 + u * 256] = i0 + u * 256 >= n ? 0xffffffffu : id[u] >= 0 && id[u] < (long long)rows ? (unsigned)id[u] : rows;
    }
    __syncthreads();
    const int mine = blockIdx.x * (256 / SHARES) + threadIdx.x / SHARES, share = threadIdx.x % SHARES;
    if (mine >= n) return;                       // whole groups of SHARES lanes
    const unsigned key = list[mine];
    int below = 0;
#pragma unroll 4
    for (int j = share * 4; j < padded; j += 4 * SHARES) {
        typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
        const u32x4 x = *(const u32x4*)&list[j];
#pragma unroll
        for (int e = 0; e < 4; ++e) below += x[e] < key + (j + e < mine ? 1u : 0u) ? 1 : 0;
    }
#pragma unroll
    for (int o = 1; o < SHARES; o <<= 1) below += __shfl_xor(below, o, 64);
    if (share == 0) { keys[below] = key; pos[below] = mine; }
}

// ---- sort: any number of ids, least significant digit first ---------------------------------------------------------
// Bits of a pass: as even as at most 8 a pass allow.  Each is three launches - digits of a tile counted, prefix sums over the tiles,
// entries moved to their places, in order within a tile by ballots over the waves' digits - bound by their chains, not by bytes:
// 262143 ids of 16384 rows, two passes: 45 us, of it 10 us each move.  No atomic decides an order.
// FIRST: the input is the id list itself (position = index); else (keys, pos) of the previous pass.
template <bool FIRST>
__device__ __forceinline__ unsigned pass_key(const void* ids, int ids64, const unsigned* keys, size_t i, unsigned rows) {
    if (!FIRST) return keys[i];
    const long long id = load_id(ids, ids64, i);
    return id >= 0 && id < (long long)rows ? (unsigned)id : rows;
}

template <bool FIRST>
__global__ __launch_bounds__(256) void radix_count_kernel(const void* __restrict__ ids, int ids64, const unsigned* __restrict__ keys,
                                                          int n, unsigned rows, int shift, unsigned mask, int tiles,
                                                          unsigned* __restrict__ counts) {
    __shared__ unsigned hist[MAXBINS];
    hist[threadIdx.x] = 0;
    __syncthreads();
    const int base = blockIdx.x * TILE;
#pragma unroll
    for (int u = 0; u < TILE / 256; ++u) {
        const int i = base + u * 256 + threadIdx.x;
        if (i < n) atomicAdd(&hist[(pass_key<FIRST>(ids, ids64, keys, i, rows) >> shift) & mask], 1u);
    }
    __syncthreads();
    if (threadIdx.x <= mask) counts[(size_t)threadIdx.x * tiles + blockIdx.x] = hist[threadIdx.x];
}

// counts[bin][tile] -> exclusive prefix sums along the tiles, and the bin's total: a wave per bin.
__global__ __launch_bounds__(256) void scan_kernel(unsigned* __restrict__ counts, unsigned* __restrict__ totals, int bins, int tiles) {
    const int lane = threadIdx.x & 63, bin = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (bin >= bins) return;
    unsigned* row = counts + (size_t)bin * tiles;
    unsigned carry = 0;
    for (int base = 0; base < tiles; base += 64) {
        const int i = base + lane;
        const unsigned v = i < tiles ? row[i] : 0u;
        unsigned inc = v;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const unsigned t = __shfl_up(inc, o, 64);
            if (lane >= o) inc += t;
        }
        if (i < tiles) row[i] = carry + inc - v;
        carry += __shfl(inc, 63, 64);
    }
    if (lane == 0) totals[bin] = carry;
}

template <bool FIRST>
__global__ __launch_bounds__(256) void radix_scatter_kernel(const void* __restrict__ ids, int ids64, const unsigned* __restrict__ keys,
                                                            const unsigned* __restrict__ pos, int n, unsigned rows, int shift, int bits,
                                                            int tiles, const unsigned* __restrict__ starts,
                                                            const unsigned* __restrict__ totals,
                                                            unsigned* __restrict__ keys_out, unsigned* __restrict__ pos_out) {
    constexpr int ROUNDS = TILE / 256;
    __shared__ unsigned cnt[4][MAXBINS];
    __shared__ unsigned wsum[4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const unsigned mask = (1u << bits) - 1;
#pragma unroll
    for (int w = 0; w < 4; ++w) cnt[w][threadIdx.x] = 0;
    __syncthreads();
    const int base = blockIdx.x * TILE + wave * (TILE / 4);
    unsigned key[ROUNDS], rank[ROUNDS];
#pragma unroll
    for (int u = 0; u < ROUNDS; ++u) {
        const int i = base + u * 64 + lane;
        const bool in = i < n;
        key[u] = in ? pass_key<FIRST>(ids, ids64, keys, i, rows) : 0u;
        const unsigned d = (key[u] >> shift) & mask;
        unsigned long long same = __ballot(in);              // lanes of this step that hold the same digit
        for (int b = 0; b < bits; ++b) {
            const unsigned long long has = __ballot((d >> b) & 1);
            same &= (d >> b) & 1 ? has : ~has;
        }
        const unsigned long long below = same & ((1ull << lane) - 1);
        const unsigned old = in ? cnt[wave][d] : 0u;
        rank[u] = old + __popcll(below);
        __builtin_amdgcn_wave_barrier();
        if (in && below == 0) cnt[wave][d] = old + __popcll(same);
        __builtin_amdgcn_wave_barrier();
    }
    __syncthreads();
    {   // counts of the four waves -> where each wave's first entry of a digit goes
        const unsigned d = threadIdx.x, total = d <= mask ? totals[d] : 0u;
        unsigned inc = total;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const unsigned t = __shfl_up(inc, o, 64);
            if (lane >= o) inc += t;
        }
        if (lane == 63) wsum[wave] = inc;
        __syncthreads();
        unsigned at = inc - total + (d <= mask ? starts[(size_t)d * tiles + blockIdx.x] : 0u);
#pragma unroll
        for (int w = 0; w < 4; ++w) if (w < wave) at += wsum[w];
#pragma unroll
        for (int w = 0; w < 4; ++w) { const unsigned c = cnt[w][d]; cnt[w][d] = at; at += c; }
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < ROUNDS; ++u) {
        const int i = base + u * 64 + lane;
        if (i < n) {
            const unsigned at = cnt[wave][(key[u] >> shift) & mask] + rank[u];
            keys_out[at] = key[u];
            pos_out[at] = FIRST ? (unsigned)i : pos[i];
        }
    }
}

// ---- sums -----------------------------------------------------------------------------------------------------------
// Adds `count` rows src[idx(j)][col0 ..] to acc in order: a wave, VEC columns per lane and sweep, up to FLY rows in flight.  A
// batch issues all its loads (lanes past the row's end repeat its last columns, what they add up is not stored): a load
// behind a condition is waited for on the spot.
constexpr int SWEEPS = 3;            // of 64 * VEC columns
template <int FLY, int VEC, typename T>
__device__ __forceinline__ void add_batch(f32x4 (&acc)[SWEEPS], const T* __restrict__ src, int width, const int (&col)[SWEEPS], int sweeps,
                                          unsigned mine, int j) {
    const T* r[FLY];
#pragma unroll
    for (int e = 0; e < FLY; ++e) r[e] = src + (size_t)(unsigned)__builtin_amdgcn_readlane((int)mine, j + e) * width;
    typename Raw<T, VEC>::t v[FLY][SWEEPS];
#pragma unroll
    for (int s = 0; s < SWEEPS; ++s)
        if (s < sweeps) {
#pragma unroll
            for (int e = 0; e < FLY; ++e) v[e][s] = *(const typename Raw<T, VEC>::t*)(r[e] + col[s]);
        }
#pragma unroll
    for (int s = 0; s < SWEEPS; ++s)
        if (s < sweeps) {
#pragma unroll
            for (int e = 0; e < FLY; ++e) {
                if constexpr (VEC == 4) acc[s] = acc[s] + f32x4{(float)v[e][s][0], (float)v[e][s][1], (float)v[e][s][2], (float)v[e][s][3]};
                else acc[s][0] += (float)v[e][s];
            }
        }
}
template <int VEC, typename T, typename IDX>
__device__ __forceinline__ void add_rows(f32x4 (&acc)[SWEEPS], const T* __restrict__ src, int width, int col0, int count, IDX idx) {
    const int lane = threadIdx.x & 63;
    int col[SWEEPS];
#pragma unroll
    for (int s = 0; s < SWEEPS; ++s) col[s] = min(col0 + (s * 64 + lane) * VEC, width - VEC);
    const int sweeps = min(SWEEPS, (width - col0 + 64 * VEC - 1) / (64 * VEC));
    for (int b = 0; b < count; b += 64) {
        const int n = min(64, count - b);
        const unsigned mine = idx(b + min(lane, n - 1));
        int j = 0;
        constexpr int FLY = 16;
        for (; j + FLY <= n; j += FLY) add_batch<FLY, VEC>(acc, src, width, col, sweeps, mine, j);
        if (FLY == 16 && (n & 8)) { add_batch<8, VEC>(acc, src, width, col, sweeps, mine, j); j += 8; }
        if (n & 4) { add_batch<4, VEC>(acc, src, width, col, sweeps, mine, j); j += 4; }
        if (n & 2) { add_batch<2, VEC>(acc, src, width, col, sweeps, mine, j); j += 2; }
        if (n & 1) add_batch<1, VEC>(acc, src, width, col, sweeps, mine, j);
    }
}
template <int VEC, typename T>
__device__ __forceinline__ void put_row(T* __restrict__ dst, const f32x4 (&acc)[SWEEPS], int width, int col0, float scale) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int s = 0; s < SWEEPS; ++s) {
        const int c = col0 + s * 64 * VEC + lane * VEC;
        if (c < width) {
            if constexpr (VEC == 4) st4(dst + c, acc[s] * scale);
            else dst[c] = (T)(acc[s][0] * scale);
        }
    }
}

// Ids that make up much of a batch would leave one wave with most of the work, so aligned chunks whose CHUNK positions all belong
// to one id are summed ahead, by a wave each (blockIdx.y: SWEEPS * 64 * VEC columns), wherever they lie.  Bound by reading rows:
// 262143 of 768 bf16, 57 us, most of 403 MB, 16 rows of a wave under way at a time (8 were slower, at twice the occupancy too).
template <typename T, int VEC>
__global__ __launch_bounds__(256) void chunk_sum_kernel(const unsigned* __restrict__ keys, const unsigned* __restrict__ pos, int n,
                                                        unsigned rows, const T* __restrict__ dy, int width, float* __restrict__ part) {
    const int c = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6));
    const int lo = c * CHUNK;
    if (lo + CHUNK > n) return;
    const unsigned k = keys[lo], last = keys[lo + CHUNK - 1], mine = pos[lo + (threadIdx.x & (CHUNK - 1))];
    if (k >= rows || last != k) return;
    const int col0 = blockIdx.y * SWEEPS * 64 * VEC;
    f32x4 acc[SWEEPS] = {};
    add_rows<VEC>(acc, dy, width, col0, CHUNK, [&](int) { return mine; });       // (CHUNK <= 64: lane j asks for j)
    put_row<VEC>(part + (size_t)c * width, acc, width, col0, 1.f);
}
// ... and aligned runs of SUPER such chunks.
template <int VEC>
__global__ __launch_bounds__(64) void super_sum_kernel(const unsigned* __restrict__ keys, int n, unsigned rows, int width,
                                                       const float* __restrict__ part, float* __restrict__ part2) {
    const int lo = blockIdx.x * (CHUNK * SUPER);
    if (lo + CHUNK * SUPER > n) return;
    const unsigned k = keys[lo];
    if (k >= rows || keys[lo + CHUNK * SUPER - 1] != k) return;
    const int col0 = blockIdx.y * SWEEPS * 64 * VEC, c0 = blockIdx.x * SUPER;
    f32x4 acc[SWEEPS] = {};
    add_rows<VEC>(acc, part, width, col0, SUPER, [&](int j) { return (unsigned)(c0 + j); });
    put_row<VEC>(part2 + (size_t)blockIdx.x * width, acc, width, col0, 1.f);
}

// Every row of the table, written once: a wave takes the sorted positions of its id (found by binary search) in order, whole
// aligned chunks and runs of chunks from their sums; an id without positions gets zeros.  Bound by the chain of search, positions,
// rows and store: 16384 x 768 fp32 (50 MB) of 1601 ids 15.5 us, of 262143 ids 63 us with the rows that no chunk holds.
constexpr int ROWS_PER_WG = 7;       // eight boundaries: two for each of four waves
template <typename T, typename TO, int VEC>
__global__ __launch_bounds__(256) void table_grad_kernel(const unsigned* __restrict__ keys, const unsigned* __restrict__ pos, int n,
                                                         unsigned rows, const T* __restrict__ dy, int width, float scale,
                                                         const float* __restrict__ part, const float* __restrict__ part2,
                                                         TO* __restrict__ dtable) {
    __shared__ int start[ROWS_PER_WG + 1];
    const unsigned v0 = blockIdx.x * ROWS_PER_WG;
    // first index with keys[index] >= v, for each v of the workgroup: a wave takes two v and probes 64 places a step for each
    static_assert(ROWS_PER_WG == 7, "two boundaries for each of four waves");
    {
        const int lane = threadIdx.x & 63, r = threadIdx.x >> 6;
        int lo[2] = {0, 0}, hi[2] = {n, n};
        while (lo[0] < hi[0] || lo[1] < hi[1]) {
            unsigned key[2];
            int step[2];
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                step[q] = (hi[q] - lo[q] + 63) / 64;
                key[q] = keys[min(lo[q] + lane * step[q], n - 1)];
            }
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                if (lo[q] >= hi[q]) continue;
                const int below = __popcll(__ballot(lo[q] + lane * step[q] < hi[q] && key[q] < v0 + r + 4 * q));
                if (below == 0) { hi[q] = lo[q]; continue; }      // keys[lo] >= v
                const int last = lo[q] + (below - 1) * step[q];   // keys[last] < v
                lo[q] = last + 1;
                hi[q] = min(hi[q], last + step[q]);
            }
        }
        if (lane == 0) { start[r] = lo[0]; start[r + 4] = lo[1]; }
    }
    __syncthreads();
    for (int r = threadIdx.x >> 6; r < ROWS_PER_WG; r += 4) {
        const unsigned v = v0 + r;
        if (v >= rows) break;
        const int s = __builtin_amdgcn_readfirstlane(start[r]), e = __builtin_amdgcn_readfirstlane(start[r + 1]);
        for (int col0 = 0; col0 < width; col0 += SWEEPS * 64 * VEC) {
            f32x4 acc[SWEEPS] = {};
            for (int i = s; i < e;) {
                if (part2 && i % (CHUNK * SUPER) == 0 && i + CHUNK * SUPER <= e) {
                    const int count = (e - i) / (CHUNK * SUPER), c0 = i / (CHUNK * SUPER);
                    add_rows<VEC>(acc, part2, width, col0, count, [&](int j) { return (unsigned)(c0 + j); });
                    i += count * CHUNK * SUPER;
                } else if (part && i % CHUNK == 0 && i + CHUNK <= e) {
                    int stop = e / CHUNK * CHUNK;             // as far as whole chunks go, or to the next run of chunks
                    const int next = (i / (CHUNK * SUPER) + 1) * (CHUNK * SUPER);
                    if (part2 && next < stop) stop = next;
                    const int c0 = i / CHUNK;
                    add_rows<VEC>(acc, part, width, col0, (stop - i) / CHUNK, [&](int j) { return (unsigned)(c0 + j); });
                    i = stop;
                } else {
                    int stop = e;
                    const int next = (i / CHUNK + 1) * CHUNK;
                    if (part && next < stop) stop = next;
                    const int i0 = i;
                    add_rows<VEC>(acc, dy, width, col0, stop - i, [&](int j) { return pos[i0 + j]; });
                    i = stop;
                }
            }
            put_row<VEC>(dtable + (size_t)v * width, acc, width, col0, scale);
        }
    }
}

struct GradPlan {
    int n, tiles, passes, bits, keybits;
    size_t keys, pos, keys2, pos2, counts, totals, part, part2, bytes;   // byte offsets into the workspace
};
static GradPlan grad_plan(long long n, long long rows, int width) {
    GradPlan g = {};
    g.n = (int)n;
    g.keybits = 1;
    while ((1ll << g.keybits) <= rows) ++g.keybits;               // `rows` itself is the key of an id out of range
    g.passes = (g.keybits + 7) / 8;
    g.bits = (g.keybits + g.passes - 1) / g.passes;
    g.tiles = (int)((n + TILE - 1) / TILE);
    size_t at = 0;
    auto take = [&](size_t b) { const size_t o = at; at += (b + 255) / 256 * 256; return o; };
    g.keys = take((size_t)n * 4);
    g.pos = take((size_t)n * 4);
    if (n > RANKED) {
        g.keys2 = take((size_t)n * 4);
        g.pos2 = take((size_t)n * 4);
        g.counts = take((size_t)g.tiles * MAXBINS * 4);
        g.totals = take(MAXBINS * 4);
    }
    g.part = take((size_t)(n / CHUNK) * width * 4);
    g.part2 = take((size_t)(n / (CHUNK * SUPER)) * width * 4);
    g.bytes = at;
    return g;
}

static const char* bad_shape(long long n, long long rows, long long width) {
    if (n < 0 || rows < 1 || width < 1) return "negative count or empty table";
    if (n > (1ll << 30) || rows > (1ll << 30) || width > (1 << 20)) return "more than 2^30 ids or rows, or 2^20 columns";
    // a launch has fewer than 2^32 threads in whole workgroups of 256, and rows of an odd width take a thread for each element
    if (n * width > (1ll << 32) - 256) return "more than 2^32 - 256 elements";
    return nullptr;
}

template <typename T, typename TO, int VEC>
static void launch_grad(const GradPlan& g, char* ws, const unsigned* keys, const unsigned* pos, unsigned rows, const void* dy, int width,
                        float scale, void* dtable, hipStream_t st) {
    const int cols = (width + SWEEPS * 64 * VEC - 1) / (SWEEPS * 64 * VEC);
    const int chunks = g.n / CHUNK, supers = g.n < SUPERS_FROM ? 0 : g.n / (CHUNK * SUPER);
    float *part = (float*)(ws + g.part), *part2 = (float*)(ws + g.part2);
    if (chunks) hipLaunchKernelGGL((chunk_sum_kernel<T, VEC>), dim3((chunks + 3) / 4, cols), dim3(256), 0, st, keys, pos, g.n, rows,
                                   (const T*)dy, width, part);
    if (supers) hipLaunchKernelGGL((super_sum_kernel<VEC>), dim3(supers, cols), dim3(64), 0, st, keys, g.n, rows, width, part, part2);
    hipLaunchKernelGGL((table_grad_kernel<T, TO, VEC>), dim3((rows + ROWS_PER_WG - 1) / ROWS_PER_WG), dim3(256), 0, st, keys, pos, g.n,
                       rows, (const T*)dy, width, scale, chunks ? part : nullptr, supers ? part2 : nullptr, (TO*)dtable);
}

template <typename TI, typename TO>
static void launch_rows(const void* ids, int ids64, long long n, const void* table, long long rows, int width, float scale, void* out,
                        bool vec, hipStream_t st) {
    const unsigned per_row = vec ? width / 8 : width, total = (unsigned)(n * per_row);
    const dim3 grid((unsigned)(((size_t)total + 255) / 256)), blk(256);
#define ROWS(VEC, PAST) hipLaunchKernelGGL((embed_rows_kernel<TI, TO, VEC, PAST>), grid, blk, 0, st, ids, ids64, (const TI*)table, (TO*)out, \
                                           total, per_row, rows, width, scale)
    if (!vec) ROWS(1, false);
    else if ((size_t)n * width * sizeof(TO) > (128u << 20)) ROWS(8, true);
    else ROWS(8, false);
#undef ROWS
}

}  // namespace

extern "C" {

int mi355_embedding_fwd(const void* ids, int ids64, long long n, const void* table, int table_bf16, long long rows, int width, float scale,
                        void* out, int out_bf16, void* stream) {
    if (const char* why = bad_shape(n, rows, width)) return mi355_fail(MI355_ERR_ARG, "embedding: %s", why);
    if (n == 0) return MI355_OK;
    if (!ids || !table || !out) return mi355_fail(MI355_ERR_ARG, "embedding: null pointer");
    const hipStream_t st = (hipStream_t)stream;
    const bool vec = width % 8 == 0 && (uintptr_t)table % 16 == 0 && (uintptr_t)out % 16 == 0;
    ProfScope prof(FAM_ELEM, st, (double)n * width * ((table_bf16 ? 2 : 4) + (out_bf16 ? 2 : 4)));
    if (table_bf16) {
        if (out_bf16) launch_rows<bf16_t, bf16_t>(ids, ids64, n, table, rows, width, scale, out, vec, st);
        else launch_rows<bf16_t, float>(ids, ids64, n, table, rows, width, scale, out, vec, st);
    } else {
        if (out_bf16) launch_rows<float, bf16_t>(ids, ids64, n, table, rows, width, scale, out, vec, st);
        else launch_rows<float, float>(ids, ids64, n, table, rows, width, scale, out, vec, st);
    }
    return mi355_check_launch("embedding_fwd");
}

size_t mi355_embedding_bwd_workspace_bytes(long long n, long long rows, int width) {
    if (bad_shape(n, rows, width)) return 0;
    return grad_plan(n, rows, width).bytes;
}

int mi355_embedding_bwd(const void* ids, int ids64, long long n, const void* dy, int dy_bf16, long long rows, int width, float scale,
                        void* dtable, int out_bf16, void* ws, size_t ws_bytes, void* stream) {
    if (const char* why = bad_shape(n, rows, width)) return mi355_fail(MI355_ERR_ARG, "embedding_bwd: %s", why);
    if (rows > (1ll << 26)) return mi355_fail(MI355_ERR_ARG, "embedding_bwd: more than 2^26 rows");
    if (!dtable || (n > 0 && (!ids || !dy || !ws))) return mi355_fail(MI355_ERR_ARG, "embedding_bwd: null pointer");
    const GradPlan g = grad_plan(n, rows, width);
    if (ws_bytes < g.bytes) return mi355_fail(MI355_ERR_ARG, "embedding_bwd: workspace of %zu bytes, %zu needed", ws_bytes, g.bytes);
    if ((uintptr_t)ws % 16) return mi355_fail(MI355_ERR_ARG, "embedding_bwd: workspace not 16-byte aligned");
    const hipStream_t st = (hipStream_t)stream;
    ProfScope prof(FAM_ELEM, st, (double)n * width * (dy_bf16 ? 2 : 4) + (double)rows * width * (out_bf16 ? 2 : 4));
    char* w = (char*)ws;
    unsigned *keys = (unsigned*)(w + g.keys), *pos = (unsigned*)(w + g.pos);
    const unsigned R = (unsigned)rows;
    if (n > 0 && n <= RANKED) {
        hipLaunchKernelGGL(rank_sort_kernel, dim3((unsigned)((n + 256 / SHARES - 1) / (256 / SHARES))), dim3(256), ((size_t)n + 4 * SHARES - 1) / (4 * SHARES) * (16 * SHARES), st, ids, ids64, (int)n, R, keys, pos);
    } else if (n > 0) {
        unsigned* counts = (unsigned*)(w + g.counts);
        unsigned *k2 = (unsigned*)(w + g.keys2), *p2 = (unsigned*)(w + g.pos2);
        const unsigned mask = (1u << g.bits) - 1;
        unsigned* totals = (unsigned*)(w + g.totals);
        for (int p = 0; p < g.passes; ++p) {
            const bool into2 = ((g.passes - p) & 1) == 0;        // the last pass ends in (keys, pos)
            const unsigned *ki = into2 ? keys : k2, *pi = into2 ? pos : p2;
            unsigned *ko = into2 ? k2 : keys, *po = into2 ? p2 : pos;
            const int shift = p * g.bits;
            if (p == 0) hipLaunchKernelGGL((radix_count_kernel<true>), dim3(g.tiles), dim3(256), 0, st, ids, ids64, ki, g.n, R, shift, mask, g.tiles, counts);
            else hipLaunchKernelGGL((radix_count_kernel<false>), dim3(g.tiles), dim3(256), 0, st, ids, ids64, ki, g.n, R, shift, mask, g.tiles, counts);
            hipLaunchKernelGGL(scan_kernel, dim3((mask + 4) / 4), dim3(256), 0, st, counts, totals, (int)(mask + 1), g.tiles);
            if (p == 0) hipLaunchKernelGGL((radix_scatter_kernel<true>), dim3(g.tiles), dim3(256), 0, st, ids, ids64, ki, pi, g.n, R, shift, g.bits, g.tiles, counts, totals, ko, po);
            else hipLaunchKernelGGL((radix_scatter_kernel<false>), dim3(g.tiles), dim3(256), 0, st, ids, ids64, ki, pi, g.n, R, shift, g.bits, g.tiles, counts, totals, ko, po);
        }
    }
    const bool vec = width % 4 == 0 && (uintptr_t)dy % (dy_bf16 ? 8 : 16) == 0 && (uintptr_t)dtable % (out_bf16 ? 8 : 16) == 0;
#define GRAD(T, TO) (vec ? launch_grad<T, TO, 4>(g, w, keys, pos, R, dy, width, scale, dtable, st) \
                         : launch_grad<T, TO, 1>(g, w, keys, pos, R, dy, width, scale, dtable, st))
    if (dy_bf16) { if (out_bf16) GRAD(bf16_t, bf16_t); else GRAD(bf16_t, float); }
    else { if (out_bf16) GRAD(float, bf16_t); else GRAD(float, float); }
#undef GRAD
    return mi355_check_launch("embedding_bwd");
}

}  // extern "C"
