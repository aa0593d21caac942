// Attention over packed documents: entry points.
#include "doc_tiles.h"

namespace {

static const char* bad_sizes(int docs, int Tq, int Tk, int Hq, int Hkv, int D) {
    if (docs < 1 || docs > (1 << 30) || Tq < 0 || Tk < 0) return "no document, more than 2^30 documents, or a negative number of tokens";
    if (Hq < 1 || Hkv < 1 || Hq % Hkv) return "query heads must be a multiple of key heads";
    if (D < 8 || D > 128 || D % 8) return "heads must be a multiple of 8 wide, at most 128";
    if ((long long)Tq * Hq >= (1ll << 30) || (long long)Tk * Hkv >= (1ll << 30)) return "2^30 rows or more";
    return nullptr;
}
static size_t bwd_rows_bytes(int Tq, int Hq) { return ((size_t)Tq * 16 + (size_t)Tq * Hq * 4 + 255) / 256 * 256; }
static size_t part_q_bytes(int Tq, int Tk, int Hq, int Hkv, int D, int docs) {
    const int s = key_runs(Tq, Tk, Hq, Hkv, docs);
    return s > 1 ? ((size_t)s * Tq * Hq * D * 4 + 255) / 256 * 256 : 0;
}
static bool off16(const void* a) { return ((uintptr_t)a & 15) != 0; }
static bool bad_ld(long long ld) { return ld < 0 || ld % 8 != 0 || ld > (1 << 23); }

static int fill(DocArgs& a, const char* who, int docs, int Tq, int Tk, int Hq, int Hkv, int D, const int* q_off, const int* k_off,
                const int* prefix, const float* slopes, float cap, int causal, int align_start, float scale, float drop_p, unsigned seed) {
    if (const char* why = bad_sizes(docs, Tq, Tk, Hq, Hkv, D)) return mi355_fail(MI355_ERR_ARG, "%s: %s", who, why);
    if (!q_off || !k_off) return mi355_fail(MI355_ERR_ARG, "%s: null pointer", who);
    if (prefix && !causal) return mi355_fail(MI355_ERR_ARG, "%s: a prefix without the causal mask it lifts", who);
    // the tanh is 1 - 2 / (1 + 2^x), good to 2^-22 of the cap: 2^-12 of a nat at the limit
    // and below the normal range 1 / cap is infinite
    if (!(cap == 0.f || (cap >= 0x1p-126f && cap <= 1024.f))) return mi355_fail(MI355_ERR_ARG, "%s: cap %g, neither 0 (none) nor between 2^-126 and 1024", who, (double)cap);
    if (!(drop_p >= 0.f && drop_p < 1.f)) return mi355_fail(MI355_ERR_ARG, "%s: dropout %g", who, (double)drop_p);
    a.docs = docs; a.Tq = Tq; a.Tk = Tk; a.Hq = Hq; a.Hkv = Hkv; a.G = Hq / Hkv; a.D = D;
    a.q_off = q_off; a.k_off = k_off; a.prefix = prefix; a.slopes = slopes;
    a.causal = causal != 0; a.align_start = align_start != 0;
    a.scale = scale; a.cap = cap; a.rcap = cap > 0.f ? 1.f / cap : 0.f;
    a.drop_thresh = (unsigned)((double)drop_p * 4294967296.0);
    a.drop_scale = 1.f / (1.f - drop_p);
    a.seed = seed;
    return MI355_OK;
}

}  // namespace

extern "C" {

size_t mi355_doc_attention_fwd_workspace_bytes(int Tq, int Tk, int Hq, int Hkv, int D, int docs) {
    if (bad_sizes(docs, Tq, Tk, Hq, Hkv, D)) return 0;
    return doc_fwd_workspace(Tq, Tk, Hq, Hkv, D, docs);
}

int mi355_doc_attention_fwd(const void* q, const void* k, const void* v, void* out, float* lse, const int* q_off, const int* k_off, int docs,
                            const int* prefix, const float* slopes, float cap, int causal, int align_start, int Tq, int Tk, int Hq, int Hkv,
                            int D, long long ldq, long long ldk, long long ldv, long long ldo, float scale, float drop_p, unsigned seed,
                            void* ws, size_t ws_bytes, void* stream) {
    DocArgs a = {};
    if (const int rc = fill(a, "doc_attention", docs, Tq, Tk, Hq, Hkv, D, q_off, k_off, prefix, slopes, cap, causal, align_start, scale, drop_p, seed)) return rc;
    if (Tq == 0) return MI355_OK;
    if (!q || !out || !lse || (Tk > 0 && (!k || !v))) return mi355_fail(MI355_ERR_ARG, "doc_attention: null pointer");
    if (off16(q) || off16(k) || off16(v) || off16(out)) return mi355_fail(MI355_ERR_ARG, "doc_attention: operands not 16-byte aligned");
    if (bad_ld(ldq) || bad_ld(ldk) || bad_ld(ldv) || bad_ld(ldo) || ldo < (long long)Hq * D)
        return mi355_fail(MI355_ERR_ARG, "doc_attention: row strides must be multiples of 8, at most 2^23");
    const size_t need = mi355_doc_attention_fwd_workspace_bytes(Tq, Tk, Hq, Hkv, D, docs);
    if (need && (!ws || ws_bytes < need || off16(ws))) return mi355_fail(MI355_ERR_ARG, "doc_attention: workspace of %zu bytes, %zu needed, 16-byte aligned", ws ? ws_bytes : 0, need);
    a.q = (const bf16_t*)q; a.k = (const bf16_t*)k; a.v = (const bf16_t*)v; a.out = (bf16_t*)out; a.lse = lse;
    a.ldq = ldq; a.ldk = ldk; a.ldv = ldv; a.ldo = ldo;
    const hipStream_t st = (hipStream_t)stream;
    ProfScope prof(FAM_ATTN, st, 4.0 * Tq * (double)Tk / docs * Hq * D);
    a.part = (float*)ws;
    return doc_fwd_tiles(a, st);
}

size_t mi355_doc_attention_bwd_workspace_bytes(int Tq, int Tk, int Hq, int Hkv, int D, int docs, int causal) {
    if (bad_sizes(docs, Tq, Tk, Hq, Hkv, D)) return 0;
    const int splits = doc_bwd_kv_splits(Tq, Tk, Hq, Hkv, docs, causal != 0);
    return bwd_rows_bytes(Tq, Hq) + part_q_bytes(Tq, Tk, Hq, Hkv, D, docs) + (splits > 1 ? (size_t)splits * Tk * Hkv * 2 * D * 4 : 0) + 16;
}

int mi355_doc_attention_bwd(const void* q, const void* k, const void* v, const void* o, const void* dout, const float* lse, void* dq, void* dk,
                            void* dv, const int* q_off, const int* k_off, int docs, const int* prefix, const float* slopes, float cap,
                            int causal, int align_start, int Tq, int Tk, int Hq, int Hkv, int D, long long ldq, long long ldk, long long ldv,
                            long long ldo, long long lddo, long long lddq, long long lddk, long long lddv, float scale, float drop_p,
                            unsigned seed, void* ws, size_t ws_bytes, void* stream) {
    DocArgs a = {};
    if (const int rc = fill(a, "doc_attention_bwd", docs, Tq, Tk, Hq, Hkv, D, q_off, k_off, prefix, slopes, cap, causal, align_start, scale, drop_p, seed)) return rc;
    if (Tq == 0 && Tk == 0) return MI355_OK;
    if ((Tq > 0 && (!q || !o || !dout || !lse || !dq)) || (Tk > 0 && (!k || !v || !dk || !dv)))
        return mi355_fail(MI355_ERR_ARG, "doc_attention_bwd: null pointer");
    if (off16(q) || off16(k) || off16(v) || off16(o) || off16(dout) || off16(dq) || off16(dk) || off16(dv))
        return mi355_fail(MI355_ERR_ARG, "doc_attention_bwd: operands not 16-byte aligned");
    if (bad_ld(ldq) || bad_ld(ldk) || bad_ld(ldv) || bad_ld(ldo) || bad_ld(lddo) || bad_ld(lddq) || bad_ld(lddk) || bad_ld(lddv))
        return mi355_fail(MI355_ERR_ARG, "doc_attention_bwd: row strides must be multiples of 8, at most 2^23");
    if (lddq < (long long)Hq * D || lddk < (long long)Hkv * D || lddv < (long long)Hkv * D)
        return mi355_fail(MI355_ERR_ARG, "doc_attention_bwd: rows of a gradient overlap");
    const size_t need = mi355_doc_attention_bwd_workspace_bytes(Tq, Tk, Hq, Hkv, D, docs, causal);
    if (!ws || ws_bytes < need || off16(ws)) return mi355_fail(MI355_ERR_ARG, "doc_attention_bwd: workspace of %zu bytes, %zu needed, 16-byte aligned", ws ? ws_bytes : 0, need);
    a.q = (const bf16_t*)q; a.k = (const bf16_t*)k; a.v = (const bf16_t*)v; a.o = (const bf16_t*)o; a.dout = (const bf16_t*)dout;
    a.dq = (bf16_t*)dq; a.dk = (bf16_t*)dk; a.dv = (bf16_t*)dv; a.lse = (float*)lse;
    a.ldq = ldq; a.ldk = ldk; a.ldv = ldv; a.ldo = ldo; a.lddo = lddo; a.lddq = lddq; a.lddk = lddk; a.lddv = lddv;
    a.rows = (int4*)ws;
    a.delta = (float*)((char*)ws + (size_t)Tq * 16);
    a.part_q = (float*)((char*)ws + bwd_rows_bytes(Tq, Hq));
    a.splits_q = key_runs(Tq, Tk, Hq, Hkv, docs);
    a.part = (float*)((char*)ws + bwd_rows_bytes(Tq, Hq) + part_q_bytes(Tq, Tk, Hq, Hkv, D, docs));
    a.splits = doc_bwd_kv_splits(Tq, Tk, Hq, Hkv, docs, a.causal);
    const hipStream_t st = (hipStream_t)stream;
    ProfScope prof(FAM_ATTN, st, 10.0 * Tq * (double)Tk / docs * Hq * D);
    if (Tq > 0) if (const int rc = doc_bwd_q_tiles(a, st)) return rc;
    return Tk > 0 ? doc_bwd_kv_tiles(a, st) : MI355_OK;
}

}  // extern "C"
