// The C ABI's operators on device memory: the checks of their arguments, the
// device they run on, and the launches of kv4.hip and logprobs.hip.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "ana_internal.h"
#include "kv4.h"
#include "logprobs.h"

using namespace ana;

static_assert(ANA_T_F32 == ET_F32 && ANA_T_BF16 == ET_BF16 && ANA_T_F16 == ET_F16, "one numbering of types");

namespace {

// the current device for a call, and the caller's again after it
struct OnDevice {
  int before = -1;
  hipError_t e;
  explicit OnDevice(int device) {
    e = hipGetDevice(&before);
    if (e != hipSuccess || before == device) before = -1;
    else e = hipSetDevice(device);
  }
  ~OnDevice() {
    if (before >= 0) (void)hipSetDevice(before);
  }
};

size_t size_of(int type) { return type == ANA_T_F32 ? 4 : 2; }

// nullptr, or why a cache's shape is refused
const char* shape_problem(uint32_t seqs, uint32_t slots, uint32_t heads, uint32_t hd) {
  if (!kv4_fits(hd)) return "head size is not 32, 64 or 128";
  if (seqs == 0 || slots == 0 || heads == 0) return "no sequences, slots or heads";
  if (heads > 65535) return "more than 65535 heads";
  if (slots > 0x7FFFFFE0u) return "more than 2^31 - 32 slots";
  if ((double)seqs * heads * ((slots + 31) / 32) * kv4_record(hd) > 1e18) return "a cache beyond any memory";
  return nullptr;
}

int check_cache(const char* fn, const ana_kv4* c, Kv4* o) {
  if (!c || !c->data) return fail_call(ANA_EINVAL, "%s: null cache", fn);
  if (const char* why = shape_problem(c->seqs, c->slots, c->heads, c->hd)) return fail_call(ANA_EINVAL, "%s: %s", fn, why);
  if ((uintptr_t)c->data % 16) return fail_call(ANA_EINVAL, "%s: the cache is not on a 16-byte border", fn);
  *o = Kv4{(uint8_t*)c->data, kv4_seq_bytes(c->slots, c->heads, c->hd), c->seqs, c->slots, (c->slots + 31) / 32, c->heads,
           c->hd};
  return ANA_OK;
}

int check_rows(const char* fn, const ana_kv4* c, const ana_kv4_rows* r, Kv4Rows* o) {
  if (!r) return fail_call(ANA_EINVAL, "%s: null rows", fn);
  if (r->n && !r->pos) return fail_call(ANA_EINVAL, "%s: null positions", fn);
  if (!r->off && r->rows != r->n)
    return fail_call(ANA_EINVAL, "%s: %u rows of %u sequences without offsets", fn, r->rows, r->n);
  if (!r->seq && r->n > c->seqs)
    return fail_call(ANA_EINVAL, "%s: %u sequences in a cache of %u", fn, r->n, c->seqs);
  if (r->rows > kKv4MaxRows || r->n > kKv4MaxRows) return fail_call(ANA_EINVAL, "%s: more than 2^26 rows or sequences", fn);
  *o = Kv4Rows{r->seq, r->pos, r->off, r->n, r->rows};
  return ANA_OK;
}

// (out: no two rows' heads may share elements)
int check_mat(const char* fn, const char* name, const ana_mat* x, int type, const ana_kv4_rows* r, uint32_t heads,
              uint32_t hd, bool out, Kv4Mat* o) {
  if (!x || (!x->p && r->rows)) return fail_call(ANA_EINVAL, "%s: null %s", fn, name);
  if ((uintptr_t)x->p % size_of(type)) return fail_call(ANA_EINVAL, "%s: %s is not on an element's border", fn, name);
  if ((r->rows > 1 && x->row < hd) || (heads > 1 && x->head < hd))
    return fail_call(ANA_EINVAL, "%s: rows or heads of %s overlap", fn, name);
  if (out && r->rows > 1 && heads > 1) {
    const bool by_row = x->row >= x->head;   // (whole heads of a row, or whole rows of a head, lie together)
    const uint64_t in = by_row ? x->head : x->row, cnt = by_row ? heads : r->rows;
    if (in > (UINT64_MAX - hd) / cnt || std::max(x->row, x->head) < (cnt - 1) * in + hd)
      return fail_call(ANA_EINVAL, "%s: rows and heads of %s overlap", fn, name);
  }
  *o = Kv4Mat{x->p, x->row, x->head};
  return ANA_OK;
}

int check_type(const char* fn, int type) {
  if (type != ANA_T_F32 && type != ANA_T_BF16 && type != ANA_T_F16) return fail_call(ANA_EINVAL, "%s: unknown type %d", fn, type);
  return ANA_OK;
}

int launched(const char* fn, hipError_t e) {
  if (e == hipSuccess) return ANA_OK;
  return fail_call(ANA_EDEVICE, "%s: device fault: %s", fn, hipGetErrorString(e));
}

}  // namespace

extern "C" uint64_t ana_kv4_bytes(uint32_t seqs, uint32_t slots, uint32_t heads, uint32_t hd) {
  if (shape_problem(seqs, slots, heads, hd)) return 0;
  return seqs * kv4_seq_bytes(slots, heads, hd);
}

extern "C" int ana_kv4_write(const ana_kv4* c, const ana_kv4_rows* r, int type, const ana_mat* k, const ana_mat* v,
                             void* stream) {
  const char* fn = "ana_kv4_write";
  Kv4 kc;
  Kv4Rows kr;
  Kv4Mat km, vm;
  if (int e = check_cache(fn, c, &kc)) return e;
  if (int e = check_rows(fn, c, r, &kr)) return e;
  if (int e = check_type(fn, type)) return e;
  if (int e = check_mat(fn, "k", k, type, r, c->heads, c->hd, false, &km)) return e;
  if (int e = check_mat(fn, "v", v, type, r, c->heads, c->hd, false, &vm)) return e;
  if (r->n == 0 || r->rows == 0) return ANA_OK;
  OnDevice on(c->device);
  if (on.e != hipSuccess) return launched(fn, on.e);
  return launched(fn, launch_kv4_write(kc, kr, type, km, vm, nullptr, nullptr, nullptr, 0, (hipStream_t)stream));
}

extern "C" int ana_kv4_read(const ana_kv4* c, const ana_kv4_rows* r, int type, const ana_mat* k, const ana_mat* v,
                            void* stream) {
  const char* fn = "ana_kv4_read";
  Kv4 kc;
  Kv4Rows kr;
  Kv4Mat km, vm;
  if (int e = check_cache(fn, c, &kc)) return e;
  if (int e = check_rows(fn, c, r, &kr)) return e;
  if (int e = check_type(fn, type)) return e;
  if (int e = check_mat(fn, "k", k, type, r, c->heads, c->hd, true, &km)) return e;
  if (int e = check_mat(fn, "v", v, type, r, c->heads, c->hd, true, &vm)) return e;
  if (r->n == 0 || r->rows == 0) return ANA_OK;
  OnDevice on(c->device);
  if (on.e != hipSuccess) return launched(fn, on.e);
  return launched(fn, launch_kv4_read(kc, kr, type, km, vm, (hipStream_t)stream));
}

static int check_heads(const char* fn, const ana_kv4* c, const ana_kv4_rows* r, uint32_t hq) {
  if (hq == 0 || hq % c->heads) return fail_call(ANA_EINVAL, "%s: %u query heads over %u key heads", fn, hq, c->heads);
  // (the pairs of a sequence are counted in 32 bits)
  if ((uint64_t)r->rows * hq > 0x7FFFFFFFull || kv4_attend_groups(c->heads, r->n, r->rows, r->off != nullptr, hq) > kKv4MaxGroups)
    return fail_call(ANA_EINVAL, "%s: %u rows of %u query heads are more than a launch takes", fn, r->rows, hq);
  return ANA_OK;
}

extern "C" uint64_t ana_kv4_attend_ws(const ana_kv4* c, const ana_kv4_rows* r, uint32_t hq, uint64_t live) {
  if (!c || !r || hq == 0 || shape_problem(c->seqs, c->slots, c->heads, c->hd) || hq % c->heads) return 0;
  const Kv4 kc{nullptr, 0, c->seqs, c->slots, (c->slots + 31) / 32, c->heads, c->hd};
  const uint32_t ns = kv4_split(kc, r->n, r->rows, r->off != nullptr, hq, live);
  return 4 * kv4_part_floats(r->rows, hq, c->hd, ns);
}

extern "C" int ana_kv4_attend(const ana_kv4* c, const ana_kv4_rows* r, int type, const ana_mat* q, uint32_t hq,
                              float scale, const float* sink, const ana_mat* o, uint64_t live, void* ws,
                              uint64_t ws_bytes, void* stream) {
  const char* fn = "ana_kv4_attend";
  Kv4Attend a{};
  if (int e = check_cache(fn, c, &a.c)) return e;
  if (int e = check_rows(fn, c, r, &a.r)) return e;
  if (int e = check_type(fn, type)) return e;
  if (int e = check_heads(fn, c, r, hq)) return e;
  if (int e = check_mat(fn, "q", q, type, r, hq, c->hd, false, &a.q)) return e;
  if (int e = check_mat(fn, "o", o, type, r, hq, c->hd, true, &a.o)) return e;
  if (r->n == 0 || r->rows == 0) return ANA_OK;
  a.nsplit = kv4_split(a.c, r->n, r->rows, r->off != nullptr, hq, live);
  const uint64_t need = 4 * kv4_part_floats(r->rows, hq, c->hd, a.nsplit);
  if (need && (!ws || ws_bytes < need))
    return fail_call(ANA_EINVAL, "%s: a workspace of %llu bytes, not %llu", fn, (unsigned long long)need,
                     (unsigned long long)(ws ? ws_bytes : 0));
  if (need && (uintptr_t)ws % 16) return fail_call(ANA_EINVAL, "%s: the workspace is not on a 16-byte border", fn);
  a.hq = hq;
  a.scale = scale;
  a.sink = sink;
  a.part = (float*)ws;
  OnDevice on(c->device);
  if (on.e != hipSuccess) return launched(fn, on.e);
  return launched(fn, launch_kv4_attend(a, type, (hipStream_t)stream));
}

extern "C" uint64_t ana_row_logprobs_ws(uint32_t n, uint32_t vocab, uint32_t top) {
  if (vocab == 0 || vocab > kLpMaxVocab || top > kLpMaxTop) return 0;
  return 4 * logprobs_part_words(n, vocab, top);
}

extern "C" int ana_row_logprobs(int device, int type, const void* logits, uint64_t ld, uint32_t n, uint32_t vocab,
                                const uint32_t* tok, uint32_t top, float* lp, float* ent, uint32_t* rank,
                                uint32_t* top_tok, float* top_lp, void* ws, uint64_t ws_bytes, void* stream) {
  const char* fn = "ana_row_logprobs";
  if (int e = check_type(fn, type)) return e;
  if (vocab == 0 || vocab > kLpMaxVocab) return fail_call(ANA_EINVAL, "%s: a vocabulary of %u (1 .. %u)", fn, vocab, kLpMaxVocab);
  if (top > kLpMaxTop || top > vocab) return fail_call(ANA_EINVAL, "%s: %u alternatives of %u tokens (at most %u)", fn, top, vocab, kLpMaxTop);
  if (n > 1 && ld < vocab) return fail_call(ANA_EINVAL, "%s: rows of %u logits overlap", fn, vocab);
  if (n == 0) return ANA_OK;
  if (!logits || !ent || (tok && (!lp || !rank)) || (top && (!top_tok || !top_lp))) return fail_call(ANA_EINVAL, "%s: null argument", fn);
  if ((uintptr_t)logits % size_of(type)) return fail_call(ANA_EINVAL, "%s: the logits are not on an element's border", fn);
  if (n > logprobs_max_rows(vocab))
    return fail_call(ANA_EINVAL, "%s: %u rows (at most %u of %u logits)", fn, n, logprobs_max_rows(vocab), vocab);
  const uint64_t need = ana_row_logprobs_ws(n, vocab, top);
  if (need && (!ws || ws_bytes < need || (uintptr_t)ws % 4))
    return fail_call(ANA_EINVAL, "%s: a workspace of %llu bytes, not %llu", fn, (unsigned long long)need,
                     (unsigned long long)(ws ? ws_bytes : 0));
  OnDevice on(device);
  if (on.e != hipSuccess) return launched(fn, on.e);
  LogprobArgs a{logits, n > 1 ? ld : vocab, n, vocab, top, tok, lp, ent, rank, top_tok, top_lp, (uint32_t*)ws};
  return launched(fn, launch_logprobs(a, type, (hipStream_t)stream));
}
