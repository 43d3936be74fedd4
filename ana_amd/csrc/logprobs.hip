// Log probabilities of given tokens, their ranks, the entropy and the top
// alternatives of rows of logits (gfx950).
//
// One pass over a row: a workgroup keeps its piece of the row in registers,
// so the maximum m, then l = sum e^(x - m) and w = sum e^(x - m) (x - m), the
// given token's rank and the alternatives all come from one read.
//   lp(t) = x_t - m - log l        H = log l - w / l
// The entries at the maximum are counted (c), not summed: log l is
// log1p(c - 1 + sum of the others), which keeps a probability next to 1 and
// an entropy next to 0 to their own last bits.
//
// Alternatives: logits are ordered by value, then by the lower index (a NaN
// after every number), so an order key (value bits, ~index) is unique. The
// k-th largest of 64 group maxima is a bound that at least k logits reach and
// few more do; those go to LDS, where each counts the keys above its own.
// Where ties, or k near 64, make them too many, or rows of few numbers too
// few, a bisection over the keys finds a bound first (500 rows of 50021 bf16
// logits, 64 alternatives: 74 us, 280 by 64 rounds of a maximum; 256 group
// maxima take 48 there, but with the registers of their code 3000 rows with
// eight alternatives take 95 for 89).
#include <hip/hip_runtime.h>

#include <algorithm>

#include "kv4.h"
#include "logprobs.h"
#include "mfma.h"
#include "order.h"
#include "wave.h"

namespace ana {

namespace {

constexpr uint32_t kJoinKeys = 2048;   // keys that a row's join takes into LDS
constexpr uint32_t kJoinRank = 256;    // of them, those that it ranks by counting
constexpr uint32_t kHead = 8;   // a piece's words before its keys: m, c, l, w, rank

// the largest over the wave by DPP moves, as wmax's
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t dpp_u(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, CTRL, ROWS, 0xF, false);
}
__device__ __forceinline__ uint32_t wave_max32(uint32_t v) {
  v = max(v, dpp_u<0xB1, 0xF>(v));
  v = max(v, dpp_u<0x4E, 0xF>(v));
  v = max(v, dpp_u<0x141, 0xF>(v));
  v = max(v, dpp_u<0x140, 0xF>(v));
  v = max(v, dpp_u<0x142, 0xA>(v));
  v = max(v, dpp_u<0x143, 0xC>(v));
  return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}
__device__ __forceinline__ u64 wave_max64(u64 v) {
  const uint32_t hi = wave_max32((uint32_t)(v >> 32));
  return (u64)hi << 32 | wave_max32((uint32_t)(v >> 32) == hi ? (uint32_t)v : 0u);
}

// the larger of two, NaN if either is
__device__ __forceinline__ float max_or_nan(float a, float b) { return __builtin_elementwise_maximum(a, b); }

// a row's results from its sums: entries at the maximum m are c, the others'
// sums l and w
struct RowSums {
  float m, c, l, w;
  // a NaN among the logits makes l one
  __device__ __forceinline__ bool bad() const { return m == INFINITY || l != l; }
  __device__ __forceinline__ float log_sum() const { return log1pf((c - 1.0f) + l); }
  __device__ __forceinline__ float lp(float x, float ls) const {
    if (bad() || x != x) return __builtin_nanf("");
    if (x == -INFINITY) return x;
    return (x - m) - ls;
  }
  __device__ __forceinline__ float entropy(float ls) const {
    if (bad()) return __builtin_nanf("");
    return m == -INFINITY ? 0.0f : ls - w / (c + l);
  }
};

// Piece z of row r, elements z C .. (C a multiple of 16 bytes of elements, at
// most NT V W). The row may start anywhere: whole 16-byte vectors from its
// first border on, the elements before and after them one each for the first
// threads. Places that no logit fills hold -inf, which changes no sum and
// nothing that is compared with a finite bound; the paths without one look at
// the places. Alone (one piece) it writes the row's results, else its sums
// and keys.
template <typename T, int NT, int V>
__global__ __launch_bounds__(NT) __attribute__((amdgpu_waves_per_eu(8))) void k_logprobs(LogprobArgs a, uint32_t C, uint32_t S) {
  constexpr int W = 16 / sizeof(T), NW = NT / 64, CAP = 512;
  typedef T vec_t __attribute__((ext_vector_type(W)));
  __shared__ float tmax[NW][64];
  __shared__ __align__(16) float gmax[64];
  __shared__ float red[NW][3];
  __shared__ uint32_t redu[NW], reach_s[NW];
  __shared__ float bound_s;
  __shared__ uint32_t ncand;
  __shared__ u64 cand[CAP], best[kLpMaxTop];
  const uint32_t tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
  const uint32_t r = blockIdx.x / S, z = blockIdx.x % S;
  const T* row = (const T*)a.logits + (uint64_t)r * a.ld;
  const uint32_t e0 = z * C, cnt = min(C, a.vocab - e0);
  const T* p = row + e0;
  const uint32_t head = min((uint32_t)((16 - (uintptr_t)p % 16) % 16 / sizeof(T)), cnt);
  const uint32_t nvec = (cnt - head) / W, tail0 = head + nvec * W;
  const uint32_t k = a.top;
  vec_t x[V];
#pragma unroll
  for (int u = 0; u < V; u++) {
    const uint32_t v = u * NT + tid;
    if (v < nvec) {
      x[u] = *reinterpret_cast<const vec_t*>(p + head + v * W);
    } else {
#pragma unroll
      for (int e = 0; e < W; e++) x[u][e] = (T)-INFINITY;
    }
  }
  // this thread's element before or after the vectors
  const uint32_t edge = tid < head ? tid : tail0 + (tid - head);
  const bool has_edge = tid < head || edge < cnt;
  const float xe = has_edge ? (float)p[edge] : -INFINITY;
  const uint32_t tk = a.tok ? a.tok[r] : 0xFFFFFFFFu;
  const bool given = tk < a.vocab;
  const float xt = given ? (float)row[tk] : 0.0f;
  if (tid == 0) ncand = 0;

  // f(value, index) over the thread's share of the piece, read again: the
  // rare paths, which would take the common ones' registers
  auto each = [&](auto&& f) {
    uint32_t i = tid;
    asm volatile("" : "+v"(i));   // (nor their addresses' registers)
#pragma unroll 4
    for (; i < cnt; i += NT) f((float)p[i], e0 + i);
  };

  float m = fmaxf(xe, -INFINITY);
#pragma unroll
  for (int u = 0; u < V; u++)
    if (u * NT < nvec) {
#pragma unroll
      for (int e = 0; e < W; e++) m = fmaxf(m, (float)x[u][e]);
    }
  const float tm = m;
  tmax[wv][lane] = tm;
  __syncthreads();
  // group l: lane l of every wave
  float gm = tmax[0][lane];
#pragma unroll
  for (int i = 1; i < NW; i++) gm = fmaxf(gm, tmax[i][lane]);
  m = wmax(gm);
  // the k-th largest group maximum: the least that fewer than k are above
  if (wv == NW - 1 && k) {
    gmax[lane] = gm;
    __builtin_amdgcn_wave_barrier();
    uint32_t above = 0;
#pragma unroll
    for (int i = 0; i < 16; i++) {
      const f32x4_t o = reinterpret_cast<const f32x4_t*>(gmax)[i];
      above += (o[0] > gm) + (o[1] > gm) + (o[2] > gm) + (o[3] > gm);
    }
    const float b = -wmax(above < k ? -gm : -INFINITY);
    if (lane == 0) bound_s = b;
  }
  // (+inf: the row's results are NaN whatever the sums)
  const float ms = m == -INFINITY || m == INFINITY ? 0.0f : m;
  constexpr float log2e = 1.4426950408889634f;
  float l = 0.0f, w = 0.0f, c = 0.0f;
  auto sums = [&](auto top) {
    // (far below the maximum, and at -inf, both terms are 0)
    auto term = [&](float v) {
      const float d = max_or_nan(v - ms, -200.0f);
      float t = __builtin_amdgcn_exp2f(d * log2e);
      if constexpr (decltype(top)::value) {
        t = v == m ? 0.0f : t;
        c += v == m ? 1.0f : 0.0f;
      }
      l += t;
      w = fmaf(t, d, w);
    };
    term(xe);
#pragma unroll
    for (int u = 0; u < V; u++)
      if (u * NT < nvec) {
#pragma unroll
        for (int e = 0; e < W; e++) term((float)x[u][e]);
      }
  };
  if (__any(tm == m)) sums(std::true_type{});
  else sums(std::false_type{});
  uint32_t above = 0;
  if (given && xt > -INFINITY) {
    // above x_t, or before the token and not below it: above the next float down
    const uint32_t ut = __builtin_bit_cast(uint32_t, xt);
    const float xp = xt == 0.0f ? -1.401298464e-45f : __builtin_bit_cast(float, xt > 0.0f ? ut - 1 : ut + 1);
    above += has_edge && xe > (e0 + edge < tk ? xp : xt);
#pragma unroll
    for (int u = 0; u < V; u++)
      if (u * NT < nvec) {
        const uint32_t i = e0 + head + (u * NT + tid) * W;
        const float t = i + W <= tk ? xp : xt;
#pragma unroll
        for (int e = 0; e < W; e++) above += (float)x[u][e] > t;
        if (__any(i <= tk && tk < i + W)) {
#pragma unroll
          for (int e = 0; e < W; e++) above += i + W > tk && i + e < tk && (float)x[u][e] == xt;
        }
      }
  } else if (given) {
    const u64 kt = key_of(xt, tk);
    each([&](float v, uint32_t i) { above += key_of(v, i) > kt; });
  }
  float s3[3] = {l, w, c};
  wsum_n(s3);
#pragma unroll
  for (int mk = 32; mk >= 1; mk >>= 1) above += __shfl_xor(above, mk, 64);
  if (lane == 0) {
    red[wv][0] = s3[0];
    red[wv][1] = s3[1];
    red[wv][2] = s3[2];
    redu[wv] = above;
  }
  __syncthreads();
  if (k) {
    const float bound = bound_s;
    const uint32_t want = min(k, cnt);
    uint32_t nc = 0;
    if (bound > -INFINITY) {
      if (__any(tm >= bound)) {
        auto offer = [&](float v, uint32_t i) {
          if (v >= bound) {
            const uint32_t at = atomicAdd(&ncand, 1u);
            if (at < CAP) cand[at] = key_of(v, i);
          }
        };
        offer(xe, e0 + edge);
#pragma unroll
        for (int u = 0; u < V; u++)
          if (u * NT < nvec) {
            float t = (float)x[u][0];
#pragma unroll
            for (int e = 1; e < W; e++) t = fmaxf(t, (float)x[u][e]);
            if (__any(t >= bound)) {
#pragma unroll
              for (int e = 0; e < W; e++) offer((float)x[u][e], e0 + head + (u * NT + tid) * W + e);
            }
          }
      }
      __syncthreads();
      nc = ncand;
    }
    if (tid < k && tid >= want) best[tid] = 0;
    if (nc > CAP || nc < want) {
      // a key that `want` to CAP of the piece's reach: more than CAP reach lo,
      // fewer than want hi
      auto reach = [&](u64 t) {
        uint32_t n = 0;
        each([&](float v, uint32_t at) { n += key_of(v, at) >= t; });
#pragma unroll
        for (int mk = 32; mk >= 1; mk >>= 1) n += __shfl_xor(n, mk, 64);
        __syncthreads();
        if (lane == 0) reach_s[wv] = n;
        __syncthreads();
        n = 0;
#pragma unroll
        for (int o = 0; o < NW; o++) n += reach_s[o];
        return n;
      };
      // (without a bound: all of a short piece, or the numbers above -inf, or
      // -inf with them)
      constexpr u64 finite = 0x00800000ull << 32;   // (above every key of -inf)
      const bool few = nc < want;
      u64 lo = 0, hi = ((u64)order_of(m) + 1) << 32, t = few ? finite : (u64)order_of(bound) << 32;
      if (few && cnt <= CAP) {
        t = 0;
        nc = cnt;
      }
      for (uint32_t n = 0; nc > CAP || nc < want; n++) {
        if (few || n) nc = reach(t);
        if (nc <= CAP && nc >= want) break;
        if (nc > CAP) lo = t;
        else hi = t;
        if (few && n == 0 && nc < want) {
          t = finite - (1ull << 32);
          continue;
        }
        if (lo >> 32 == (hi - 1) >> 32) {   // one value: only the piece's places are left
          const u64 o = lo >> 32 << 32;
          lo = max(lo, o | (0xFFFFFFFFu - (e0 + cnt - 1)));
          hi = min(hi, (o | (0xFFFFFFFFu - e0)) + 1);
        }
        t = lo + (hi - lo) / 2;
      }
      if (tid == 0) ncand = 0;
      __syncthreads();
      each([&](float v, uint32_t at) {
        const u64 q = key_of(v, at);
        if (q >= t) cand[atomicAdd(&ncand, 1u)] = q;
      });
      __syncthreads();
    }
    for (uint32_t i = tid; i < nc; i += NT) {
      const u64 mine = cand[i];
      uint32_t over = 0;
      for (uint32_t o = 0; o < nc; o++) over += cand[o] > mine ? 1u : 0u;
      if (over < k) best[over] = mine;
    }
    __syncthreads();
  }
  // the piece's sums, in the waves' order
  RowSums rs{m, 0.0f, 0.0f, 0.0f};
  uint32_t rk = 0;
#pragma unroll
  for (int i = 0; i < NW; i++) {
    rs.l += red[i][0];
    rs.w += red[i][1];
    rs.c += red[i][2];
    rk += redu[i];
  }
  if (S > 1) {
    uint32_t* out = a.part + (uint64_t)blockIdx.x * (kHead + 2 * k);
    if (tid == 0) {
      out[0] = __builtin_bit_cast(uint32_t, rs.m);
      out[1] = __builtin_bit_cast(uint32_t, rs.c);
      out[2] = __builtin_bit_cast(uint32_t, rs.l);
      out[3] = __builtin_bit_cast(uint32_t, rs.w);
      out[4] = rk;
    }
    if (tid < k) {
      out[kHead + 2 * tid] = (uint32_t)best[tid];
      out[kHead + 2 * tid + 1] = (uint32_t)(best[tid] >> 32);
    }
    return;
  }
  const float ls = rs.log_sum();
  if (tid == 0) {
    a.ent[r] = rs.entropy(ls);
    if (a.tok) {
      a.lp[r] = given ? rs.lp(xt, ls) : __builtin_nanf("");
      a.rank[r] = given ? rk : 0xFFFFFFFFu;
    }
  }
  if (tid < k) {
    a.top_tok[(uint64_t)r * k + tid] = 0xFFFFFFFFu - (uint32_t)best[tid];
    a.top_lp[(uint64_t)r * k + tid] = rs.lp(value_of((uint32_t)(best[tid] >> 32)), ls);
  }
}

// A row's pieces, a wave a row and a lane a piece: the sums brought to the
// row's maximum, and the alternatives out of the pieces' sorted keys: those
// that reach a bound, ranked in LDS, or, where LDS does not hold the lists or
// too many reach it, k rounds of a maximum over the lists' next ones (one row
// of 50021 logits, 20 alternatives: 12 us with the pieces, 17 by rounds).
template <typename T>
__global__ __launch_bounds__(64) void k_logprobs_join(LogprobArgs a, uint32_t S) {
  extern __shared__ u64 keys[];   // [S][k], where they are at most kJoinKeys
  const uint32_t r = blockIdx.x, lane = threadIdx.x, k = a.top;
  const uint32_t* p = a.part + ((uint64_t)r * S + lane) * (kHead + 2 * k);
  const bool in = lane < S;
  RowSums q{-INFINITY, 0.0f, 0.0f, 0.0f};
  uint32_t rk = 0;
  if (in) {
    q.m = __builtin_bit_cast(float, p[0]);
    q.c = __builtin_bit_cast(float, p[1]);
    q.l = __builtin_bit_cast(float, p[2]);
    q.w = __builtin_bit_cast(float, p[3]);
    rk = p[4];
  }
  const uint32_t tk = a.tok ? a.tok[r] : 0xFFFFFFFFu;
  const bool given = tk < a.vocab;
  const float xt = given ? (float)((const T*)a.logits + (uint64_t)r * a.ld)[tk] : 0.0f;
  RowSums t{wmax(q.m), 0.0f, 0.0f, 0.0f};
  // e^(x - M) = f e^(x - m), (x - M) = (x - m) + dm; a piece below the
  // maximum has no entry at it
  const float dm = fmaxf(q.m - t.m, -200.0f);
  const bool at = q.m == t.m, none = q.m == -INFINITY;
  const float f = none ? 0.0f : __expf(dm);   // (a NaN in l stays one)
  float s[3];
  s[0] = at ? q.c : 0.0f;
  s[1] = at ? q.l : f * (q.c + q.l);
  s[2] = at ? q.w : f * (q.w + dm * (q.c + q.l));
  wsum_n(s);
  t.c = s[0];
  t.l = s[1];
  t.w = s[2];
#pragma unroll
  for (int mk = 32; mk >= 1; mk >>= 1) rk += __shfl_xor(rk, mk, 64);
  const float ls = t.log_sum();
  if (lane == 0) {
    a.ent[r] = t.entropy(ls);
    if (a.tok) {
      a.lp[r] = given ? t.lp(xt, ls) : __builtin_nanf("");
      a.rank[r] = given ? rk : 0xFFFFFFFFu;
    }
  }
  auto pick = [&](u64 key, uint32_t i) {
    a.top_tok[(uint64_t)r * k + i] = 0xFFFFFFFFu - (uint32_t)key;
    a.top_lp[(uint64_t)r * k + i] = t.lp(value_of((uint32_t)(key >> 32)), ls);
  };
  const bool staged = S * k <= kJoinKeys;
  if (staged && k) {
    const uint32_t* row = a.part + (uint64_t)r * S * (kHead + 2 * k) + kHead;
    for (uint32_t i = lane; i < S * k; i += 64) {
      const uint32_t* q2 = row + (uint64_t)(i / k) * (kHead + 2 * k) + 2 * (i % k);
      keys[i] = (u64)q2[1] << 32 | q2[0];
    }
    __syncthreads();
    // Of the pieces' d-th keys the m-th largest is one that m d of them reach,
    // k at least; m about three quarters of the pieces makes it a close one (a piece of
    // fewer keys has zeros behind them)
    const uint32_t d = (4 * k + 3 * S - 1) / (3 * S), m = (k + d - 1) / d;
    const u64 own = in ? keys[lane * k + d - 1] : 0;
    uint32_t above = 0;
    for (uint32_t o = 0; o < S; o++) above += keys[o * k + d - 1] > own ? 1u : 0u;
    const u64 bound = max(1ull, ~wave_max64(in && above < m ? ~own : 0ull));
    uint32_t nc = 0;
    for (uint32_t i = lane; i - lane < S * k; i += 64) nc += __popcll(__ballot(i < S * k && keys[i] >= bound));
    if (nc <= kJoinRank) {
      // those move to the front (never past what was read), and each counts
      // the ones above it
      nc = 0;
      for (uint32_t i = lane; i - lane < S * k; i += 64) {
        const u64 q2 = i < S * k ? keys[i] : 0;
        const unsigned long long on = __ballot(q2 >= bound);
        if (q2 >= bound) keys[nc + __popcll(on & ((1ull << lane) - 1))] = q2;
        nc += __popcll(on);
        __syncthreads();
      }
      for (uint32_t i = lane; i < nc; i += 64) {
        const u64 mine = keys[i];
        uint32_t over = 0;
#pragma unroll 4
        for (uint32_t o = 0; o < nc; o++) over += keys[o] > mine ? 1u : 0u;
        if (over < k) pick(mine, over);
      }
      return;
    }
  }
  uint32_t at_i = 0;
  auto next = [&]() -> u64 {
    if (!in || at_i >= k) return 0ull;
    return staged ? keys[lane * k + at_i] : (u64)p[kHead + 2 * at_i + 1] << 32 | p[kHead + 2 * at_i];
  };
  u64 mine = k ? next() : 0;
  for (uint32_t i = 0; i < k; i++) {
    const u64 b = wave_max64(mine);
    if (mine == b) {
      pick(b, i);
      at_i++;
      mine = next();
    }
  }
}

// How a row is cut. Whole rows of up to 32768 logits in one launch of 1024
// threads (512 rows of 32768 f32 logits take 20 us so, 30 in pieces of 8192
// with the join). Longer ones in pieces of 256 threads, of which a CU holds
// eight: each thread has up to eight vectors, and the pieces are as many as
// leave the fewest places empty (3000 rows of 50021 bf16 logits: 104 us in
// seven pieces of 3.5 vectors a thread, 98 in five of 4.9). Pieces of 32768
// where those would be too many for one wave to join.
struct Plan {
  uint32_t C, S;
  bool wide;   // 1024 threads and up to 32768 logits a workgroup, else 256
};
// (es: an element's bytes)
Plan plan_of(uint32_t vocab, uint32_t es) {
  const uint32_t step = 256 * 16 / es, cap = 8 * step;   // logits of a vector a thread, of eight
  Plan p;
  p.wide = (vocab > cap && vocab <= 32768) || vocab > 64 * cap;
  const uint32_t most = p.wide ? 32768u : cap;
  p.S = (vocab + most - 1) / most;
  if (!p.wide && p.S > 1) {
    // a piece's own work is about that of half a vector a thread
    uint32_t best = ~0u;
    for (uint32_t s = p.S, n = p.S; s <= std::min(2 * n, 64u); s++) {
      const uint32_t cost = s * (2 * ((vocab + s * step - 1) / (s * step)) + 1);
      if (cost < best) {
        best = cost;
        p.S = s;
      }
    }
  }
  p.C = ((vocab + p.S - 1) / p.S + 7) & ~7u;
  p.S = (vocab + p.C - 1) / p.C;
  return p;
}

}  // namespace

uint64_t logprobs_part_words(uint32_t n, uint32_t vocab, uint32_t top) {
  // (for either size of element)
  const uint32_t S = std::max(plan_of(vocab, 2).S, plan_of(vocab, 4).S);
  return S > 1 ? (uint64_t)n * S * (kHead + 2 * top) : 0;
}

uint32_t logprobs_max_rows(uint32_t vocab) {
  uint64_t most = 0;   // threads a row, of either size of element
  for (uint32_t es : {2u, 4u}) {
    const Plan p = plan_of(vocab, es);
    most = std::max<uint64_t>(most, p.S * (p.wide ? 1024u : 256u));
  }
  return (uint32_t)(0xFFFFFFFFull / most);
}

hipError_t launch_logprobs(const LogprobArgs& a, int type, hipStream_t st) {
  if (!a.logits || a.vocab == 0 || a.vocab > kLpMaxVocab || a.top > kLpMaxTop || a.top > a.vocab || a.ld < a.vocab || !a.ent)
    return hipErrorInvalidValue;
  if (a.n == 0) return hipSuccess;
  const Plan p = plan_of(a.vocab, type == ET_F32 ? 4 : 2);
  if ((p.S > 1 && !a.part) || a.n > logprobs_max_rows(a.vocab)) return hipErrorInvalidValue;
  auto go = [&](auto t) -> hipError_t {
    using T = decltype(t);
    constexpr int W = 16 / sizeof(T);
    const dim3 g(a.n * p.S);
    if (p.wide)
      hipLaunchKernelGGL((k_logprobs<T, 1024, 32 / W>), g, dim3(1024), 0, st, a, p.C, p.S);
    else
      hipLaunchKernelGGL((k_logprobs<T, 256, 8>), g, dim3(256), 0, st, a, p.C, p.S);
    const uint32_t keys = p.S * a.top;
    if (p.S > 1)
      hipLaunchKernelGGL((k_logprobs_join<T>), dim3(a.n), dim3(64), keys <= kJoinKeys ? keys * 8 : 0, st, a, p.S);
    return hipGetLastError();
  };
  switch (type) {
    case ET_F32: return go(float{});
    case ET_BF16: return go(__bf16{});
    case ET_F16: return go(_Float16{});
    default: return hipErrorInvalidValue;
  }
}

}  // namespace ana
