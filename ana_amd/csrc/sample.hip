// A token of each row of logits from a given random number, with a
// temperature, top-k, top-p and min-p (gfx950).
//
// Logits stand in order by value, then the lower index. With m the largest, a
// token weighs w = e^((x - m) / t). Kept are the first k; of these, as many
// as it takes to reach p of their mass; of these, the ones that weigh q or
// more. All three leave a beginning of the order, so what is kept is a mass C
// of it, and the token for u is where the running mass passes u C.
//
// A border that falls a hair to either side is another token, so masses are
// exact: a weight (a series of 2^x in 64 bits, right to 1e-12) is rounded
// once, to a multiple of 2^-42, and whole numbers add up the same in any
// order, on any number of threads. A weight below 2^-43 is 0.
//
// A workgroup takes a row. One pass finds the largest, the next puts every
// token's mass into one of 2048 bins of a 47th of an octave, likeliest first
// (43.6 octaves: all that has a mass). Where a running mass is reached is
// then a bin, whose few tokens go to LDS and are told apart there; the
// likeliest 300 or so have been noted on the way, so that a nucleus of
// few tokens needs no pass more. A top-k of up to 256 needs no masses but its
// own: the k-th largest of 64 group maxima is a bound that at least k logits
// reach and few more do, and the least of them one that some 300 reach, k
// among them mostly.
//
// Each pass reads the row again, from the caches mostly: a row held in
// registers (64 of them for 32768 f32 logits, 512 threads) leaves too few for
// the code, which then waits for what it has put aside: 97 us for 512 rows
// with a nucleus, 57 so.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "mfma.h"
#include "order.h"
#include "sample.h"
#include "wave.h"

namespace ana {

namespace {

constexpr uint32_t kPartBits = 9, NT = 1 << kPartBits, NW = NT / 64;
constexpr uint32_t kBins = kSampleBins, kBinsOctave = 47, BT = kBins / NT;   // (BT: bins a thread)
constexpr uint32_t kList = NT;     // tokens that LDS takes, one a thread
constexpr uint32_t kWave = 64;     // of them, a wave's
constexpr uint32_t kFew = 64;      // those that one wave tells apart
constexpr uint32_t kTop = 256;     // a top-k that is looked for among the likeliest alone
constexpr double kUnit = 0x1p-42;  // of a mass
static_assert(kBins == 4 * NT && kBins / kBinsOctave >= 43, "all that has a mass is in a bin");

typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));

// 2^x of four x from -64 to 0: a series on half an octave about 0, relative
// error 8e-13 (each coefficient by iteration for the least largest error). x +
// 3 2^51 has the nearest whole number in its low word. The four chains go side
// by side, in one block with the coefficients in scalar registers: the
// compiler takes a move of each and an instruction that adds to its own
// operand.
__device__ __forceinline__ void exp2_of(const double (&x)[4], double (&w)[4]) {
  constexpr double magic = 0x1.8p52;
  double a[4], f[4], s[4];
#pragma unroll
  for (int i = 0; i < 4; i++) {
    a[i] = x[i] + magic;
    f[i] = x[i] - (a[i] - magic);
  }
#define ANA_ROW(c)                    \
  "v_fma_f64 %0, %4, %0, " c "\n\t"   \
  "v_fma_f64 %1, %5, %1, " c "\n\t"   \
  "v_fma_f64 %2, %6, %2, " c "\n\t"   \
  "v_fma_f64 %3, %7, %3, " c "\n\t"
  asm("v_fma_f64 %0, %4, %8, %9\n\t"
      "v_fma_f64 %1, %5, %8, %9\n\t"
      "v_fma_f64 %2, %6, %8, %9\n\t"
      "v_fma_f64 %3, %7, %8, %9\n\t"
      ANA_ROW("%10") ANA_ROW("%11") ANA_ROW("%12") ANA_ROW("%13") ANA_ROW("%14") ANA_ROW("%15")
      : "=&v"(s[0]), "=&v"(s[1]), "=&v"(s[2]), "=&v"(s[3])
      : "v"(f[0]), "v"(f[1]), "v"(f[2]), "v"(f[3]), "v"(0x1.61c4f09d828bap-20), "s"(0x1.00d8535005e2dp-16),
        "s"(0x1.430aa88338cf8p-13), "s"(0x1.5d874d06e4851p-10), "s"(0x1.3b2ab5ed6f3f2p-7), "s"(0x1.c6b08dced3710p-5),
        "s"(0x1.ebfbdff8ede8fp-3), "s"(0x1.62e42fef89d1dp-1));
#undef ANA_ROW
#pragma unroll
  for (int i = 0; i < 4; i++) {
    u32x2_t y = __builtin_bit_cast(u32x2_t, fma(f[i], s[i], 1.0));
    y[1] += __builtin_bit_cast(u32x2_t, a[i])[0] << 20;
    w[i] = __builtin_bit_cast(double, y);
  }
}
// a weight (0 .. 1) in units: the sum with 2^10 has steps of one
__device__ __forceinline__ u64 units_of(double w) {
  u32x2_t n = __builtin_bit_cast(u32x2_t, w + 1024.0);
  n[1] -= 0x40900000u;   // (1024's own bits)
  return __builtin_bit_cast(u64, n);
}

// v's inclusive sum over the lanes up to this one, by DPP moves: within rows of
// 16, then the rows' last lanes into the rows after them
template <int CTRL, int ROWS>
__device__ __forceinline__ u64 dpp_64(u64 v) {
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)v, CTRL, ROWS, 0xF, false);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(v >> 32), CTRL, ROWS, 0xF, false);
  return (u64)hi << 32 | lo;
}
__device__ __forceinline__ u64 wave_scan(u64 v) {
  v += dpp_64<0x111, 0xF>(v);
  v += dpp_64<0x112, 0xF>(v);
  v += dpp_64<0x114, 0xF>(v);
  v += dpp_64<0x118, 0xF>(v);
  v += dpp_64<0x142, 0xA>(v);
  v += dpp_64<0x143, 0xC>(v);
  return v;
}
__device__ __forceinline__ u64 lane_64(u64 v, uint32_t l) {
  return (u64)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(v >> 32), l) << 32 |
         (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, l);
}

// a value that all lanes have, in scalar registers
__device__ __forceinline__ uint32_t uni(uint32_t v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ float uni(float v) { return __builtin_bit_cast(float, uni(__builtin_bit_cast(uint32_t, v))); }
__device__ __forceinline__ u64 uni(u64 v) { return (u64)uni((uint32_t)(v >> 32)) << 32 | uni((uint32_t)v); }
__device__ __forceinline__ double uni(double v) { return __builtin_bit_cast(double, uni(__builtin_bit_cast(u64, v))); }

// the mass to reach for a number (others than 0 .. 1 count as the nearest): 1 .. C
__device__ __forceinline__ u64 draw_of(float u, u64 C) {
  const double x = (double)fminf(fmaxf(u, 0.0f), 1.0f) * (double)C;
  return x >= (double)C ? C : min(C, (u64)x + 1);
}
// and for a share of S: 1 .. S
__device__ __forceinline__ u64 share_of(float p, u64 S) {
  const double y = __builtin_ceil((double)p * (double)S);
  return y >= (double)S ? S : max(1ull, (u64)y);
}

// What a launch does: whole rows (kWhole), or, where rows are few and long, a
// row in S pieces: their group maxima, then their masses, to `part`, then the
// tokens of the bins that the nucleus' end and the draw can be in, and the rest
// by one workgroup, which goes over those alone (or over the row, where they are
// more than there is room for, or a top-k is asked for). (Four rows of 200003 f32
// with a nucleus: 31 us; 116 when that workgroup went over the row itself, each
// time 10 us. The lambdas that take others are inlined by force: one that is
// not puts all they refer to in memory, 59 us.)
enum Step { kWhole, kMax, kMass, kGather, kRest };

template <typename T, Step STEP>
__global__ __launch_bounds__(NT) __attribute__((amdgpu_waves_per_eu(STEP == kRest ? 2 : 4))) void k_sample(SampleArgs a, uint32_t S, uint32_t piece) {
  constexpr uint32_t W = 16 / sizeof(T);
  typedef T vec_t __attribute__((ext_vector_type(W)));
  // (a row may start on any element's border)
  typedef vec_t vec_any __attribute__((aligned(sizeof(T))));
  // (hist: after the bins a place a lane for what has none)
  __shared__ u64 hist[kBins + 64], sub[NT], list[kList];
  __shared__ float tmax[NW][64];
  __shared__ u64 wsum[NW];
  __shared__ uint32_t nlist, bin_s, bin2_s[2], found[NW];
  __shared__ u64 before_s, key_s, incl_s, lo_s, hi_s;
  const uint32_t tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
  constexpr bool kPiece = STEP == kMax || STEP == kMass || STEP == kGather;
  const uint32_t r = kPiece ? blockIdx.x / S : blockIdx.x;
  // the elements e0 .. of the row that this workgroup looks at
  const uint32_t e0 = kPiece ? (blockIdx.x % S) * piece : 0;
  const uint32_t cnt_e = kPiece ? min(piece, a.vocab - e0) : a.vocab;
  const T* row = (const T*)a.logits + (uint64_t)r * a.ld + e0;
  const float t = a.ts ? a.ts[r] : a.t, p = a.ps ? a.ps[r] : a.p, q_ = a.qs ? a.qs[r] : a.q;
  const float q = q_ > 0.0f ? fminf(q_, 1.0f) : 0.0f;   // (above 1 is 1: what is as likely as the first stays; NaN is 0)
  const uint32_t k_ = a.ks ? a.ks[r] : a.k, k = k_ < a.vocab ? k_ : 0;   // (0: all)
  const uint32_t nvec = cnt_e / W;
  u64* const ghist = a.part + (uint64_t)r * sample_part_words(S);   // a split row's words
  float* const gmaxs = (float*)(ghist + kBins + 2);
  u64* const gtok = ghist + kBins + 2 + 32 * S;

  bool inf = false;   // +inf is the largest: those are alike, the others nothing
  auto load = [&](uint32_t v) {
    vec_t y;
    if (v < nvec) {
      y = *reinterpret_cast<const vec_any*>(row + (uint64_t)v * W);
    } else {
#pragma unroll
      for (uint32_t e = 0; e < W; e++) y[e] = (T)-INFINITY;
    }
    if (inf) {
#pragma unroll
      for (uint32_t e = 0; e < W; e++) y[e] = (float)y[e] == INFINITY ? (T)0.0f : (T)-INFINITY;
    }
    return y;
  };
  // the elements after the last whole vector, one each for the first threads
  const uint32_t ie = nvec * W + tid;
  float xe = ie < cnt_e ? (float)row[ie] : -INFINITY;
  uint32_t ntok = ~0u;   // the gathered tokens, where those do for the row
  // f(values, their indices) over the thread's share in groups of four, U
  // vectors of loads at a time; places without a logit hold -inf
  auto each = [&](auto vecs, auto&& f) __attribute__((always_inline)) {
    constexpr uint32_t U = decltype(vecs)::value;
    if constexpr (STEP == kRest) {
      if (ntok != ~0u) {
#pragma unroll 1
        for (uint32_t i = tid; i - tid < ntok; i += 4 * NT) {
          u64 key[4];
          float v[4];
#pragma unroll
          for (uint32_t e = 0; e < 4; e++) key[e] = i + e * NT < ntok ? gtok[i + e * NT] : 0;
#pragma unroll
          for (uint32_t e = 0; e < 4; e++) v[e] = key[e] ? value_of((uint32_t)(key[e] >> 32)) : -INFINITY;
          f(v, [&](uint32_t e) {
            return 0xFFFFFFFFu - (uint32_t)(e == 0 ? key[0] : e == 1 ? key[1] : e == 2 ? key[2] : key[3]);
          });
        }
        return;
      }
    }
#pragma unroll 1
    for (uint32_t i = tid; i - tid < nvec; i += U * NT) {
      vec_t y[U];
#pragma unroll
      for (uint32_t u = 0; u < U; u++) y[u] = load(i + u * NT);
#pragma unroll
      for (uint32_t u = 0; u < U; u++) {
#pragma unroll
        for (uint32_t e = 0; e < W; e += 4) {
          const float v[4] = {(float)y[u][e], (float)y[u][e + 1], (float)y[u][e + 2], (float)y[u][e + 3]};
          const uint32_t at = e0 + (i + u * NT) * W + e;
          f(v, [at](uint32_t o) { return at + o; });
        }
      }
    }
    const float v[4] = {xe, -INFINITY, -INFINITY, -INFINITY};
    f(v, [&](uint32_t o) { return e0 + ie + o; });
  };
  constexpr std::integral_constant<uint32_t, 2> two{};
  constexpr std::integral_constant<uint32_t, 8 * sizeof(T) / 4> many{};   // (for passes that do little)
  constexpr std::integral_constant<uint32_t, STEP == kRest ? 8 * sizeof(T) / 4 : 2> noting{};   // (alone on its CU)
  auto answer = [&](u64 key, float lp) {
    a.tok[r] = 0xFFFFFFFFu - (uint32_t)key;
    a.lp[r] = lp;
  };

  // ---- the largest; gm: of group l (lane l of every wave)
  float gm = -INFINITY;
  if constexpr (STEP == kWhole || STEP == kMax) {
    float m = -INFINITY;
    each(many, [&](const float (&v)[4], auto) { m = fmaxf(m, fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3]))); });
    tmax[wv][lane] = m;
    __syncthreads();
    gm = tmax[0][lane];
#pragma unroll
    for (uint32_t i = 1; i < NW; i++) gm = fmaxf(gm, tmax[i][lane]);
  } else {
#pragma unroll 4
    for (uint32_t i = 0; i < S; i++) gm = fmaxf(gm, gmaxs[i * 64 + lane]);
  }
  if constexpr (STEP == kMax) {
    if (wv == 0) gmaxs[(blockIdx.x % S) * 64 + lane] = gm;
    // (and the masses' places cleared for the next step)
    for (uint32_t i = (blockIdx.x % S) * NT + tid; i < kBins + 2; i += S * NT) ghist[i] = 0;
    return;
  }
  float m = wmax(gm);
  if (m == -INFINITY) {   // no number above it
    if (!kPiece && tid == 0) answer(~0ull << 32, __builtin_nanf(""));
    return;
  }
  if (m == INFINITY) {
    inf = true;
    xe = xe == INFINITY ? 0.0f : -INFINITY;
    gm = gm == INFINITY ? 0.0f : -INFINITY;
    m = 0.0f;
  }
  const bool greedy = !(t > 0.0f) || k == 1, short_k = k && k <= kTop;
  if ((STEP == kMass || STEP == kGather) && (greedy || k)) return;   // (those rows need none, or not all)
  if (greedy) {
    uint32_t at = ~0u;
    each(many, [&](const float (&v)[4], auto i) {
#pragma unroll
      for (int e = 0; e < 4; e++) at = v[e] == m ? min(at, i(e)) : at;
    });
#pragma unroll
    for (int s = 32; s >= 1; s >>= 1) at = min(at, (uint32_t)__shfl_xor(at, s, 64));
    if (lane == 0) wsum[wv] = at;
    __syncthreads();
    if (tid == 0) {
      for (uint32_t i = 1; i < NW; i++) at = min(at, (uint32_t)wsum[i]);
      answer(0xFFFFFFFFull - at, 0.0f);
    }
    return;
  }

  const double c = uni(1.4426950408889634 / (double)t), md = uni((double)m);
  // below it a weight is less than 2^-43
  const float light = uni((float)(md - 44.0 / c));
  // A temperature below 2^-121: bins as narrow as f32 makes them hold weights
  // below 2^-1022 too, which exp2_of does not take.
  const bool steep = c * kBinsOctave > 3.0e38;
  auto weights = [&](const float (&v)[4], double (&w)[4]) {
    const double z[4] = {((double)v[0] - md) * c, ((double)v[1] - md) * c, ((double)v[2] - md) * c, ((double)v[3] - md) * c};
    exp2_of(z, w);
    if (steep) {
#pragma unroll
      for (int e = 0; e < 4; e++) w[e] = v[e] >= light ? w[e] : 0.0;
    }
  };
  auto weight = [&](float v) {
    const double z = __builtin_fmax(((double)v - md) * c, -64.0), four[4] = {z, z, z, z};   // (-64 for a NaN)
    double w[4];
    exp2_of(four, w);
    return w[0];
  };
  auto value = [](u64 key) { return value_of((uint32_t)(key >> 32)); };
  // (the logarithm of its own share, from the logit)
  auto lp_of = [&](u64 key, u64 C) { return (float)(((double)value(key) - md) / (double)t - log((double)C * kUnit)); };
  const bool nucleus = p < 1.0f;

  // A token with yes (for all lanes at once) to the list: a wave's to its own
  // 64 places, counted in a scalar (an LDS counter's answer takes as long as 20
  // tokens).
  auto note = [&](bool yes, u64 key, uint32_t& cnt) {
    const unsigned long long mask = __ballot(yes);
    const uint32_t at = cnt + __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
    if (yes && at < kWave) list[wv * kWave + at] = key;
    cnt += __popcll(mask);
  };
  // of four, those that in(value) (the cheap test, which most fail) and keep(key) hold for
  auto note_four = [&](const float (&v)[4], auto&& i, auto&& in, auto&& keep, uint32_t& cnt) __attribute__((always_inline)) {
    unsigned long long on[4];
#pragma unroll
    for (int e = 0; e < 4; e++) on[e] = __ballot(in(v[e]));
    if (!(on[0] | on[1] | on[2] | on[3])) return;
#pragma unroll
    for (int e = 0; e < 4; e++) {
      if (!on[e]) continue;
      const u64 key = key_of(v[e], i(e));
      note((on[e] >> lane & 1) && v[e] > -INFINITY && keep(key), key, cnt);
    }
  };
  // how many all waves found: more than the list takes, where one has left some out
  auto count_all = [&](uint32_t cnt) {
    __syncthreads();
    if (lane == 0) found[wv] = cnt;
    __syncthreads();
    uint32_t sum = 0, most = 0;
#pragma unroll
    for (uint32_t i = 0; i < NW; i++) {
      sum += found[i];
      most = max(most, found[i]);
    }
    return uni(most <= kWave ? sum : kList + 1);
  };
  // key (of the threads with `in`) together at the list's start, in no order
  auto close_up = [&](bool in, u64 key) {
    __syncthreads();
    const unsigned long long mask = __ballot(in);
    if (lane == 0) found[wv] = __popcll(mask);
    __syncthreads();
    uint32_t at = 0, all = 0;
#pragma unroll
    for (uint32_t i = 0; i < NW; i++) {
      at += i < wv ? found[i] : 0;
      all += found[i];
    }
    if (in) list[at + __popcll(mask & ((1ull << lane) - 1))] = key;
    __syncthreads();
    return uni(all);
  };

  // the sum over the threads up to this one, and of all
  auto scan = [&](u64 v, u64* total) {
    v = wave_scan(v);
    __syncthreads();
    if (lane == 63) wsum[wv] = v;
    __syncthreads();
    u64 base = 0, all = 0;
#pragma unroll
    for (uint32_t i = 0; i < NW; i++) {
      const u64 s = wsum[i];
      if (i < wv) base += s;
      all += s;
    }
    *total = uni(all);
    return base + v;
  };

  if (short_k) {
    // the k-th largest group maximum, or the least: the least that fewer than k are above
    uint32_t above = 0;
#pragma unroll 4
    for (int i = 0; i < 64; i++) above += lane_f(gm, i) > gm;
    const float bound = uni(-wmax(above < k ? -gm : -INFINITY));
    uint32_t cnt = 0;
    each(noting, [&](const float (&v)[4], auto i) {
      note_four(v, i, [&](float x) { return x >= bound; }, [](u64) { return true; }, cnt);
    });
    const uint32_t nc = count_all(cnt);
    if (nc <= kList && (nc >= k || bound == -INFINITY)) {
      close_up(lane < cnt, lane < cnt ? list[tid] : 0);
      if (tid < nc) {
        const u64 mine = list[tid];
        uint32_t over = 0;
#pragma unroll 4
        for (uint32_t o = 0; o < nc; o++) over += list[o] > mine ? 1u : 0u;
        if (over < k) sub[over] = mine;
      }
      __syncthreads();
      const bool in = tid < min(k, nc);
      const u64 key = in ? sub[tid] : 0;
      const double wd = in ? weight(value(key)) : 0.0;
      const u64 w = units_of(wd);
      if (k <= 64) {
        if (wv) return;
        const u64 incl = wave_scan(w), sum = lane_64(incl, 63);
        const bool keep = in && (!nucleus || lane == 0 || incl - w < share_of(p, sum)) && (wd >= (double)q || lane == 0);
        const uint32_t last = 63 - __clzll(__ballot(keep));
        const u64 C = lane_64(incl, last), want = draw_of(a.u[r], C);
        if (incl >= want && incl - w < want) answer(key, lp_of(key, C));
        return;
      }
      u64 sum;
      const u64 incl = scan(w, &sum);
      // (what is kept is a beginning: its last token's sum is the largest)
      const bool keep = in && (!nucleus || tid == 0 || incl - w < share_of(p, sum)) && (wd >= (double)q || tid == 0);
      if (tid == 0) hi_s = 0;
      __syncthreads();
      if (keep) atomicMax(&hi_s, incl);
      __syncthreads();
      const u64 C = uni(hi_s), want = draw_of(a.u[r], C);
      if (in && incl >= want && incl - w < want) answer(key, lp_of(key, C));
      return;
    }
    __syncthreads();
  }

  // ---- the masses of all
  const float cb = uni(fminf((float)(c * kBinsOctave), 3.0e38f));
  // Where a logit is, in bins; what has no mass is past them (a NaN too), at a
  // place of its lane's, so that few meet there.
  const float none = (float)(kBins + lane);
  auto place_of = [&](float v) { return fminf((m - v) * cb, none); };
  u64 cut = 0;   // keys below it are out (top-k)

  // hist as running sums
  auto run_up = [&]() -> u64 {
    __syncthreads();
    u64 h[BT], all;
#pragma unroll
    for (uint32_t i = 0; i < BT; i++) h[i] = hist[BT * tid + i] + (i ? h[i - 1] : 0);
    const u64 below = scan(h[BT - 1], &all) - h[BT - 1];
#pragma unroll
    for (uint32_t i = 0; i < BT; i++) hist[BT * tid + i] = below + h[i];
    __syncthreads();
    return all;
  };
  auto clear = [&]() {
#pragma unroll
    for (uint32_t i = 0; i < BT; i++) hist[i * NT + tid] = 0;
    __syncthreads();
  };
  // f(bin) by the thread of the one that a running sum reaches R in
  auto reaching = [&](u64 R, auto&& f) {
#pragma unroll
    for (uint32_t i = 0; i < BT; i++) {
      const uint32_t b = BT * tid + i;
      if ((b ? hist[b - 1] : 0) < R && R <= hist[b]) f(b);
    }
  };

  // What the list holds: every token of bins below `top`, or of the bins b0, b1
  // .. b2; each wave's first `cnt` places.
  uint32_t top = 0, b0 = kBins, b1 = kBins, b2 = 0, cnt = 0;
  bool counts = k != 0;   // (the running sums are of tokens, not of masses)
  auto val = [&](float v) -> u64 { return counts ? 1 : units_of(weight(v)); };
  auto of_bins = [&](float v, uint32_t lo, uint32_t hi) {
    const float y = (m - v) * cb;
    return y >= (float)lo && y < (float)(hi + 1);
  };
  // The key at which the running sum reaches R (1 .. the sum of all), and the
  // sum up to it. also0, also1: sums that will be asked for next.
  auto find = [&](u64 R, u64 also0, u64 also1, u64* incl) __attribute__((always_inline)) -> u64 {
    reaching(R, [&](uint32_t i) { bin_s = i; });
    if (also0) {
      reaching(also0, [&](uint32_t i) { bin2_s[0] = i; });
      reaching(also1, [&](uint32_t i) { bin2_s[1] = i; });
    }
    sub[tid] = 0;
    __syncthreads();
    const uint32_t b = uni(bin_s);
    u64 before = b ? uni(hist[b - 1]) : 0, lo = cut, hi = ~0ull;
    float y0 = (float)b, y1 = (float)(b + 1);   // where the key is, in bins
    auto here = [&](float v) {
      const float y = (m - v) * cb;
      return y >= y0 && y < y1;
    };
    auto of_keys = [&](u64 key) { return key >= lo && key <= hi; };
    // the part of `sub` that the sum reaches R in
    auto part_of = [&]() -> uint32_t {
      __syncthreads();
      const u64 mine = sub[tid];
      u64 all;
      const u64 up = before + scan(mine, &all);
      if (up - mine < R && R <= up) {
        bin_s = tid;
        before_s = up - mine;
      }
      if (tid == 0) nlist = 0;
      __syncthreads();
      before = uni(before_s);
      return uni(bin_s);
    };
    // a bin's NT parts: the next bits of what chose it
    auto part_at = [&](float v) { return (uint32_t)(place_of(v) * NT) & (NT - 1); };
    uint32_t nc;
    bool spread = false;   // the list is the waves' own places yet
    if (b < top || b == b0 || (b >= b1 && b <= b2)) {
      spread = true;
      nc = kList;   // (at most)
    } else {
      top = b2 = 0;
      b0 = b1 = kBins;
      // a bin's tokens weigh about the same: how many there are in i .. j
      auto about = [&](uint32_t i, uint32_t j) {
        const float own = (float)(uni(hist[j]) - (i ? uni(hist[i - 1]) : 0));
        return counts ? own : own * (float)kUnit * exp2f((float)j / kBinsOctave);
      };
      if (about(b, b) > kList * 0.6f) {
        // more than the list takes: its parts' sums first
        each(two, [&](const float (&v)[4], auto i) {
          if (!__any(here(v[0]) || here(v[1]) || here(v[2]) || here(v[3]))) return;
          double w[4] = {};
          if (!counts) weights(v, w);
#pragma unroll
          for (int e = 0; e < 4; e++)
            if (here(v[e]) && key_of(v[e], i(e)) >= cut) atomicAdd(&sub[part_at(v[e])], counts ? 1 : units_of(w[e]));
        });
        const uint32_t part = part_of();
        y0 = (float)b + (float)part / NT;
        y1 = (float)b + (float)(part + 1) / NT;
        cnt = 0;
        each(noting, [&](const float (&v)[4], auto i) { note_four(v, i, here, of_keys, cnt); });
        nc = count_all(cnt);
        if (nc <= kList) nc = close_up(lane < cnt, lane < cnt ? list[tid] : 0);
      } else {
        b0 = b;
        if (also0) {
          const uint32_t i = uni(bin2_s[0]), j = uni(bin2_s[1]);
          if (about(b, b) + about(i, j) <= kList * 0.6f) {
            b1 = i;
            b2 = j;
          }
        }
        cnt = 0;
        each(noting, [&](const float (&v)[4], auto i) {
          note_four(v, i, [&](float x) { return here(x) || of_bins(x, b1, b2); }, of_keys, cnt);
        });
        nc = count_all(cnt);
        spread = nc <= kList;
        if (!spread) {
          b0 = b1 = kBins;
          b2 = 0;
        }
      }
    }
    u64 mine = 0;
    if (spread) {
      // its own tokens of the list; what else is there stays for the next
      mine = lane < cnt ? list[tid] : 0;
      const bool in = lane < cnt && here(value(mine)) && of_keys(mine);
      const unsigned long long mask = __ballot(in);
      __syncthreads();
      if (lane == 0) found[wv] = __popcll(mask);
      __syncthreads();
      nc = 0;
#pragma unroll
      for (uint32_t i = 0; i < NW; i++) nc += found[i];
      nc = uni(nc);
      bool go = in;
      if (nc > kFew) {
        const uint32_t at = in ? part_at(value(mine)) : 0;
        if (in) atomicAdd(&sub[at], val(value(mine)));
        const uint32_t part = part_of();
        go = in && at == part;
      } else {
        if (tid == 0) nlist = 0;
        __syncthreads();
      }
      // (few: to `sub`, which is done with)
      __syncthreads();
      if (go) sub[atomicAdd(&nlist, 1u)] = mine;
      __syncthreads();
      nc = uni(nlist);
    }
    // The keys of `members` into NT parts, the highest first: the part that the
    // sum reaches R in (its keys are lo .. hi then).
    auto narrow = [&](u64 least, u64 most, auto&& members) __attribute__((always_inline)) {
      // the extent of the members' keys
#pragma unroll
      for (int s = 32; s >= 1; s >>= 1) {
        least = min(least, __shfl_xor(least, s, 64));
        most = max(most, __shfl_xor(most, s, 64));
      }
      __syncthreads();
      if (tid == 0) {
        lo_s = ~0ull;
        hi_s = 0;
      }
      sub[tid] = 0;
      __syncthreads();
      if (lane == 0) {
        atomicMin(&lo_s, least);
        atomicMax(&hi_s, most);
      }
      __syncthreads();
      least = uni(lo_s);
      most = uni(hi_s);
      const uint32_t bits = 64 - __clzll((long long)(most - least)), shift = bits > kPartBits ? bits - kPartBits : 0;
      members([&](u64 key) { atomicAdd(&sub[(most - key) >> shift], val(value(key))); });
      const u64 part = part_of();
      hi = most - (part << shift);
      const u64 width = (1ull << shift) - 1;
      lo = hi - least > width ? hi - width : least;
    };
    // (more of one value than the list takes)
#pragma unroll 1
    while (nc > kList) {
      u64 least = ~0ull, most = 0;
      auto each_key = [&](auto&& f) __attribute__((always_inline)) {
        each(two, [&](const float (&v)[4], auto i) {
#pragma unroll 1
          for (uint32_t e = 0; e < 4; e++) {
            const float x = e == 0 ? v[0] : e == 1 ? v[1] : e == 2 ? v[2] : v[3];
            const u64 key = key_of(x, i(e));
            if (here(x) && x > -INFINITY && of_keys(key)) f(key);
          }
        });
      };
      each_key([&](u64 key) {
        least = min(least, key);
        most = max(most, key);
      });
      narrow(least, most, each_key);
      cnt = 0;
      each(noting, [&](const float (&v)[4], auto i) { note_four(v, i, here, of_keys, cnt); });
      nc = count_all(cnt);
      if (nc <= kList) nc = close_up(lane < cnt, lane < cnt ? list[tid] : 0);
    }
    u64* const at = spread ? sub : list;
#pragma unroll 1
    while (nc > kFew) {
      const bool in = tid < nc;
      const u64 key = in ? at[tid] : 0;
      narrow(in ? key : ~0ull, key, [&](auto&& f) {
        if (in) f(key);
      });
      __syncthreads();
      if (in && of_keys(key)) at[atomicAdd(&nlist, 1u)] = key;
      __syncthreads();
      nc = uni(nlist);
    }
    if (wv == 0) {
      const bool in = lane < nc;
      const u64 key = in ? at[lane] : 0, w = in ? val(value(key)) : 0;
      u64 up = before + w;
      for (uint32_t o = 0; o < nc; o++) up += lane_64(key, o) > key ? lane_64(w, o) : 0;
      if (in && up >= R && up - w < R) {
        key_s = key;
        incl_s = up;
      }
    }
    __syncthreads();
    *incl = uni(incl_s);
    return uni(key_s);
  };

  u64 sq = 0;   // the mass of those of weight q or more
  const double qd = uni((double)q);
  auto masses = [&](auto all) __attribute__((always_inline)) {
    // (the least group maximum: some 300 reach it; no list is kept of pieces)
    const float likely = STEP == kWhole ? uni(-wmax(-gm)) : INFINITY;
    cnt = 0;
    each(two, [&](const float (&v)[4], auto i) {
      if (!__any(fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])) >= light)) return;
      double w[4];
      weights(v, w);
#pragma unroll
      for (int e = 0; e < 4; e++) {
        if constexpr (!decltype(all)::value) w[e] = key_of(v[e], i(e)) >= cut ? w[e] : 0.0;
        // (past the bins w is anything, and no one looks)
        atomicAdd(&hist[(uint32_t)place_of(v[e])], units_of(w[e]));
      }
      if (qd > 0.0) {
#pragma unroll
        for (int e = 0; e < 4; e++) sq += w[e] >= qd && place_of(v[e]) < (float)kBins ? units_of(w[e]) : 0;
      }
      if constexpr (STEP == kWhole) note_four(v, i, [&](float x) { return x >= likely; }, [](u64) { return true; }, cnt);
    });
    // whole bins above it are in the list, if that took them (all, where a group has none)
    if (STEP == kWhole && count_all(cnt) <= kList) top = (uint32_t)fminf((m - likely) * cb, (float)kBins);
  };
  u64 up = 0;
  if (counts) {
    clear();
    each(two, [&](const float (&v)[4], auto) {
#pragma unroll
      for (int e = 0; e < 4; e++) atomicAdd(&hist[(uint32_t)place_of(v[e])], 1ull);
    });
    if (run_up() >= k) cut = find((u64)k, 0, 0, &up);   // (fewer that have a mass: all of them)
    counts = false;
    top = b2 = 0;
    b0 = b1 = kBins;
    __syncthreads();
  }
  clear();
  u64 heavy = 0;
  if (STEP == kGather || (STEP == kRest && k == 0)) {
#pragma unroll
    for (uint32_t i = 0; i < BT; i++) hist[i * NT + tid] = ghist[i * NT + tid];
    heavy = ghist[kBins];
    if constexpr (STEP == kRest) {
      const u64 n = uni(ghist[kBins + 1]);
      ntok = n <= kSampleGather ? (uint32_t)n : ~0u;
    }
  } else {
    if (cut) masses(std::false_type{});
    else masses(std::true_type{});
    if (q > 0.0f) (void)scan(sq, &heavy);
    if constexpr (STEP == kMass) {
      __syncthreads();
#pragma unroll
      for (uint32_t i = 0; i < BT; i++)
        if (const u64 h = hist[i * NT + tid]) atomicAdd(&ghist[i * NT + tid], h);
      if (tid == 0 && heavy) atomicAdd(&ghist[kBins], heavy);
      return;
    }
  }
  u64 C = run_up();
  const float u = a.u[r];
  u64 R = share_of(p, C), least = 0, most = 0;
  if (q > 0.0f) C = max(min(C, uni(heavy)), (u64)(1.0 / kUnit));   // (the likeliest stays)
  if (nucleus) {
    // the draw's sum is known to within the mass of the bin that R is in
    reaching(R, [&](uint32_t b) {
      lo_s = b ? hist[b - 1] : 0;
      hi_s = hist[b];
    });
    __syncthreads();
    least = draw_of(u, min(C, uni(lo_s) + 1));
    most = draw_of(u, min(C, uni(hi_s)));
  }
  if constexpr (STEP == kGather) {
    // (R's bin, and behind a nucleus the bins that the draw can be in)
    if (!nucleus) R = draw_of(u, C);
    reaching(R, [&](uint32_t b) { bin_s = b; });
    if (nucleus) {
      reaching(least, [&](uint32_t b) { bin2_s[0] = b; });
      reaching(most, [&](uint32_t b) { bin2_s[1] = b; });
    }
    __syncthreads();
    const uint32_t b = uni(bin_s), i0 = nucleus ? uni(bin2_s[0]) : b, i1 = nucleus ? uni(bin2_s[1]) : b;
    cnt = 0;
    each(two, [&](const float (&v)[4], auto i) {
      note_four(v, i, [&](float x) { return of_bins(x, b, b) || of_bins(x, i0, i1); }, [](u64) { return true; }, cnt);
    });
    const uint32_t n = count_all(cnt);
    if (n <= kList) close_up(lane < cnt, lane < cnt ? list[tid] : 0);
    // (a piece whose list is too short for them makes the count say so)
    if (tid == 0) before_s = atomicAdd(&ghist[kBins + 1], n <= kList ? (u64)n : (u64)kSampleGather + 1);
    __syncthreads();
    const u64 at = uni(before_s) + tid;
    if (n <= kList && tid < n && at < kSampleGather) gtok[at] = list[tid];
    return;
  }
  // the nucleus' last token, then the one that is drawn
#pragma unroll 1
  for (bool last = !nucleus;; last = true) {
    if (last) {
      R = draw_of(u, C);
      least = 0;
    }
    const u64 key = find(R, least, most, &up);
    if (last) {
      if (tid == 0) answer(key, lp_of(key, C));
      return;
    }
    C = min(C, up);
    __syncthreads();
  }
}

// How many pieces a row is cut into: where rows are few, as many as give every
// CU one, of 8192 logits or more, and three at least. In pieces and whole (f32, us; a
// nucleus of 0.9 / the likeliest alone): 64 rows of 131072 46 and 76 / 18 and 14, 85
// of 65536 in three 39 and 46 / 15 and 9. In two, which are left out: 128 of 131072 71
// and 91 / 26 and 22, 128 of 65536 45 and 47 / 16 and 9. (16 rows of 32768 with a
// nucleus 27.7 and in four pieces 26, with a top-k of 40 11 and 12.7, their likeliest
// 8.7 and 12.8: rows that short stay whole.)
uint32_t pieces_of(uint32_t n, uint32_t vocab) {
  if (n == 0 || vocab < 65536) return 1;
  const uint32_t s = std::min(256 / n, vocab / 8192);
  return s < 3 ? 1 : s;
}

}  // namespace

uint64_t sample_ws_words(uint32_t n, uint32_t vocab) {
  const uint32_t S = pieces_of(n, vocab);
  return S > 1 ? n * sample_part_words(S) : 0;
}

hipError_t launch_sample(const SampleArgs& a, int type, hipStream_t st) {
  if (!a.logits || a.vocab == 0 || a.vocab > kSampleMaxVocab || a.n > kSampleMaxRows || (a.n > 1 && a.ld < a.vocab) ||
      !a.u || !a.tok || !a.lp)
    return hipErrorInvalidValue;
  if (a.n == 0) return hipSuccess;
  const uint32_t S = pieces_of(a.n, a.vocab), piece = ((a.vocab + S - 1) / S + 7) & ~7u, made = (a.vocab + piece - 1) / piece;
  if (S > 1 && !a.part) return hipErrorInvalidValue;
  auto go = [&](auto t) {
    using T = decltype(t);
    if (S == 1) {
      hipLaunchKernelGGL((k_sample<T, kWhole>), dim3(a.n), dim3(NT), 0, st, a, 1u, 0u);
      return;
    }
    hipLaunchKernelGGL((k_sample<T, kMax>), dim3(a.n * made), dim3(NT), 0, st, a, made, piece);
    if ((a.ts || a.t > 0.0f) && (a.ks || a.k == 0 || a.k >= a.vocab)) {   // (some row may ask for all masses)
      hipLaunchKernelGGL((k_sample<T, kMass>), dim3(a.n * made), dim3(NT), 0, st, a, made, piece);
      hipLaunchKernelGGL((k_sample<T, kGather>), dim3(a.n * made), dim3(NT), 0, st, a, made, piece);
    }
    hipLaunchKernelGGL((k_sample<T, kRest>), dim3(a.n), dim3(NT), 0, st, a, made, piece);
  };
  switch (type) {
    case ET_F32: go(float{}); break;
    case ET_BF16: go(__bf16{}); break;
    case ET_F16: go(_Float16{}); break;
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

}  // namespace ana
