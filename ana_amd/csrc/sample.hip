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
// A workgroup takes a row and keeps it in registers (longer rows are read
// again for each pass). One pass puts every token's mass into one of 2048 bins
// of a 64th of an octave, likeliest first; where a running mass is reached is
// then a bin, whose few tokens go to LDS and are told apart there. A top-k of
// up to 64 needs no masses but its own: the k-th largest of 64 group maxima is
// a bound that at least k logits reach and few more do.
#include <hip/hip_runtime.h>

#include "mfma.h"
#include "order.h"
#include "sample.h"
#include "wave.h"

namespace ana {

namespace {

constexpr uint32_t kPartBits = 9, NT = 1 << kPartBits, NW = NT / 64;
constexpr uint32_t kBins = 4 * NT, kBinsOctave = 64;   // 32 octaves; what is below them is in the last bin
constexpr uint32_t kList = NT;     // tokens of a bin that LDS takes, one a thread
constexpr uint32_t kFew = 64;      // of them, those that one wave tells apart
constexpr double kUnit = 0x1p-42;  // of a mass

// 2^x for x <= 0 (0 for a NaN): a series on half an octave about 0, relative
// error 8e-13 (each coefficient by iteration for the least largest error)
__device__ __forceinline__ double exp2_of(double x) {
  x = __builtin_fmax(x, -64.0);
  const double n = __builtin_rint(x), f = x - n;
  double s = fma(f, 0x1.61c4f09d828bap-20, 0x1.00d8535005e2dp-16);
  s = fma(f, s, 0x1.430aa88338cf8p-13);
  s = fma(f, s, 0x1.5d874d06e4851p-10);
  s = fma(f, s, 0x1.3b2ab5ed6f3f2p-7);
  s = fma(f, s, 0x1.c6b08dced3710p-5);
  s = fma(f, s, 0x1.ebfbdff8ede8fp-3);
  s = fma(f, s, 0x1.62e42fef89d1dp-1);
  return __builtin_amdgcn_ldexp(fma(f, s, 1.0), (int)n);
}
// a weight (0 .. 1) in units: the sum with 2^10 has steps of one
__device__ __forceinline__ u64 units_of(double w) {
  return __builtin_bit_cast(u64, w + 1024.0) - __builtin_bit_cast(u64, 1024.0);
}

// v's inclusive sum over the lanes up to this one
__device__ __forceinline__ u64 wave_scan(u64 v, uint32_t lane) {
#pragma unroll
  for (uint32_t s = 1; s < 64; s <<= 1) {
    const u64 o = __shfl_up(v, s, 64);
    if (lane >= s) v += o;
  }
  return v;
}

// (1 <= target <= C for 0 <= u < 1; others count as the nearest)
__device__ __forceinline__ u64 draw_of(float u, u64 C) {
  const double x = (double)fminf(fmaxf(u, 0.0f), 1.0f) * (double)C;
  return x >= (double)C ? C : min(C, (u64)x + 1);
}

// the vectors of a row that a thread holds
template <typename T>
constexpr uint32_t kVecs = sizeof(T) == 4 ? 16 : 13;

template <typename T, bool ONE>
__global__ __launch_bounds__(NT) __attribute__((amdgpu_waves_per_eu(4))) void k_sample(SampleArgs a) {
  constexpr uint32_t W = 16 / sizeof(T), V = kVecs<T>;
  typedef T vec_t __attribute__((ext_vector_type(W)));
  // (a row may start on any element's border)
  typedef vec_t vec_any __attribute__((aligned(sizeof(T))));
  __shared__ u64 hist[kBins], sub[NT], list[kList];
  __shared__ float tmax[NW][64];
  __shared__ u64 wsum[NW];
  __shared__ uint32_t nlist, bin_s;
  __shared__ u64 before_s, key_s, incl_s, lo_s, hi_s;
  __shared__ float bound_s;
  const uint32_t tid = threadIdx.x, lane = tid & 63, wv = tid >> 6, r = blockIdx.x;
  const T* row = (const T*)a.logits + (uint64_t)r * a.ld;
  const float t = a.ts ? a.ts[r] : a.t, p = a.ps ? a.ps[r] : a.p, q = a.qs ? a.qs[r] : a.q;
  const uint32_t k_ = a.ks ? a.ks[r] : a.k, k = k_ < a.vocab ? k_ : 0;   // (0: all)
  const uint32_t nvec = a.vocab / W;

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
  float xe = ie < a.vocab ? (float)row[ie] : -INFINITY;
  vec_t x[V];
  if constexpr (ONE) {
#pragma unroll
    for (uint32_t u = 0; u < V; u++) x[u] = load(u * NT + tid);
  }
  // f(value, index) over the thread's share of the row; places without a logit hold -inf
  auto each = [&](auto&& f) {
    if constexpr (ONE) {
#pragma unroll
      for (uint32_t u = 0; u < V; u++)
        if (u * NT < nvec) {
          // (or the compiler keeps what a pass forms of every element for the next)
          uint32_t i = (u * NT + tid) * W;
          asm volatile("" : "+v"(x[u]), "+v"(i));
#pragma unroll
          for (uint32_t e = 0; e < W; e++) f((float)x[u][e], i + e);
        }
    } else {
#pragma unroll 1
      for (uint32_t v = tid; v - tid < nvec; v += 2 * NT) {
        const vec_t y0 = load(v), y1 = load(v + NT);
#pragma unroll
        for (uint32_t e = 0; e < W; e++) f((float)y0[e], v * W + e);
#pragma unroll
        for (uint32_t e = 0; e < W; e++) f((float)y1[e], (v + NT) * W + e);
      }
    }
    f(xe, ie);
  };
  // the same from memory, for the rare paths: less code
  auto each_again = [&](auto&& f) {
#pragma unroll 1
    for (uint32_t i = tid; i - tid < a.vocab; i += NT) {
      float v = i < a.vocab ? (float)row[i] : -INFINITY;
      if (inf) v = v == INFINITY ? 0.0f : -INFINITY;
      f(v, i);
    }
  };
  // a token of the lanes with `in` to the list (all of the wave call it)
  auto put = [&](bool in, float v, uint32_t i) {
    const unsigned long long on = __ballot(in);
    if (on) {
      uint32_t at = 0;
      if (lane == 0) at = atomicAdd(&nlist, (uint32_t)__popcll(on));
      at = __builtin_amdgcn_readfirstlane(at) + __popcll(on & ((1ull << lane) - 1));
      if (in && at < kList) list[at] = key_of(v, i);
    }
  };
  auto answer = [&](u64 key, float lp) {
    a.tok[r] = 0xFFFFFFFFu - (uint32_t)key;
    a.lp[r] = lp;
  };

  float m = -INFINITY;
  each([&](float v, uint32_t) { m = fmaxf(m, v); });
  tmax[wv][lane] = m;
  if (tid == 0) nlist = 0;
  __syncthreads();
  // group l: lane l of every wave
  float gm = tmax[0][lane];
#pragma unroll
  for (uint32_t i = 1; i < NW; i++) gm = fmaxf(gm, tmax[i][lane]);
  m = wmax(gm);
  if (m == -INFINITY) {   // no number above it
    if (tid == 0) answer(~0ull << 32, __builtin_nanf(""));
    return;
  }
  if (m == INFINITY) {
    inf = true;
    if constexpr (ONE) {
#pragma unroll
      for (uint32_t u = 0; u < V; u++) x[u] = load(u * NT + tid);
    }
    xe = xe == INFINITY ? 0.0f : -INFINITY;
    gm = gm == INFINITY ? 0.0f : -INFINITY;
    m = 0.0f;
  }
  if (!(t > 0.0f) || k == 1) {
    uint32_t at = ~0u;
    each([&](float v, uint32_t i) { at = v == m ? min(at, i) : at; });
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

  const double c = 1.4426950408889634 / (double)t, md = m;
  auto weight = [&](float v) { return exp2_of(((double)v - md) * c); };
  // (the logarithm of its own share, from the logit)
  auto lp_of = [&](u64 key, u64 C) {
    return (float)(((double)value_of((uint32_t)(key >> 32)) - md) / (double)t - log((double)C * kUnit));
  };
  // mass to reach for a share p of S: 1 .. S
  auto share = [&](u64 S) {
    const double y = __builtin_ceil((double)p * (double)S);
    return y >= (double)S ? S : max(1ull, (u64)y);
  };
  const bool nucleus = p < 1.0f;

  if (k && k <= kFew) {
    if (wv == 0) {
      uint32_t above = 0;
#pragma unroll 4
      for (int i = 0; i < 64; i++) above += lane_f(gm, i) > gm;
      const float b = -wmax(above < k ? -gm : -INFINITY);
      if (lane == 0) bound_s = b;
    }
    __syncthreads();
    const float bound = bound_s;
    each([&](float v, uint32_t i) { put(v >= bound && v > -INFINITY, v, i); });
    __syncthreads();
    const uint32_t nc = nlist;
    if (nc <= kList) {
      if (tid < nc) {
        const u64 mine = list[tid];
        uint32_t over = 0;
        for (uint32_t o = 0; o < nc; o++) over += list[o] > mine ? 1u : 0u;
        if (over < k) sub[over] = mine;
      }
      __syncthreads();
      if (wv) return;
      const bool in = lane < min(k, nc);
      const u64 key = in ? sub[lane] : 0;
      const double wd = in ? weight(value_of((uint32_t)(key >> 32))) : 0.0;
      const u64 w = units_of(wd), incl = wave_scan(w, lane);
      const u64 S = __shfl(incl, 63, 64);
      const bool keep = in && (!nucleus || lane == 0 || incl - w < share(S)) && (wd >= (double)q || lane == 0);
      const uint32_t last = 63 - __clzll(__ballot(keep));
      const u64 C = __shfl(incl, last, 64), want = draw_of(a.u[r], C);
      if (incl >= want && incl - w < want) answer(key, lp_of(key, C));
      return;
    }
    __syncthreads();
  }

  // ---- the masses of all
  const float cb = (float)(c * kBinsOctave);
  auto bin_of = [&](float v) { return (uint32_t)fminf((m - v) * cb, (float)(kBins - 1)); };
  // the sum over the threads up to this one, and of all
  auto scan = [&](u64 v, u64* total) {
    v = wave_scan(v, lane);
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
    *total = all;
    return base + v;
  };
  // hist as running sums
  auto run_up = [&]() -> u64 {
    __syncthreads();
    u64 h[4], all;
#pragma unroll
    for (uint32_t i = 0; i < 4; i++) h[i] = hist[4 * tid + i] + (i ? h[i - 1] : 0);
    const u64 below = scan(h[3], &all) - h[3];
#pragma unroll
    for (uint32_t i = 0; i < 4; i++) hist[4 * tid + i] = below + h[i];
    __syncthreads();
    return all;
  };
  auto clear = [&]() {
#pragma unroll
    for (uint32_t i = 0; i < 4; i++) hist[i * NT + tid] = 0;
    __syncthreads();
  };
  u64 cut = 0;   // keys below it are out (top-k)
  // The key at which the running sum reaches R (1 .. the sum of all), of masses
  // or of counts, and the sum up to it.
  bool counts = k != 0;
  auto val = [&](float v) -> u64 { return counts ? 1 : units_of(weight(v)); };
  auto find = [&](u64 R, u64* incl) -> u64 {
#pragma unroll
    for (uint32_t i = 0; i < 4; i++) {
      const uint32_t b = 4 * tid + i;
      const u64 prev = b ? hist[b - 1] : 0;
      if (prev < R && R <= hist[b]) {
        bin_s = b;
        before_s = prev;
      }
    }
    if (tid == 0) nlist = 0;
    __syncthreads();
    const uint32_t b = bin_s;
    u64 before = before_s, lo = cut, hi = ~0ull;
    auto take = [&](float v, uint32_t i) {
      bool in = v > -INFINITY && bin_of(v) == b;
      if (__any(in)) {
        const u64 key = key_of(v, i);
        put(in && key >= lo && key <= hi, v, i);
      }
    };
    each(take);
    __syncthreads();
    uint32_t nc = nlist;
    // The keys lo .. hi of `members` into NT parts, the highest first: the part
    // that the sum reaches R in (its keys are lo .. hi then).
    auto narrow = [&](u64 least, u64 most, auto&& members) {
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
      least = lo_s;
      most = hi_s;
      const uint32_t bits = 64 - __clzll((long long)(most - least)), shift = bits > kPartBits ? bits - kPartBits : 0;
      members([&](u64 key) { atomicAdd(&sub[(most - key) >> shift], val(value_of((uint32_t)(key >> 32)))); });
      __syncthreads();
      const u64 mine = sub[tid];
      u64 all;
      const u64 up = before + scan(mine, &all);
      if (up - mine < R && R <= up) {
        bin_s = tid;
        before_s = up - mine;
      }
      __syncthreads();
      const u64 part = bin_s;
      before = before_s;
      hi = most - (part << shift);
      const u64 width = (1ull << shift) - 1;
      lo = hi - least > width ? hi - width : least;
    };
#pragma unroll 1
    while (nc > kList) {
      u64 least = ~0ull, most = 0;
      each_again([&](float v, uint32_t i) {
        const u64 key = key_of(v, i);
        if (v > -INFINITY && bin_of(v) == b && key >= lo && key <= hi) {
          least = min(least, key);
          most = max(most, key);
        }
      });
      const u64 lo0 = lo, hi0 = hi;
      narrow(least, most, [&](auto&& f) {
        each_again([&](float v, uint32_t i) {
          const u64 key = key_of(v, i);
          if (v > -INFINITY && bin_of(v) == b && key >= lo0 && key <= hi0) f(key);
        });
      });
      if (tid == 0) nlist = 0;
      __syncthreads();
      each_again(take);
      __syncthreads();
      nc = nlist;
    }
#pragma unroll 1
    while (nc > kFew) {
      const bool in = tid < nc;
      const u64 key = in ? list[tid] : 0;
      narrow(in ? key : ~0ull, key, [&](auto&& f) {
        if (in) f(key);
      });
      if (tid == 0) nlist = 0;
      __syncthreads();
      if (in && key >= lo && key <= hi) list[atomicAdd(&nlist, 1u)] = key;
      __syncthreads();
      nc = nlist;
    }
    if (wv == 0) {
      const bool in = lane < nc;
      const u64 key = in ? list[lane] : 0, w = in ? val(value_of((uint32_t)(key >> 32))) : 0;
      u64 up = before + w;
      for (uint32_t o = 0; o < nc; o++) {
        const u64 ok = __shfl(key, o, 64), ow = __shfl(w, o, 64);
        if (ok > key) up += ow;
      }
      if (in && up >= R && up - w < R) {
        key_s = key;
        incl_s = up;
      }
    }
    __syncthreads();
    *incl = incl_s;
    return key_s;
  };

  if (counts) {
    clear();
    each([&](float v, uint32_t) {
      if (v > -INFINITY) atomicAdd(&hist[bin_of(v)], 1ull);
    });
  }
  u64 C = 0, R = k;
  // the k-th token, the nucleus' last, the one that is drawn
#pragma unroll 1
  for (uint32_t stage = counts ? 0 : 1; stage < 3; stage++) {
    if (stage == 0 && run_up() < k) {   // (fewer numbers than that)
      counts = false;
      continue;
    }
    if (stage == 1) {
      clear();
      u64 sq = 0;   // of those of weight q or more
      const double qd = q;
      auto masses = [&](auto all) {
        each([&](float v, uint32_t i) {
          double w = weight(v);
          if constexpr (!decltype(all)::value) w = key_of(v, i) >= cut ? w : 0.0;
          const u64 n = units_of(w);
          sq += w >= qd ? n : 0;
          if (n) atomicAdd(&hist[bin_of(v)], n);
        });
      };
      if (cut) masses(std::false_type{});
      else masses(std::true_type{});
      C = run_up();
      R = share(C);
      if (q > 0.0f) (void)scan(sq, &C);
      C = max(C, (u64)(1.0 / kUnit));   // (the likeliest stays)
      if (!nucleus) continue;
    }
    if (stage == 2) R = draw_of(a.u[r], C);
    u64 up;
    const u64 key = find(R, &up);
    if (stage == 0) cut = key;
    if (stage == 1) C = min(C, up);
    if (stage == 2 && tid == 0) answer(key, lp_of(key, C));
    counts = false;
    __syncthreads();
  }
}

}  // namespace

hipError_t launch_sample(const SampleArgs& a, int type, hipStream_t st) {
  if (!a.logits || a.vocab == 0 || a.vocab > kSampleMaxVocab || a.n > kSampleMaxRows || (a.n > 1 && a.ld < a.vocab) ||
      !a.u || !a.tok || !a.lp)
    return hipErrorInvalidValue;
  if (a.n == 0) return hipSuccess;
  auto go = [&](auto t) {
    using T = decltype(t);
    if (a.vocab / (16 / sizeof(T)) <= NT * kVecs<T>) hipLaunchKernelGGL((k_sample<T, true>), dim3(a.n), dim3(NT), 0, st, a);
    else hipLaunchKernelGGL((k_sample<T, false>), dim3(a.n), dim3(NT), 0, st, a);
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
