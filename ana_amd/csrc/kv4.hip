// Keys and values held in 4 bits, and softmax attention over them (gfx950).
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

#include <algorithm>

#include "kv4.h"
#include "mfma.h"
#include "wave.h"

namespace ana {

namespace {

typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef float f32x2_t __attribute__((ext_vector_type(2)));

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__bf16 x) { return (float)x; }
__device__ __forceinline__ float to_f(_Float16 x) { return (float)x; }

// eight consecutive elements (vec: on a 16-byte border)
template <typename T>
__device__ __forceinline__ void load8(const T* p, bool vec, float (&x)[8]) {
  if (vec) {
    if constexpr (sizeof(T) == 4) {
      const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
      x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
      x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
    } else {
      typedef T vec8 __attribute__((ext_vector_type(8)));
      const vec8 a = *reinterpret_cast<const vec8*>(p);
#pragma unroll
      for (int e = 0; e < 8; e++) x[e] = to_f((T)a[e]);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; e++) x[e] = to_f(p[e]);
  }
}
template <typename T>
__device__ __forceinline__ void store8(T* p, bool vec, const float (&x)[8]) {
  if (vec) {
    if constexpr (sizeof(T) == 4) {
      reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
      reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
    } else {
      typedef T vec8 __attribute__((ext_vector_type(8)));
      vec8 a;
#pragma unroll
      for (int e = 0; e < 8; e++) a[e] = (T)x[e];
      *reinterpret_cast<vec8*>(p) = a;
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; e++) p[e] = (T)x[e];
  }
}

// the last i < n with off[i] <= r (0 when there is none), for the whole wave:
// 64 of the remaining places at a time
__device__ __forceinline__ uint32_t find_seq(const uint32_t* off, uint32_t n, uint32_t r) {
  const uint32_t lane = threadIdx.x & 63;
  uint32_t lo = 0, cnt = n;
  while (cnt > 1) {
    const uint32_t step = (cnt + 63) / 64, k = lane * step;
    const bool t = k < cnt && off[lo + k] <= r;
    const uint32_t c = __popcll(__ballot(t));
    if (c == 0) break;
    lo += (c - 1) * step;
    cnt = min(step, cnt - (c - 1) * step);
  }
  return lo;
}

// where a row is: its sequence's index in the call, place in the cache,
// position, and the last position of its sequence in the call
struct RowAt {
  uint32_t i, q, p, last;
  bool on;    // a row of some sequence (else nothing is read or written)
  bool ok;    // with a place in the cache
};
// (i0: find_seq of a row at or before `row`)
__device__ __forceinline__ RowAt row_at(const Kv4& c, const Kv4Rows& r, uint32_t row, uint32_t i0) {
  RowAt a{i0, 0, 0, 0, row < r.rows, false};
  if (!a.on) return a;
  uint32_t o0 = row, o1 = row + 1;
  if (r.off) {
    while (a.i + 1 < r.n && r.off[a.i + 1] <= row) a.i++;
    o0 = r.off[a.i];
    o1 = r.off[a.i + 1];
    a.on = row >= o0 && row < o1;
  } else {
    a.i = row;
    a.on = row < r.n;
  }
  if (!a.on) return a;
  a.q = r.seq ? r.seq[a.i] : a.i;
  a.ok = a.q < c.seqs;
  a.p = r.pos[a.i] + (row - o0);
  a.last = r.pos[a.i] + (o1 - 1 - o0);
  return a;
}

__device__ __forceinline__ uint8_t* record_of(const Kv4& c, uint32_t q, uint32_t head, uint32_t tile) {
  return c.data + (((uint64_t)q * c.heads + head) * c.tiles + tile) * kv4_record(c.hd);
}

// |x| 2^(127 - b) as an E2M1 code, to the nearest, ties to the even code.
// From 1 up a code is the float's exponent and first mantissa bit; below, the
// halves.
__device__ __forceinline__ uint32_t e2m1(float y) {
  const uint32_t u = __builtin_bit_cast(uint32_t, y);
  const uint32_t hi = ((u + 0x1FFFFFu + ((u >> 22) & 1)) >> 22) - 252;
  const uint32_t lo = (uint32_t)(int)rintf(y + y);
  return min(y < 1.0f ? lo : hi, 7u);
}

// A call's keys and values into the cache: a workgroup takes 32 rows of one
// head, eight dims a thread (a slot's codes of one lane of the attention are
// hd / 4 dims of a key and hd / 16 of a value). z = 0 the keys, 1 the
// values, 2 the query rows, which are only qk-normed in place. The block's
// largest magnitude comes from the quad of threads that share it, in the
// floats' bits, where a block that is not finite shows itself too.
// A row that a later one of the call overwrites (a ring shorter than the
// call), and rows of a sequence that the call lists a second time, are left
// out, so that what is stored does not depend on the order of the threads.
template <typename T, int D>
__global__ __launch_bounds__(4 * D) void k_kv4_write(Kv4 c, Kv4Rows r, Kv4Mat k, Kv4Mat v, uint32_t vec,
                                                     const float* gk, const float* gq, Kv4Mat qm, uint32_t kh) {
  constexpr uint32_t TPR = D / 8;
  const uint32_t tid = threadIdx.x, sub = tid % TPR, row = blockIdx.x * 32 + tid / TPR, head = blockIdx.y;
  const uint32_t z = blockIdx.z;
  if (z < 2 && head >= kh) return;
  const uint32_t i0 = r.off ? find_seq(r.off, r.n, blockIdx.x * 32) : 0;
  const RowAt a = row_at(c, r, row, i0);
  const Kv4Mat& src = z == 0 ? k : z == 1 ? v : qm;
  T* p = (T*)src.p + (uint64_t)row * src.row + (uint64_t)head * src.head + sub * 8;
  float x[8] = {};
  if (a.on) load8(p, vec, x);
  const float* g = z == 0 ? gk : z == 2 ? gq : nullptr;
  if (g) {
    // M.qkn (bend/Dense/Model.bend:39-42)
    float s = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; e++) s = fmaf(x[e], x[e], s);
#pragma unroll
    for (uint32_t mk = 1; mk < TPR; mk <<= 1) s += __shfl_xor(s, mk, 64);
    const float n = 1.0f / sqrtf(s / (float)D + 1.0e-5f);
#pragma unroll
    for (int e = 0; e < 8; e++) x[e] = (x[e] * n) * (1.0f + g[sub * 8 + e]);
  }
  if (z == 2) {
    if (a.on) store8(p, vec, x);
    return;
  }
  bool put = a.ok && a.last - a.p < c.slots;
  if (r.seq && put) {
    uint32_t dup = 0;
    for (uint32_t j = sub; j < a.i; j += TPR)
      if (r.seq[j] == a.q && (!r.off || r.off[j + 1] > r.off[j])) dup = 1;
#pragma unroll
    for (uint32_t mk = 1; mk < TPR; mk <<= 1) dup |= __shfl_xor(dup, mk, 64);
    put = !dup;
  }
  uint32_t top = 0;
#pragma unroll
  for (int e = 0; e < 8; e++) top = max(top, __builtin_bit_cast(uint32_t, x[e]) & 0x7FFFFFFFu);
  top = max(top, (uint32_t)__builtin_amdgcn_mov_dpp((int)top, 0xB1, 0xF, 0xF, true));
  top = max(top, (uint32_t)__builtin_amdgcn_mov_dpp((int)top, 0x4E, 0xF, 0xF, true));
  const bool bad = top >= 0x7F800000u;
  const int e8 = (int)(top >> 23) - 2 + ((top & 0x7FFFFFu) > 0x600000u ? 1 : 0);
  const uint32_t b = bad ? 255u : (uint32_t)min(max(e8, 2), 252);
  const float f = __builtin_bit_cast(float, (254u - min(b, 252u)) << 23);
  uint32_t w = 0;
#pragma unroll
  for (int e = 0; e < 8; e++)
    w |= (e2m1(fabsf(x[e]) * f) | (__builtin_bit_cast(uint32_t, x[e]) >> 31 << 3)) << (4 * e);
  if (bad) w = 0;
  if (!put) return;
  const uint32_t slot = a.p % c.slots, s = slot % 32, h = s / 16, m = s % 16, dim = sub * 8;
  uint8_t* rec = record_of(c, a.q, head, slot / 32);
  if (z == 0) {
    const uint32_t j = dim / (D / 4);
    *reinterpret_cast<uint32_t*>(rec + (j * 16 + m) * (D / 4) + h * (D / 8) + dim % (D / 4) / 2) = w;
    if (sub % 4 == 0) rec[32 * D + (dim / 32 * 16 + m) * 2 + h] = (uint8_t)b;
  } else {
    const uint32_t j = m / 4, e = h * 4 + m % 4;
    uint8_t* at = rec + 16 * D + (j * 16 + dim / (D / 16)) * (D / 4) + e * (D / 32);
    if constexpr (D == 128) {
      *reinterpret_cast<uint32_t*>(at) = w;
    } else if constexpr (D == 64) {
      *reinterpret_cast<uint16_t*>(at) = (uint16_t)w;
      *reinterpret_cast<uint16_t*>(at + D / 4) = (uint16_t)(w >> 16);
    } else {
#pragma unroll
      for (int u = 0; u < 4; u++) at[u * (D / 4)] = (uint8_t)(w >> (8 * u));
    }
    if (sub % 4 == 0) rec[33 * D + (dim / 32 * 4 + j) * 8 + e] = (uint8_t)b;
  }
}

// k_kv4_write the other way: the values that the cache holds for the rows
// (zeros for a sequence without a place in the cache)
template <typename T, int D>
__global__ __launch_bounds__(4 * D) void k_kv4_read(Kv4 c, Kv4Rows r, Kv4Mat k, Kv4Mat v, uint32_t vec) {
  constexpr uint32_t TPR = D / 8;
  const uint32_t tid = threadIdx.x, sub = tid % TPR, row = blockIdx.x * 32 + tid / TPR, head = blockIdx.y;
  const uint32_t i0 = r.off ? find_seq(r.off, r.n, blockIdx.x * 32) : 0;
  const RowAt a = row_at(c, r, row, i0);
  if (!a.on) return;
  uint32_t w = 0, b = 2;
  if (a.ok) {
    const uint32_t slot = a.p % c.slots, s = slot % 32, h = s / 16, m = s % 16, dim = sub * 8;
    const uint8_t* rec = record_of(c, a.q, head, slot / 32);
    if (blockIdx.z == 0) {
      const uint32_t j = dim / (D / 4);
      w = *reinterpret_cast<const uint32_t*>(rec + (j * 16 + m) * (D / 4) + h * (D / 8) + dim % (D / 4) / 2);
      b = rec[32 * D + (dim / 32 * 16 + m) * 2 + h];
    } else {
      const uint32_t j = m / 4, e = h * 4 + m % 4;
      const uint8_t* at = rec + 16 * D + (j * 16 + dim / (D / 16)) * (D / 4) + e * (D / 32);
      if constexpr (D == 128) {
        w = *reinterpret_cast<const uint32_t*>(at);
      } else if constexpr (D == 64) {
        w = *reinterpret_cast<const uint16_t*>(at) | (uint32_t)*reinterpret_cast<const uint16_t*>(at + D / 4) << 16;
      } else {
#pragma unroll
        for (int u = 0; u < 4; u++) w |= (uint32_t)at[u * (D / 4)] << (8 * u);
      }
      b = rec[33 * D + (dim / 32 * 4 + j) * 8 + e];
    }
  }
  const float f = b == 255 ? __builtin_nanf("") : __builtin_bit_cast(float, b << 23);
  float x[8];
  static_for<4>([&](auto u) {
    const f32x2_t t = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, decltype(u)::value);
    x[2 * u] = t[0] * f;
    x[2 * u + 1] = t[1] * f;
  });
  const Kv4Mat& dst = blockIdx.z == 0 ? k : v;
  store8((T*)dst.p + (uint64_t)row * dst.row + (uint64_t)head * dst.head + sub * 8, vec, x);
}

// ---------------------------------------------------------------- attention
//
// With the scores transposed, S^T = K Q^T (a tile's slots are the MFMA's
// rows, up to 16 (row, query head) pairs of one key head its columns), a lane
// ends with the scores of its pair for slots 4 j + i and 16 + 4 j + i of the
// tile: the operand that O^T = V^T P^T wants from it, once the values' slots
// are taken in the same order. So the scores and the probabilities never
// leave their registers, a pair's running maximum is one shared by four
// lanes, and the cache's records are ordered so that a lane's consecutive
// bytes are its part of both operands. An E2M1 code times a power of two is a
// bf16, so keys and values enter the products as they are; a query is the
// exact sum of NP bf16 parts (three for f32, two for f16) and a probability
// is taken in NPP parts (f32: three, the whole of it; 16-bit outputs: two,
// 2^-17 of it), each product of parts exact in the f32 sum.

template <typename T> struct Parts;
template <> struct Parts<float> { static constexpr int q = 3, p = 3; };
template <> struct Parts<__bf16> { static constexpr int q = 1, p = 2; };
template <> struct Parts<_Float16> { static constexpr int q = 2, p = 2; };

// eight floats as N bf16 operands whose sum they are (to 2^-(8 N + 1)); a
// value next to the largest float is kept from rounding to infinity
template <int N>
__device__ __forceinline__ void split8(const float (&x)[8], bf16x8_t (&o)[N]) {
  constexpr float M = 3.3895313892515355e38f;   // the largest bf16
  float r[8];
#pragma unroll
  for (int e = 0; e < 8; e++) r[e] = x[e];
#pragma unroll
  for (int n = 0; n < N; n++)
#pragma unroll
    for (int e = 0; e < 8; e++) {
      const __bf16 h = (__bf16)(n == 0 && N == 3 ? __builtin_amdgcn_fmed3f(r[e], -M, M) : r[e]);
      o[n][e] = h;
      r[e] -= (float)h;
    }
}

// a record as a lane reads it
template <int D>
struct Raw {
  uint32_t k[D / 16], v[D / 16];
  uint32_t ks;     // the key scales of slots m (low byte) and 16 + m
  uint32_t vs[2];  // the value scales of its eight slots
};
template <int D>
__device__ __forceinline__ void load_words(uint32_t (&w)[D / 16], const uint8_t* p) {
  if constexpr (D == 32) {
    const uint2 t = *reinterpret_cast<const uint2*>(p);
    w[0] = t.x; w[1] = t.y;
  } else {
#pragma unroll
    for (int i = 0; i < D / 64; i++) {
      const uint4 t = reinterpret_cast<const uint4*>(p)[i];
      w[4 * i] = t.x; w[4 * i + 1] = t.y; w[4 * i + 2] = t.z; w[4 * i + 3] = t.w;
    }
  }
}
template <int D>
__device__ __forceinline__ void load_k(Raw<D>& r, const uint8_t* rec, uint32_t lane) {
  load_words<D>(r.k, rec + lane * (D / 4));
  r.ks = *reinterpret_cast<const uint16_t*>(rec + 32 * D + ((lane >> 4) * D / 128 * 16 + (lane & 15)) * 2);
}
template <int D>
__device__ __forceinline__ void load_v(Raw<D>& r, const uint8_t* rec, uint32_t lane) {
  load_words<D>(r.v, rec + 16 * D + lane * (D / 4));
  const uint2 t = *reinterpret_cast<const uint2*>(rec + 33 * D + ((lane & 15) * D / 512 * 4 + (lane >> 4)) * 8);
  r.vs[0] = t.x;
  r.vs[1] = t.y;
}

// whether some byte of w is 255 (the scale of a block that is not finite)
__device__ __forceinline__ uint32_t has255(uint32_t w) {
  return ((w & 0x7F7F7F7Fu) + 0x01010101u) & w & 0x80808080u;
}
__device__ __forceinline__ float scale_of(uint32_t w, int byte) {
  return __builtin_bit_cast(float, ((w >> (8 * byte)) & 0xFFu) << 23);
}
template <int B>
__device__ __forceinline__ uint32_t two_of(uint32_t w, float s) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, B));
}
// the key operand of slots 16 h + m, step s of the head's dims (eight codes)
template <int D>
__device__ __forceinline__ bf16x8_t key_op(const Raw<D>& r, int h, int s, float sc) {
  const uint32_t w = r.k[h * (D / 32) + s];
  const u32x4_t o = {two_of<0>(w, sc), two_of<1>(w, sc), two_of<2>(w, sc), two_of<3>(w, sc)};
  return __builtin_bit_cast(bf16x8_t, o);
}
// the value operands of dims m D / 16 + 2 u and + 1 over the lane's eight slots
template <int D, int U>
__device__ __forceinline__ void val_ops(const Raw<D>& r, const float (&sc)[8], bf16x8_t& a, bf16x8_t& b) {
  uint32_t x[8];
  static_for<8>([&](auto e_) {
    constexpr int e = decltype(e_)::value, byte = e * (D / 32) + U;
    x[e] = two_of<byte % 4>(r.v[byte / 4], sc[e]);
  });
  u32x4_t lo, hi;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    lo[i] = __builtin_amdgcn_perm(x[2 * i + 1], x[2 * i], 0x05040100u);
    hi[i] = __builtin_amdgcn_perm(x[2 * i + 1], x[2 * i], 0x07060302u);
  }
  a = __builtin_bit_cast(bf16x8_t, lo);
  b = __builtin_bit_cast(bf16x8_t, hi);
}

// the maximum, or the sum, over the four lanes of a pair (lanes m, m + 16,
// m + 32, m + 48), in all of them
__device__ __forceinline__ float pair_max(float x) {
  auto a = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, x), false, false);
  x = fmaxf(__builtin_bit_cast(float, (uint32_t)a[0]), __builtin_bit_cast(float, (uint32_t)a[1]));
  auto b = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, x), false, false);
  return fmaxf(__builtin_bit_cast(float, (uint32_t)b[0]), __builtin_bit_cast(float, (uint32_t)b[1]));
}
__device__ __forceinline__ float pair_sum(float x) {
  x += __shfl_xor(x, 16, 64);
  return x + __shfl_xor(x, 32, 64);
}
__device__ __forceinline__ uint32_t pair_or(uint32_t x) {
  x |= __shfl_xor(x, 16, 64);
  return x | __shfl_xor(x, 32, 64);
}

// What a workgroup's pairs see: slot s holds a position of the ring's last
// turn (up to slot cur) or of the one before.
struct View {
  uint32_t cur, live;   // the last position's slot; live slots
  int64_t turn;         // position of slot 0 in the last turn
  uint32_t slots;
  __device__ __forceinline__ View(uint32_t last, uint32_t slots_) : slots(slots_) {
    cur = last % slots;
    turn = (int64_t)last - cur;
    live = last < slots ? last + 1 : slots;
  }
  __device__ __forceinline__ bool sees(uint32_t s, uint32_t p) const {
    const int64_t at = s <= cur ? turn + s : turn - slots + s;
    return s < live && at <= (int64_t)p;
  }
  // whether every slot of tile t is live and holds a position up to p (the
  // positions above p are those of slots after p's up to cur)
  __device__ __forceinline__ bool whole(uint32_t t, uint32_t last, uint32_t p) const {
    const uint32_t s0 = t * 32, s1 = s0 + 31;
    if (s1 >= live) return false;
    if (last == p) return true;
    if (last - p >= slots) return false;
    const uint32_t a = (p + 1) % slots;
    return a <= cur ? (s1 < a || s0 > cur) : (s1 < a && s0 > cur);
  }
};

// Pairs of a sequence: c = row * G + query head within the key head's group.
// One tile's scores for 16 pairs, its probabilities and their product with
// the values, with the pairs' running maxima and sums; K and V operands come
// from key(h, s) and val(t).
template <int D, int NPP>
struct Acc {
  f32x4_t o[D / 16];
  float m, l;
  uint32_t nan;   // blocks of dims that a seen value which is not finite makes so
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int t = 0; t < D / 16; t++) o[t] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
    m = -INFINITY;
    l = 0.0f;
    nan = 0;
  }
  // scores (already scaled to base 2, masked) of the pair's eight slots of a
  // tile: the probabilities in parts
  __device__ __forceinline__ void soften(float (&x)[8], bf16x8_t (&p)[NPP]) {
    float t = x[0];
#pragma unroll
    for (int e = 1; e < 8; e++) t = fmaxf(t, x[e]);
    t = pair_max(t);
    if (__any(t > m)) {
      const float n = fmaxf(m, t);
      const float f = n == m ? 1.0f : __builtin_amdgcn_exp2f(m - n);
      m = n;
      l *= f;
#pragma unroll
      for (int i = 0; i < D / 16; i++) o[i] *= f;
    }
    const float b = m == -INFINITY ? 0.0f : m;
#pragma unroll
    for (int e = 0; e < 8; e++) {
      x[e] = __builtin_amdgcn_exp2f(x[e] - b);
      l += x[e];
    }
    split8(x, p);
  }
};

// the query operand of a pair: dims j D / 4 + 8 s + e of its row, in parts
template <typename T, int D, int NP>
__device__ __forceinline__ void query_ops(const Kv4Mat& q, uint32_t row, uint32_t head, uint32_t j, bool on, bool vec,
                                          bf16x8_t (&o)[NP][D / 32]) {
  const T* p = (const T*)q.p + (uint64_t)row * q.row + (uint64_t)head * q.head + j * (D / 4);
#pragma unroll
  for (int s = 0; s < D / 32; s++) {
    float x[8] = {};
    if (on) load8(p + 8 * s, vec, x);
    bf16x8_t t[NP];
    split8(x, t);
#pragma unroll
    for (int n = 0; n < NP; n++) o[n][s] = t[n];
  }
}

constexpr float kLog2e = 1.4426950408889634f;
// pairs of a sequence up to which the few-row kernel takes it
constexpr uint32_t kFewPairs = 16;

// a pair's finished output dims j D / 4 .. (n = D / 4 of them in a lane):
// with a sink, then normalised
template <typename T>
__device__ __forceinline__ float finish_sum(float m, float l, const float* sink, uint32_t head, float* f) {
  // the weight of what was summed with maximum m, and the denominator
  float den = l;
  *f = 1.0f;
  if (sink) {
    const float s = sink[head] * kLog2e;
    const float n = fmaxf(m, s);
    if (n != -INFINITY) {
      *f = __builtin_amdgcn_exp2f(m - n);
      den = l * *f + __builtin_amdgcn_exp2f(s - n);
    }
    if (s != s) den = s;
  }
  return den;
}

// Few rows (up to 16 pairs of one sequence and key head): one workgroup per
// (sequence, key head, piece of the slots), its four waves taking every
// fourth tile with the next one's loads in flight, each with a running
// softmax of its own; they meet in LDS. Bound by the records' bytes.
template <typename T, int D>
__global__ __launch_bounds__(256) void k_kv4_few(Kv4Attend a, uint32_t vec, uint32_t nt16) {
  constexpr int NP = Parts<T>::q, NPP = Parts<T>::p;
  __shared__ float om[4][16][D + 4];
  __shared__ float mm[4][16], ll[4][16];
  const uint32_t tid = threadIdx.x, lane = tid & 63, wv = tid >> 6, m = lane & 15, j = lane >> 4;
  uint32_t w = blockIdx.x;
  const uint32_t sub = w % nt16;
  w /= nt16;
  const uint32_t head = w % a.c.heads, i = w / a.c.heads, z = blockIdx.y;
  const uint32_t G = a.hq / a.c.heads;
  uint32_t row0 = i, len = 1;
  if (a.r.off) {
    const uint32_t o0 = a.r.off[i], o1 = a.r.off[i + 1];
    if (o1 <= o0 || o1 > a.r.rows) return;
    row0 = o0;
    len = o1 - o0;
    if ((uint64_t)len * G > kFewPairs) return;
  }
  const uint32_t q = a.r.seq ? a.r.seq[i] : i;
  const uint32_t pos = a.r.pos[i], last = pos + len - 1;
  const uint32_t np = min(len * G - sub * 16, 16u);   // pairs here
  const uint32_t c0 = sub * 16;
  const bool ok = q < a.c.seqs;
  const View view(last, a.c.slots);
  const uint32_t tiles = ok ? (view.live + 31) / 32 : 0u;
  const uint32_t t0 = z * a.tps, t1 = z + 1 == a.nsplit ? tiles : min(tiles, t0 + a.tps);
  if (a.nsplit > 1 && t0 >= t1) return;
  const uint32_t pr = c0 + m, t = pr / G, g = pr % G;
  const bool on = m < np;
  bf16x8_t qo[NP][D / 32];
  query_ops<T, D, NP>(a.q, row0 + t, head * G + g, j, on, vec, qo);
  const uint32_t p = pos + t;
  const float sc = a.scale * kLog2e;
  Acc<D, NPP> acc;
  acc.clear();
  const uint8_t* base = record_of(a.c, ok ? q : 0, head, 0);
  Raw<D> cur, nxt;
  uint32_t tile = t0 + wv;
  if (tile < t1) {
    load_k(cur, base + (uint64_t)tile * (34 * D), lane);
    load_v(cur, base + (uint64_t)tile * (34 * D), lane);
  }
  for (; tile < t1; tile += 4) {
    if (tile + 4 < t1) {
      load_k(nxt, base + (uint64_t)(tile + 4) * (34 * D), lane);
      load_v(nxt, base + (uint64_t)(tile + 4) * (34 * D), lane);
    }
    const bool whole = view.whole(tile, last, pos);
    if (!whole) {
      // the values of slots that hold nothing are not to count
#pragma unroll
      for (int e = 0; e < 8; e++)
        if (tile * 32 + 16 * (e / 4) + 4 * j + e % 4 >= view.live) cur.vs[e / 4] &= ~(0xFFu << (8 * (e % 4)));
    }
    const bool bad = __any(has255(cur.ks) | has255(cur.vs[0]) | has255(cur.vs[1]));
    f32x4_t s[2];
#pragma unroll
    for (int h = 0; h < 2; h++) {
      s[h] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
      const float ksc = scale_of(cur.ks, h);
#pragma unroll
      for (int d = 0; d < D / 32; d++) {
        bf16x8_t ko = key_op<D>(cur, h, d, ksc);
        if (bad && ((cur.ks >> (8 * h)) & 0xFF) == 255) {
          const u32x4_t nn = {0x7FC07FC0u, 0x7FC07FC0u, 0x7FC07FC0u, 0x7FC07FC0u};
          ko = __builtin_bit_cast(bf16x8_t, nn);
        }
#pragma unroll
        for (int n = 0; n < NP; n++) s[h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ko, qo[n][d], s[h], 0, 0, 0);
      }
    }
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; e++) x[e] = s[e / 4][e % 4] * sc;
    if (!whole) {
#pragma unroll
      for (int e = 0; e < 8; e++)
        if (!view.sees(tile * 32 + 16 * (e / 4) + 4 * j + e % 4, p)) x[e] = -INFINITY;
    }
    if (bad) {
      // a value block that is not finite counts for the pairs that see it
      // alone: out of the product, and into their dims at the end
      const uint8_t* vs = base + (uint64_t)tile * (34 * D) + 33 * D + j * 8;
      for (int e = 0; e < 8; e++) {
        const uint32_t slot = tile * 32 + 16 * (e / 4) + 4 * j + e % 4;
        if (!view.sees(slot, p)) continue;
        for (int b = 0; b < D / 32; b++)
          if (vs[b * 32 + e] == 255) acc.nan |= 1u << b;
      }
#pragma unroll
      for (int e = 0; e < 8; e++)
        if (((cur.vs[e / 4] >> (8 * (e % 4))) & 0xFF) == 255) cur.vs[e / 4] &= ~(0xFFu << (8 * (e % 4)));
    }
    bf16x8_t po[NPP];
    acc.soften(x, po);
    float vsc[8];
#pragma unroll
    for (int e = 0; e < 8; e++) vsc[e] = scale_of(cur.vs[e / 4], e % 4);
    static_for<D / 32>([&](auto u_) {
      constexpr int u = decltype(u_)::value;
      bf16x8_t v0, v1;
      val_ops<D, u>(cur, vsc, v0, v1);
#pragma unroll
      for (int n = 0; n < NPP; n++) {
        acc.o[2 * u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v0, po[n], acc.o[2 * u], 0, 0, 0);
        acc.o[2 * u + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v1, po[n], acc.o[2 * u + 1], 0, 0, 0);
      }
    });
    cur = nxt;
  }
  // the four waves meet
  const float l = pair_sum(acc.l);
  const uint32_t nan = pair_or(acc.nan);
  if (j == 0) {
    mm[wv][m] = acc.m;
    ll[wv][m] = l;
  }
#pragma unroll
  for (int i4 = 0; i4 < 4; i4++)
#pragma unroll
    for (int t16 = 0; t16 < D / 16; t16++) {
      const uint32_t d = j * (D / 4) + i4 * (D / 16) + t16;
      om[wv][m][d] = (nan >> (d / 32)) & 1 ? __builtin_nanf("") : acc.o[t16][i4];
    }
  __syncthreads();
  for (uint32_t k = tid; k < np * D; k += 256) {
    const uint32_t pp = k / D, d = k % D;
    const float M = fmaxf(fmaxf(mm[0][pp], mm[1][pp]), fmaxf(mm[2][pp], mm[3][pp]));
    float lsum = 0.0f, o = 0.0f;
#pragma unroll
    for (int u = 0; u < 4; u++) {
      // (a wave without a seen slot has nothing, but a score that is not a number stays one)
      const float f = mm[u][pp] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mm[u][pp] - M);
      lsum += ll[u][pp] * f;
      o += om[u][pp][d] * f;
    }
    const uint32_t row = row0 + (c0 + pp) / G, hd = head * G + (c0 + pp) % G;
    if (a.nsplit > 1) {
      float* part = a.part + (((uint64_t)row * a.hq + hd) * a.nsplit + z) * (D + 2);
      part[2 + d] = o;
      if (d == 0) {
        part[0] = M;
        part[1] = lsum;
      }
    } else {
      float f;
      const float den = finish_sum<T>(M, lsum, a.sink, hd, &f);
      const float y = ok && (den != 0.0f) ? o * f / den : 0.0f;
      ((T*)a.o.p)[(uint64_t)row * a.o.row + (uint64_t)hd * a.o.head + d] = (T)y;
    }
  }
}

// Many rows (more than 16 pairs of one sequence and key head): a workgroup
// takes 64 NQ pairs, 16 NQ a wave, over the slots they see, 64 at a time.
// Each wave turns one of the step's four halves (two tiles' keys, two tiles'
// values) into operands in LDS, lane by lane as the MFMAs want them, so
// every read and write there is a lane's own 16 bytes; the step's records
// were loaded a step ahead, and two sets of operands leave one barrier a
// step.
template <typename T, int D>
struct Many {
  // pairs a wave: the queries' parts and the outputs share its registers
  static constexpr int NQ = D == 128 && Parts<T>::q > 1 ? 1 : 2;
  static constexpr uint32_t pairs = 64 * NQ;
};

template <typename T, int D>
__global__ __launch_bounds__(256, 2) void k_kv4_many(Kv4Attend a, uint32_t vec) {
  constexpr int NP = Parts<T>::q, NPP = Parts<T>::p, NQ = Many<T, D>::NQ;
  constexpr uint32_t PW = Many<T, D>::pairs;
  constexpr int KOPS = 2 * (D / 32), VOPS = D / 16;     // operands a tile
  __shared__ bf16x8_t kop[2][2][KOPS][64], vop[2][2][VOPS][64];
  __shared__ uint32_t flag[2][4];
  const uint32_t tid = threadIdx.x, lane = tid & 63, wv = tid >> 6, m = lane & 15, j = lane >> 4;
  const uint32_t head = blockIdx.y, z = blockIdx.z, G = a.hq / a.c.heads;
  // the workgroup's sequence and its part of that sequence's pairs
  uint32_t i = 0, part_i = 0, before = 0;
  bool found = false;
  for (uint32_t b = 0; b < a.r.n && !found; b += 64) {
    uint32_t nt = 0;
    if (b + lane < a.r.n) {
      const uint32_t o0 = a.r.off[b + lane], o1 = a.r.off[b + lane + 1];
      const uint64_t pairs = o1 > o0 && o1 <= a.r.rows ? (uint64_t)(o1 - o0) * G : 0;
      nt = pairs > kFewPairs ? (uint32_t)((pairs + PW - 1) / PW) : 0;
    }
    uint32_t sum = nt;
#pragma unroll
    for (int k = 1; k < 64; k <<= 1) {
      const uint32_t o = __shfl_up(sum, k, 64);
      if (lane >= (uint32_t)k) sum += o;
    }
    const unsigned long long hit = __ballot(before + sum > blockIdx.x);
    if (hit) {
      const int f = __ffsll((long long)hit) - 1;
      i = b + f;
      part_i = blockIdx.x - before - (__shfl(sum, f, 64) - __shfl(nt, f, 64));
      found = true;
    } else {
      before += __shfl(sum, 63, 64);
    }
  }
  if (!found) return;
  const uint32_t row0 = a.r.off[i], len = a.r.off[i + 1] - row0;
  const uint32_t q = a.r.seq ? a.r.seq[i] : i;
  const bool ok = q < a.c.seqs;
  const uint32_t pos = a.r.pos[i], last = pos + len - 1;
  const uint64_t all = (uint64_t)len * G;
  const uint64_t c0 = (uint64_t)part_i * PW;
  const View view(last, a.c.slots);
  const uint32_t p_lo = pos + (uint32_t)(c0 / G), p_hi = pos + (uint32_t)((min(all, c0 + PW) - 1) / G);
  // before the ring wraps, slots past the last row's position hold nothing
  // that any of the pairs sees
  const uint32_t seen = last < a.c.slots ? p_hi + 1 : view.live;
  const uint32_t tiles = ok ? (seen + 31) / 32 : 0u;
  const uint32_t t0 = z * a.tps, t1 = z + 1 == a.nsplit ? tiles : min(tiles, t0 + a.tps);

  bf16x8_t qo[NQ][NP][D / 32];
  uint32_t p[NQ], wave_hi = 0;
  uint64_t c[NQ];
#pragma unroll
  for (int n = 0; n < NQ; n++) {
    c[n] = c0 + (wv * NQ + n) * 16 + m;
    const bool on = c[n] < all;
    const uint32_t t = on ? (uint32_t)(c[n] / G) : 0, g = on ? (uint32_t)(c[n] % G) : 0;
    p[n] = pos + t;
    query_ops<T, D, NP>(a.q, row0 + t, head * G + g, j, on, vec, qo[n]);
  }
  {
    const uint64_t w0 = c0 + wv * NQ * 16;
    wave_hi = w0 < all ? pos + (uint32_t)((min(all, w0 + NQ * 16) - 1) / G) : 0;
    if (w0 >= all) wave_hi = pos;   // (its columns count for nothing)
  }
  const float sc = a.scale * kLog2e;
  Acc<D, NPP> acc[NQ];
#pragma unroll
  for (int n = 0; n < NQ; n++) acc[n].clear();
  const uint8_t* base = record_of(a.c, ok ? q : 0, head, 0);
  Raw<D> raw;
  const uint32_t half = wv & 1;   // 0: keys, 1: values
  auto load = [&](uint32_t step) {
    const uint32_t tile = min(step + (wv >> 1), tiles - 1);
    if (half == 0) load_k(raw, base + (uint64_t)tile * (34 * D), lane);
    else load_v(raw, base + (uint64_t)tile * (34 * D), lane);
  };
  auto stage = [&](uint32_t step, uint32_t buf) {
    const uint32_t rt = wv >> 1, tile = step + rt;
    uint32_t bad;
    if (half == 0) {
      bad = has255(raw.ks);
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const float ksc = scale_of(raw.ks, h);
        const bool nan = ((raw.ks >> (8 * h)) & 0xFF) == 255;
#pragma unroll
        for (int d = 0; d < D / 32; d++) {
          u32x4_t o = __builtin_bit_cast(u32x4_t, key_op<D>(raw, h, d, ksc));
#pragma unroll
          for (int e = 0; e < 4; e++) o[e] = nan ? 0x7FC07FC0u : o[e];
          kop[buf][rt][h * (D / 32) + d][lane] = __builtin_bit_cast(bf16x8_t, o);
        }
      }
    } else {
      bad = has255(raw.vs[0]) | has255(raw.vs[1]);
      float vsc[8];
#pragma unroll
      for (int e = 0; e < 8; e++) {
        const uint32_t slot = tile * 32 + 16 * (e / 4) + 4 * j + e % 4;
        const uint32_t b = (raw.vs[e / 4] >> (8 * (e % 4))) & 0xFF;
        vsc[e] = slot >= view.live || b == 255 ? 0.0f : __builtin_bit_cast(float, b << 23);
      }
      static_for<D / 32>([&](auto u_) {
        constexpr int u = decltype(u_)::value;
        val_ops<D, u>(raw, vsc, vop[buf][rt][2 * u][lane], vop[buf][rt][2 * u + 1][lane]);
      });
    }
    const bool any = __any(bad);
    if (lane == 0) flag[buf][wv] = any;
  };
  uint32_t buf = 0;
  if (t0 < t1) {
    load(t0);
    stage(t0, 0);
  }
  __syncthreads();
  for (uint32_t step = t0; step < t1; step += 2) {
    const bool more = step + 2 < t1;
    if (more) load(step + 2);
#pragma unroll
    for (int rt = 0; rt < 2; rt++) {
      const uint32_t tile = step + rt;
      if (tile >= t1) break;
      // a tile past every position of the wave's pairs (no wrap)
      if (last < a.c.slots && tile * 32 > wave_hi) continue;
      const bool whole = view.whole(tile, last, p_lo);
      const bool bad = flag[buf][2 * rt + 1];
      f32x4_t s[NQ][2];
#pragma unroll
      for (int n = 0; n < NQ; n++) s[n][0] = s[n][1] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int d = 0; d < D / 32; d++)
#pragma unroll
        for (int h = 0; h < 2; h++) {
          const bf16x8_t ko = kop[buf][rt][h * (D / 32) + d][lane];
#pragma unroll
          for (int n = 0; n < NQ; n++)
#pragma unroll
            for (int u = 0; u < NP; u++)
              s[n][h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ko, qo[n][u][d], s[n][h], 0, 0, 0);
        }
      bf16x8_t po[NQ][NPP];
#pragma unroll
      for (int n = 0; n < NQ; n++) {
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] = s[n][e / 4][e % 4] * sc;
        if (!whole) {
#pragma unroll
          for (int e = 0; e < 8; e++)
            if (!view.sees(tile * 32 + 16 * (e / 4) + 4 * j + e % 4, p[n])) x[e] = -INFINITY;
        }
        if (bad) {
          const uint8_t* vs = base + (uint64_t)tile * (34 * D) + 33 * D + j * 8;
          for (int e = 0; e < 8; e++) {
            if (!view.sees(tile * 32 + 16 * (e / 4) + 4 * j + e % 4, p[n])) continue;
            for (int b = 0; b < D / 32; b++)
              if (vs[b * 32 + e] == 255) acc[n].nan |= 1u << b;
          }
        }
        acc[n].soften(x, po[n]);
      }
#pragma unroll
      for (int t = 0; t < D / 16; t++) {
        const bf16x8_t vo = vop[buf][rt][t][lane];
#pragma unroll
        for (int n = 0; n < NQ; n++)
#pragma unroll
          for (int u = 0; u < NPP; u++)
            acc[n].o[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vo, po[n][u], acc[n].o[t], 0, 0, 0);
      }
    }
    if (more) stage(step + 2, buf ^ 1);
    __syncthreads();
    buf ^= 1;
  }
#pragma unroll
  for (int n = 0; n < NQ; n++) {
    const float l = pair_sum(acc[n].l);
    const uint32_t nan = pair_or(acc[n].nan);
    if (c[n] >= all) continue;
    const uint32_t row = row0 + (uint32_t)(c[n] / G), hd = head * G + (uint32_t)(c[n] % G);
    if (a.nsplit > 1) {
      float* part = a.part + (((uint64_t)row * a.hq + hd) * a.nsplit + z) * (D + 2);
#pragma unroll
      for (int i4 = 0; i4 < 4; i4++)
#pragma unroll
        for (int t = 0; t < D / 16; t++) {
          const uint32_t d = j * (D / 4) + i4 * (D / 16) + t;
          part[2 + d] = (nan >> (d / 32)) & 1 ? __builtin_nanf("") : acc[n].o[t][i4];
        }
      if (j == 0) {
        part[0] = acc[n].m;
        part[1] = l;
      }
    } else {
      float f;
      const float den = finish_sum<T>(acc[n].m, l, a.sink, hd, &f);
      const float inv = ok && den != 0.0f ? f / den : 0.0f;
      T* o = (T*)a.o.p + (uint64_t)row * a.o.row + (uint64_t)hd * a.o.head + j * (D / 4);
      float y[D / 4];
#pragma unroll
      for (int i4 = 0; i4 < 4; i4++)
#pragma unroll
        for (int t = 0; t < D / 16; t++) {
          const uint32_t d = j * (D / 4) + i4 * (D / 16) + t;
          const float v = acc[n].o[t][i4] * inv;
          y[i4 * (D / 16) + t] = (nan >> (d / 32)) & 1 ? __builtin_nanf("") : v;
        }
#pragma unroll
      for (int k = 0; k < D / 32; k++) {
        float t8[8];
#pragma unroll
        for (int e = 0; e < 8; e++) t8[e] = y[8 * k + e];
        store8(o + 8 * k, vec, t8);
      }
    }
  }
}

// The pieces of a (row, query head), a wave each: weights 2^(m_z - M), then
// the sink, then the division. The few-row kernel writes no piece past its
// sequence's last slot; the other one writes all of them.
template <typename T, int D>
__global__ __launch_bounds__(256) void k_kv4_join(Kv4Attend a) {
  constexpr uint32_t R = D / 32;
  const uint32_t lane = threadIdx.x & 63;
  const uint64_t w = (uint64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const uint32_t row = (uint32_t)(w / a.hq), hd = (uint32_t)(w % a.hq);
  if (row >= a.r.rows) return;
  uint32_t i = row, len = 1;
  if (a.r.off) {
    i = find_seq(a.r.off, a.r.n, row);
    const uint32_t o0 = a.r.off[i], o1 = a.r.off[i + 1];
    if (row < o0 || row >= o1 || o1 > a.r.rows) return;
    len = o1 - o0;
  } else if (row >= a.r.n) {
    return;
  }
  const uint32_t q = a.r.seq ? a.r.seq[i] : i;
  const View view(a.r.pos[i] + len - 1, a.c.slots);
  uint32_t nz = min(a.nsplit, ((view.live + 31) / 32 + a.tps - 1) / a.tps);
  if (q >= a.c.seqs) nz = 0;
  const float* part = a.part + ((uint64_t)row * a.hq + hd) * a.nsplit * (D + 2);
  float M = -INFINITY;
  for (uint32_t z = lane; z < nz; z += 64) M = fmaxf(M, part[(uint64_t)z * (D + 2)]);
  M = wmax(M);
  float l = 0.0f, o[(R + 1) / 2] = {};
  for (uint32_t z = 0; z < nz; z++) {
    const float* p = part + (uint64_t)z * (D + 2);
    const float m = p[0];
    const float f = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - M);
    l += p[1] * f;
#pragma unroll
    for (uint32_t u = 0; u < (R + 1) / 2; u++)
      if (lane + 64 * u < D) o[u] += p[2 + lane + 64 * u] * f;
  }
  float f;
  const float den = finish_sum<T>(M, l, a.sink, hd, &f);
#pragma unroll
  for (uint32_t u = 0; u < (R + 1) / 2; u++)
    if (lane + 64 * u < D)
      ((T*)a.o.p)[(uint64_t)row * a.o.row + (uint64_t)hd * a.o.head + lane + 64 * u] =
          (T)(nz && den != 0.0f ? o[u] * f / den : 0.0f);
}

template <typename T>
bool on16(const Kv4Mat& x) {
  return ((uintptr_t)x.p | (x.row * sizeof(T)) | (x.head * sizeof(T))) % 16 == 0;
}

// f(T{}, integral_constant hd) for a call's element type and head size
template <typename F>
hipError_t by_type(int type, uint32_t hd, F&& f) {
  auto by_hd = [&](auto t) -> hipError_t {
    switch (hd) {
      case 32: return f(t, std::integral_constant<int, 32>{});
      case 64: return f(t, std::integral_constant<int, 64>{});
      case 128: return f(t, std::integral_constant<int, 128>{});
      default: return hipErrorInvalidValue;
    }
  };
  switch (type) {
    case ET_F32: return by_hd(float{});
    case ET_BF16: return by_hd(__bf16{});
    case ET_F16: return by_hd(_Float16{});
    default: return hipErrorInvalidValue;
  }
}

}  // namespace

hipError_t launch_kv4_write(const Kv4& c, const Kv4Rows& r, int type, const Kv4Mat& k, const Kv4Mat& v,
                            const float* gk, const float* gq, const Kv4Mat* q, uint32_t qheads, hipStream_t st) {
  if (!c.data || !r.pos || c.slots == 0 || (q && type != ET_F32)) return hipErrorInvalidValue;
  if (r.rows == 0 || r.n == 0) return hipSuccess;
  return by_type(type, c.hd, [&](auto t, auto d) -> hipError_t {
    using T = decltype(t);
    constexpr int D = decltype(d)::value;
    const Kv4Mat none{nullptr, 0, 0};
    const uint32_t vec = on16<T>(k) && on16<T>(v) && (!q || on16<T>(*q));
    const uint32_t hmax = q ? std::max(c.heads, qheads) : c.heads;
    hipLaunchKernelGGL((k_kv4_write<T, D>), dim3((r.rows + 31) / 32, hmax, q ? 3 : 2), dim3(4 * D), 0, st, c, r, k, v,
                       vec, gk, gq, q ? *q : none, c.heads);
    return hipGetLastError();
  });
}

hipError_t launch_kv4_read(const Kv4& c, const Kv4Rows& r, int type, const Kv4Mat& k, const Kv4Mat& v,
                           hipStream_t st) {
  if (!c.data || !r.pos || c.slots == 0) return hipErrorInvalidValue;
  if (r.rows == 0 || r.n == 0) return hipSuccess;
  return by_type(type, c.hd, [&](auto t, auto d) -> hipError_t {
    using T = decltype(t);
    constexpr int D = decltype(d)::value;
    hipLaunchKernelGGL((k_kv4_read<T, D>), dim3((r.rows + 31) / 32, c.heads, 2), dim3(4 * D), 0, st, c, r, k, v,
                       (uint32_t)(on16<T>(k) && on16<T>(v)));
    return hipGetLastError();
  });
}

// Pieces of the slots: enough workgroups to fill the chip a few times over,
// of at least a tile a wave.
void kv4_split(const Kv4& c, uint32_t n, uint32_t rows, bool ragged, uint32_t hq, uint64_t live, uint32_t* nsplit,
               uint32_t* tps) {
  const uint64_t slots = live ? std::min<uint64_t>(live, c.slots) : c.slots;
  const uint32_t tiles = (uint32_t)((slots + 31) / 32);
  const uint64_t G = hq / c.heads;
  const uint64_t base = ragged ? ((uint64_t)rows * G + 127) / 128 * c.heads : (uint64_t)n * c.heads * ((G + 15) / 16);
  const uint64_t want = ragged ? 512 : 1024;
  uint32_t s = (uint32_t)std::min<uint64_t>((want + base - 1) / std::max<uint64_t>(base, 1), 128);
  s = std::max(1u, std::min(s, tiles / 4));
  *tps = (std::max(tiles, 1u) + s - 1) / s;
  if (ragged) *tps = (*tps + 1) & ~1u;
  *nsplit = (std::max(tiles, 1u) + *tps - 1) / *tps;
}

hipError_t launch_kv4_attend(const Kv4Attend& a, int type, hipStream_t st) {
  if (!a.c.data || !a.r.pos || a.c.slots == 0 || a.c.heads == 0 || a.hq == 0 || a.hq % a.c.heads || a.tps == 0 ||
      a.nsplit == 0 || a.nsplit > 65535 || (a.nsplit > 1 && !a.part))
    return hipErrorInvalidValue;
  if (a.r.rows == 0 || a.r.n == 0) return hipSuccess;
  return by_type(type, a.c.hd, [&](auto t, auto d) -> hipError_t {
    using T = decltype(t);
    constexpr int D = decltype(d)::value;
    const uint32_t vec = on16<T>(a.q) && on16<T>(a.o);
    const uint32_t G = a.hq / a.c.heads;
    const uint32_t nt16 = a.r.off ? 1 : (G + 15) / 16;
    hipLaunchKernelGGL((k_kv4_few<T, D>), dim3(a.r.n * a.c.heads * nt16, a.nsplit), dim3(256), 0, st, a, vec, nt16);
    if (a.r.off) {
      constexpr uint32_t PW = Many<T, D>::pairs;
      const uint32_t gx = (uint32_t)(((uint64_t)a.r.rows * G + PW - 1) / PW) + a.r.n;
      hipLaunchKernelGGL((k_kv4_many<T, D>), dim3(gx, a.c.heads, a.nsplit), dim3(256), 0, st, a, vec);
    }
    if (a.nsplit > 1)
      hipLaunchKernelGGL((k_kv4_join<T, D>), dim3((uint32_t)(((uint64_t)a.r.rows * a.hq + 3) / 4)), dim3(256), 0, st, a);
    return hipGetLastError();
  });
}

}  // namespace ana
