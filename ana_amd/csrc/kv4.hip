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

// whether a sequence has a place in the cache, and positions below 2^31 (so
// that none of its rows' passes 2^32)
__device__ __forceinline__ bool has_place(const Kv4& c, uint32_t q, uint32_t pos) {
  return q < c.seqs && pos < 0x80000000u;
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
  const uint32_t pos = r.pos[a.i];
  a.q = r.seq ? r.seq[a.i] : a.i;
  a.ok = has_place(c, a.q, pos);
  a.p = pos + (row - o0);
  a.last = pos + (o1 - 1 - o0);
  return a;
}

__device__ __forceinline__ uint8_t* record_of(const Kv4& c, uint32_t q, uint32_t head, uint32_t tile) {
  return c.data + q * c.seq_bytes + ((uint64_t)head * c.tiles + tile) * kv4_record(c.hd);
}

// A call's keys and values into the cache: a workgroup takes 32 rows of one
// head, eight dims a thread (a slot's codes of one lane of the attention are
// hd / 4 dims of a key and hd / 16 of a value). z = 0 the keys, 1 the
// values, 2 the query rows, which are only qk-normed in place. The block's
// largest magnitude comes from the quad of threads that share it, in the
// floats' bits, where a block that is not finite shows itself too.
// A row that a later one of the call overwrites (a ring shorter than the
// call), and rows of a sequence that the call lists a second time with a
// place, are left out, so that what is stored does not depend on the order of
// the threads.
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
    if (a.ok) store8(p, vec, x);
    return;
  }
  bool put = a.ok && a.last - a.p < c.slots;
  if (r.seq && put) {
    uint32_t dup = 0;
    for (uint32_t j = sub; j < a.i; j += TPR)
      if (r.seq[j] == a.q && has_place(c, a.q, r.pos[j]) && (!r.off || r.off[j + 1] > r.off[j])) dup = 1;
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
  // (to the nearest code, ties to the even one, past the largest to it; the
  // same in integer steps took 14 instructions a value where this takes 1.5,
  // and 32 us where it takes 28 for 16384 rows of 8 heads of 128 in bf16)
  uint32_t w = 0;
  static_for<4>([&](auto u) {
    constexpr int e = 2 * decltype(u)::value;
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[e] * f, x[e + 1] * f, 1.0f, decltype(u)::value);
  });
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
// (zeros for a sequence without a place in the cache). A thread takes 16
// bytes of the outputs, so that a store's lanes write whole lines (with eight
// f32 a thread, in two stores of every other 16 bytes, 8384 rows of 12 heads
// of 64 took 37 us for 20).
template <typename T, int D>
__global__ __launch_bounds__(32 * D * sizeof(T) / 16) void k_kv4_read(Kv4 c, Kv4Rows r, Kv4Mat k, Kv4Mat v, uint32_t vec) {
  constexpr uint32_t E = 16 / sizeof(T), TPR = D / E;   // outputs a thread, threads a row
  const uint32_t tid = threadIdx.x, sub = tid % TPR, row = blockIdx.x * 32 + tid / TPR, head = blockIdx.y;
  const uint32_t i0 = r.off ? find_seq(r.off, r.n, blockIdx.x * 32) : 0;
  const RowAt a = row_at(c, r, row, i0);
  if (!a.on) return;
  uint32_t w = 0, b = 2;
  if (a.ok) {
    const uint32_t slot = a.p % c.slots, s = slot % 32, h = s / 16, m = s % 16, dim = sub * E;
    const uint8_t* rec = record_of(c, a.q, head, slot / 32);
    auto codes = [&](const uint8_t* at) -> uint32_t {
      if constexpr (E == 8) return *reinterpret_cast<const uint32_t*>(at);
      else return *reinterpret_cast<const uint16_t*>(at);
    };
    if (blockIdx.z == 0) {
      const uint32_t j = dim / (D / 4);
      w = codes(rec + (j * 16 + m) * (D / 4) + h * (D / 8) + dim % (D / 4) / 2);
      b = rec[32 * D + (dim / 32 * 16 + m) * 2 + h];
    } else {
      const uint32_t j = m / 4, e = h * 4 + m % 4;
      // (a lane of the attention has D / 16 dims of a slot, its neighbours' are D / 4 bytes on)
      const uint8_t* at = rec + 16 * D + (j * 16 + dim / (D / 16)) * (D / 4) + e * (D / 32) + dim % (D / 16) / 2;
      if constexpr (E <= D / 16) {
        w = codes(at);
      } else if constexpr (D == 64) {
        w = *reinterpret_cast<const uint16_t*>(at) | (uint32_t)*reinterpret_cast<const uint16_t*>(at + D / 4) << 16;
      } else {
#pragma unroll
        for (uint32_t u = 0; u < E / 2; u++) w |= (uint32_t)at[u * (D / 4)] << (8 * u);
      }
      b = rec[33 * D + (dim / 32 * 4 + j) * 8 + e];
    }
  }
  const float f = b == 255 ? __builtin_nanf("") : __builtin_bit_cast(float, b << 23);
  float x[E];
  static_for<E / 2>([&](auto u) {
    const f32x2_t t = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, decltype(u)::value);
    x[2 * u] = t[0] * f;
    x[2 * u + 1] = t[1] * f;
  });
  const Kv4Mat& dst = blockIdx.z == 0 ? k : v;
  T* p = (T*)dst.p + (uint64_t)row * dst.row + (uint64_t)head * dst.head + sub * E;
  if (vec) {
    typedef T vec_t __attribute__((ext_vector_type(E)));
    vec_t y;
#pragma unroll
    for (uint32_t e = 0; e < E; e++) y[e] = (T)x[e];
    *reinterpret_cast<vec_t*>(p) = y;
  } else {
#pragma unroll
    for (uint32_t e = 0; e < E; e++) p[e] = (T)x[e];
  }
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
// is taken in NPP parts (f32: three, the whole of it; 16-bit outputs: two, 16
// bits of it, which is a sixteenth of half an f16's step), each product of parts
// exact in the f32 sum.

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

typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
// split8 for probabilities (never next to the largest float): a part of two
// in one conversion, and what it leaves of each, x - part, in one dot product
// of two with (-1, 0) or (0, -1), exact as every term is
template <int N>
__device__ __forceinline__ void split8_p(const float (&x)[8], bf16x8_t (&o)[N]) {
  // (kept from the compiler, which writes the first as the inline constant
  // -1.0, and that one is the second)
  uint32_t c0 = 0x0000BF80u, c1 = 0xBF800000u;
  asm("" : "+v"(c0), "+v"(c1));
  const bf16x2_t m0 = __builtin_bit_cast(bf16x2_t, c0), m1 = __builtin_bit_cast(bf16x2_t, c1);
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    f32x2_t r = {x[e], x[e + 1]};
#pragma unroll
    for (int n = 0; n < N; n++) {
      const bf16x2_t h = __builtin_convertvector(r, bf16x2_t);
      o[n][e] = h[0];
      o[n][e + 1] = h[1];
      if (n + 1 < N) {
        r[0] = __builtin_amdgcn_fdot2_f32_bf16(h, m0, r[0], false);
        r[1] = __builtin_amdgcn_fdot2_f32_bf16(h, m1, r[1], false);
      }
    }
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
__device__ __forceinline__ void val_ops(const uint32_t (&w)[D / 16], const float (&sc)[8], bf16x8_t& a, bf16x8_t& b) {
  uint32_t x[8];
  static_for<8>([&](auto e_) {
    constexpr int e = decltype(e_)::value, byte = e * (D / 32) + U;
    x[e] = two_of<byte % 4>(w[byte / 4], sc[e]);
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

// What a workgroup's pairs see. Slot s holds the position back(s) before the
// sequence's last one, last; a pair `ago` positions before the last sees the
// slots that are live and as far back or farther.
struct View {
  uint32_t slots, cur, live;   // the ring's; the last position's; live ones
  __device__ __forceinline__ View(uint32_t last, uint32_t slots_) : slots(slots_) {
    cur = last % slots;
    live = last < slots ? last + 1 : slots;
  }
  __device__ __forceinline__ uint32_t back(uint32_t s) const { return s <= cur ? cur - s : cur + slots - s; }
  __device__ __forceinline__ bool sees(uint32_t s, uint32_t ago) const { return s < live && back(s) >= ago; }
  // whether every slot of tile t is live and `ago` back or more (those that
  // are not are the `ago` slots up to cur, round the ring)
  __device__ __forceinline__ bool whole(uint32_t t, uint32_t ago) const {
    const uint32_t s0 = t * 32, s1 = s0 + 31;
    if (s1 >= live) return false;
    if (ago == 0) return true;
    if (ago >= slots) return false;
    return ago <= cur + 1 ? (s1 + ago < cur + 1 || s0 > cur) : (s1 + ago < cur + 1 + slots && s0 > cur);
  }
};

constexpr float kLog2e = 1.4426950408889634f;
// A piece's partial result: its maximum and sum, then (on 16 bytes) its D
// outputs. The first piece's third word says how many there are, or that the
// only one was finished where it was made.
constexpr uint32_t kPartHead = kKv4PartHead, kDone = 0xFFFFFFFFu;
// pairs of a sequence up to which the few-row kernel takes it
constexpr uint32_t kFewPairs = 16;
// The pieces that `tiles` tiles are cut into, at most nsplit of at least
// `least` tiles: the tiles of each but the last.
constexpr uint32_t kFewTiles = 4, kManyTiles = 8;
__device__ __forceinline__ uint32_t piece_tiles(uint32_t tiles, uint32_t nsplit, uint32_t least) {
  const uint32_t n = max(1u, min(nsplit, tiles / least));
  return (tiles + n - 1) / n;
}
// A running maximum is only raised once a score passes it by this much (in
// base 2): probabilities then reach 2^kSlack, which costs f32 and bf16 no
// digit, and most tiles rescale nothing.
constexpr float kSlack = 10.0f;

// The queries' scale: f32 queries carry it (times log2 e) into their parts,
// 16-bit ones enter as they are and only take its sign
// (or, for a scale of 0, that).
template <typename T>
__device__ __forceinline__ float query_factor(float sc) {
  if constexpr (sizeof(T) == 4) return sc;
  return sc < 0.0f ? -1.0f : sc == 0.0f ? 0.0f : 1.0f;
}
template <typename T>
__device__ __forceinline__ float score_factor(float sc) {
  if constexpr (sizeof(T) == 4) return 1.0f;
  return sc == 0.0f ? 1.0f : fabsf(sc);   // (a masked score of -inf must stay one)
}
// the query operand of a pair: dims j D / 4 + 8 s + e of its row, in parts
template <typename T, int D, int NP>
__device__ __forceinline__ void query_ops(const Kv4Mat& q, uint32_t row, uint32_t head, uint32_t j, bool on, bool vec,
                                          float f, bf16x8_t (&o)[NP][D / 32]) {
  const T* p = (const T*)q.p + (uint64_t)row * q.row + (uint64_t)head * q.head + j * (D / 4);
#pragma unroll
  for (int s = 0; s < D / 32; s++) {
    float x[8] = {};
    if (on) load8(p + 8 * s, vec, x);
#pragma unroll
    for (int e = 0; e < 8; e++) x[e] *= f;
    bf16x8_t t[NP];
    split8(x, t);
#pragma unroll
    for (int n = 0; n < NP; n++) o[n][s] = t[n];
  }
}

// the weight of what was summed with maximum m, and the denominator, with the
// head's sink
__device__ __forceinline__ float finish_sum(float m, float l, const float* sink, uint32_t head, float* f) {
  *f = 1.0f;
  if (!sink) return l;
  const float s = sink[head] * kLog2e;
  const float n = fmaxf(m, s);
  if (s != s) return s;
  if (n == -INFINITY) return l;
  *f = __builtin_amdgcn_exp2f(m - n);
  return l * *f + __builtin_amdgcn_exp2f(s - n);
}

// blocks of values that are not finite among those a pair sees, a bit a block
// of dims (read again: the rare path)
template <int D>
__device__ __forceinline__ uint32_t nan_blocks(const uint8_t* rec, uint32_t tile, const View& view, uint32_t ago, uint32_t j) {
  uint32_t n = 0;
  const uint8_t* vs = rec + 33 * D + j * 8;
#pragma unroll 1
  for (uint32_t e = 0; e < 8; e++) {
    if (!view.sees(tile * 32 + 16 * (e / 4) + 4 * j + e % 4, ago)) continue;
#pragma unroll
    for (uint32_t b = 0; b < D / 32; b++) n |= vs[b * 32 + e] == 255 ? 1u << b : 0u;
  }
  return n;
}
// which of a lane's eight slots have a key that is not finite (some block of
// it), a bit each
template <int D>
__device__ __forceinline__ uint32_t nan_keys(const uint8_t* rec, uint32_t j) {
  uint32_t n = 0;
#pragma unroll 1
  for (uint32_t i = 0; i < 8 * (D / 32); i++) {
    const uint32_t e = i % 8, b = i / 8;
    n |= rec[32 * D + (b * 16 + 4 * j + e % 4) * 2 + e / 4] == 255 ? 1u << e : 0u;
  }
  return n;
}
// the value scales of slots that are not live, and of blocks that are not
// finite, as 2^-127
__device__ __forceinline__ void quiet_values(uint32_t (&vs)[2], uint32_t tile, uint32_t live, uint32_t j) {
#pragma unroll
  for (int e = 0; e < 8; e++) {
    const uint32_t mask = 0xFFu << (8 * (e % 4));
    if (tile * 32 + 16 * (e / 4) + 4 * j + e % 4 >= live || (vs[e / 4] & mask) == mask) vs[e / 4] &= ~mask;
  }
}
template <int D>
__device__ __forceinline__ bool not_finite(const Raw<D>& r) {
  // (by the scales as they are used: fewer instructions than by the bytes)
  uint32_t t = max(__builtin_bit_cast(uint32_t, scale_of(r.ks, 0)), __builtin_bit_cast(uint32_t, scale_of(r.ks, 1)));
#pragma unroll
  for (int e = 0; e < 8; e++) t = max(t, __builtin_bit_cast(uint32_t, scale_of(r.vs[e / 4], e % 4)));
  return t == 0x7F800000u;
}

// u's DPP move within its quad of lanes
template <int CTRL>
__device__ __forceinline__ uint32_t quad(uint32_t u) {
  return (uint32_t)__builtin_amdgcn_mov_dpp((int)u, CTRL, 0xF, 0xF, true);
}
template <int CTRL>
__device__ __forceinline__ uint32_t quad(float f) { return quad<CTRL>(__builtin_bit_cast(uint32_t, f)); }

// Few rows (up to 16 pairs of one sequence and key head): one workgroup per
// (sequence, key head, piece of the slots), its four waves taking every
// fourth tile with the next one's loads in flight, each with a running
// softmax of its own; they meet in LDS.
//
// Pairs are few against the 16 columns of an MFMA, so with NC = 2 or 4 a pair
// takes NC neighbouring columns, one for each part: of the query in the first
// product (whose columns' sum is the score) and of the probability in the
// second, one MFMA each where NC = 1 takes one a part. A lane of the NC then
// has exponentials to take for only 8 / NC of its slots, which its neighbours
// get by DPP moves. (256 sequences of 2048 slots, 12 heads of 64, f32: a tile
// costs 188 vector instructions and 8 MFMAs, 80 us or 5.3 TB/s with the vector
// units busy 82% of it; with NC = 1 it was 296 and 24, 128 us.)
template <typename T, int D, int NC>
__global__ __launch_bounds__(256, (D == 128 ? 3 : 4) - (NC == 1)) void k_kv4_few(Kv4Attend a, uint32_t vec, uint32_t ncol) {
  constexpr int NP = Parts<T>::q, QP = NC == 1 ? NP : 1, NPP = NC == 1 ? Parts<T>::p : 1;
  constexpr int PC = 16 / NC;          // pairs a workgroup
  constexpr int OWN = NC == 1 ? 4 : 4 / NC;  // slots of four that a lane takes exponentials of
  __shared__ float om[4][16][D + 4];
  __shared__ float mm[4][16], ll[4][16];
  const uint32_t tid = threadIdx.x, lane = tid & 63, m = lane & 15, j = lane >> 4;
  const uint32_t wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  uint32_t w = blockIdx.x;
  const uint32_t sub = w % ncol;
  w /= ncol;
  const uint32_t head = w % a.c.heads, i = w / a.c.heads, z = blockIdx.y;
  const uint32_t G = a.hq / a.c.heads;
  uint32_t row0 = i, len = 1;
  if (a.r.off) {
    const uint32_t o0 = a.r.off[i], o1 = a.r.off[i + 1];
    if (o1 <= o0 || o1 > a.r.rows) return;
    row0 = o0;
    len = o1 - o0;
    if (len > kFewPairs || len * G > kFewPairs) return;
  }
  const uint32_t q = a.r.seq ? a.r.seq[i] : i;
  const uint32_t pos = a.r.pos[i], last = pos + len - 1;
  const uint32_t c0 = sub * PC, np = min(len * G - c0, (uint32_t)PC);   // the pairs here
  const bool ok = has_place(a.c, q, pos);
  const View view(last, a.c.slots);
  const uint32_t tiles = ok ? (view.live + 31) / 32 : 0u;
  const uint32_t per = piece_tiles(tiles, a.nsplit, kFewTiles);
  const uint32_t t0 = z * per, t1 = min(tiles, t0 + per);
  if (z && t0 >= t1) return;
  const bool split = tiles > per;
  const uint32_t pm = m / NC, part = m % NC;
  const uint32_t t = (c0 + pm) / G, g = (c0 + pm) % G;
  const float sc = a.scale * kLog2e;
  bf16x8_t qo[QP][D / 32];
  {
    bf16x8_t all[NP][D / 32];
    query_ops<T, D, NP>(a.q, row0 + t, head * G + g, j, pm < np, vec, query_factor<T>(sc), all);
    if constexpr (NC == 1) {
#pragma unroll
      for (int n = 0; n < NP; n++)
#pragma unroll
        for (int d = 0; d < D / 32; d++) qo[n][d] = all[n][d];
    } else {
#pragma unroll
      for (int d = 0; d < D / 32; d++) {
        u32x4_t o = __builtin_bit_cast(u32x4_t, all[0][d]);
        if constexpr (NP > 1) {
          const u32x4_t o1 = __builtin_bit_cast(u32x4_t, all[1][d]), o2 = __builtin_bit_cast(u32x4_t, all[NP - 1][d]);
#pragma unroll
          for (int e = 0; e < 4; e++) o[e] = part == 0 ? o[e] : part == 1 ? o1[e] : part < NP ? o2[e] : 0u;
        }
        qo[0][d] = __builtin_bit_cast(bf16x8_t, o);
      }
    }
  }
  const float sf = score_factor<T>(sc);
  const uint32_t ago = len - 1 - t;   // positions from the pair's to the last
  // a probability's part of this column, p & pm1 less p & pm0: eight bits each
  const uint32_t pm1 = part == 0 ? 0xFFFF0000u : part == 1 ? 0xFFFFFF00u : 0xFFFFFFFFu;
  const uint32_t pm0 = part == 0 ? 0u : part == 1 ? 0xFFFF0000u : part == 2 ? 0xFFFFFF00u : 0xFFFFFFFFu;
  f32x4_t o[D / 16];
#pragma unroll
  for (int d = 0; d < D / 16; d++) o[d] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
  float mx = -INFINITY, l = 0.0f;
  uint32_t nan = 0;
  const uint8_t* base = record_of(a.c, ok ? q : 0, head, 0);

  auto load = [&](Raw<D>& r, uint32_t tile) {
    const uint8_t* rec = base + (uint64_t)min(tile, t1 - 1) * (34 * D);
    load_k(r, rec, lane);
    load_v(r, rec, lane);
  };
  auto tile_of = [&](Raw<D>& r, uint32_t tile) {
    const bool whole = view.whole(tile, len - 1);
    const bool bad = __any(not_finite(r));
    f32x4_t s[2];   // (a key that is not finite makes its own slot's score anything)
#pragma unroll
    for (int h = 0; h < 2; h++) {
      s[h] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
      const float ksc = scale_of(r.ks, h);
#pragma unroll
      for (int d = 0; d < D / 32; d++) {
        const bf16x8_t ko = key_op<D>(r, h, d, ksc);
#pragma unroll
        for (int n = 0; n < QP; n++) s[h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ko, qo[n][d], s[h], 0, 0, 0);
      }
    }
    // the scores that this lane goes on with: all, or (NC > 1) of slots 4 j +
    // i those with i mod NC its column's, over the NC columns' sum
    float x[2 * OWN];
#pragma unroll
    for (int h = 0; h < 2; h++) {
      if constexpr (NC == 1) {
#pragma unroll
        for (int e = 0; e < 4; e++) x[4 * h + e] = s[h][e];
      } else {
        float u[2];
#pragma unroll
        for (int e = 0; e < 2; e++) {
          u[e] = part & 1 ? s[h][2 * e + 1] : s[h][2 * e];
          if constexpr (NP > 1)
            u[e] += __builtin_bit_cast(float, quad<0xB1>(part & 1 ? s[h][2 * e] : s[h][2 * e + 1]));
        }
        if constexpr (NC == 2) {
          x[2 * h] = u[0];
          x[2 * h + 1] = u[1];
        } else {
          x[h] = (part & 2 ? u[1] : u[0]) + __builtin_bit_cast(float, quad<0x4E>(part & 2 ? u[0] : u[1]));
        }
      }
    }
    if (!whole || bad) {
      const uint32_t nk = bad ? nan_keys<D>(base + (uint64_t)tile * (34 * D), j) : 0;
#pragma unroll
      for (int e = 0; e < 2 * OWN; e++) {
        const uint32_t in4 = NC == 1 ? e % 4 : NC == 2 ? 2 * (e % 2) + part : part;
        if ((nk >> (4 * (e / OWN) + in4)) & 1) x[e] = __builtin_nanf("");
        if (!view.sees(tile * 32 + 16 * (e / OWN) + 4 * j + in4, ago)) x[e] = -INFINITY;
      }
      if (bad) nan |= nan_blocks<D>(base + (uint64_t)tile * (34 * D), tile, view, ago, j);
      quiet_values(r.vs, tile, view.live, j);
    }
    float top = x[0];
#pragma unroll
    for (int e = 1; e < 2 * OWN; e++) top = fmaxf(top, x[e]);
    if (__any(top * sf > mx + kSlack)) {
      if constexpr (NC >= 2) top = fmaxf(top, __builtin_bit_cast(float, quad<0xB1>(top)));
      if constexpr (NC >= 4) top = fmaxf(top, __builtin_bit_cast(float, quad<0x4E>(top)));
      const float n = fmaxf(mx, pair_max(top) * sf);
      const float f = n == mx ? 1.0f : __builtin_amdgcn_exp2f(mx - n);
      mx = n;
      l *= f;
#pragma unroll
      for (int d = 0; d < D / 16; d++) o[d] *= f;
    }
    const float b = mx == -INFINITY ? 0.0f : mx;
#pragma unroll
    for (int e = 0; e < 2 * OWN; e++) {
      x[e] = __builtin_amdgcn_exp2f(sizeof(T) == 4 ? x[e] - b : fmaf(x[e], sf, -b));
      l += x[e];
    }
    bf16x8_t po[NPP];
    if constexpr (NC == 1) {
      split8_p(x, po);
    } else {
      u32x4_t pk;
      static_for<4>([&](auto e_) {
        constexpr int e = decltype(e_)::value;   // slots 2 e and 2 e + 1 of the eight
        uint32_t v[2];
        static_for<2>([&](auto i_) {
          constexpr int i = decltype(i_)::value, in4 = (2 * e + i) % 4, h = e / 2;
          uint32_t u;
          if constexpr (NC == 4) u = quad<in4 * 0x55>(x[h]);
          else u = quad<in4 % 2 ? 0xF5 : 0xA0>(x[2 * h + in4 / 2]);
          v[i] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(float, u & pm1) - __builtin_bit_cast(float, u & pm0));
        });
        pk[e] = __builtin_amdgcn_perm(v[1], v[0], 0x07060302u);
      });
      po[0] = __builtin_bit_cast(bf16x8_t, pk);
    }
    float vsc[8];
#pragma unroll
    for (int e = 0; e < 8; e++) vsc[e] = scale_of(r.vs[e / 4], e % 4);
    static_for<D / 32>([&](auto u_) {
      constexpr int u = decltype(u_)::value;
      bf16x8_t v0, v1;
      val_ops<D, u>(r.v, vsc, v0, v1);
#pragma unroll
      for (int n = 0; n < NPP; n++) {
        o[2 * u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v0, po[n], o[2 * u], 0, 0, 0);
        o[2 * u + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v1, po[n], o[2 * u + 1], 0, 0, 0);
      }
    });
  };
  {
    Raw<D> ra, rb;
    uint32_t tile = t0 + wv;
    if (tile < t1) {
      load(ra, tile);
#pragma unroll 1
      for (;;) {
        load(rb, tile + 4);
        tile_of(ra, tile);
        tile += 4;
        if (tile >= t1) break;
        load(ra, tile + 4);
        tile_of(rb, tile);
        tile += 4;
        if (tile >= t1) break;
      }
    }
  }
  // the four waves meet
  l = pair_sum(l);
  nan = pair_or(nan);
  if constexpr (NC >= 2) l += __builtin_bit_cast(float, quad<0xB1>(l));
  if constexpr (NC >= 4) l += __builtin_bit_cast(float, quad<0x4E>(l));
  if (j == 0 && part == 0) {
    mm[wv][pm] = mx;
    ll[wv][pm] = l;
  }
#pragma unroll
  for (int i4 = 0; i4 < 4; i4++)
#pragma unroll
    for (int t16 = 0; t16 < D / 16; t16++) {
      const uint32_t d = j * (D / 4) + i4 * (D / 16) + t16;
      om[wv][m][d] = (nan >> (d / 32)) & 1 ? __builtin_nanf("") : o[t16][i4];
    }
  __syncthreads();
  for (uint32_t k = tid; k < np * D; k += 256) {
    const uint32_t pp = k / D, d = k % D;
    const float M = fmaxf(fmaxf(mm[0][pp], mm[1][pp]), fmaxf(mm[2][pp], mm[3][pp]));
    float lsum = 0.0f, y = 0.0f;
#pragma unroll
    for (int u = 0; u < 4; u++) {
      // (a wave without a seen slot has nothing, but a score that is not a number stays one)
      const float f = mm[u][pp] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mm[u][pp] - M);
      lsum += ll[u][pp] * f;
      float v = om[u][pp * NC][d];
#pragma unroll
      for (int n = 1; n < NC; n++) v += om[u][pp * NC + n][d];
      y += v * f;
    }
    const uint32_t row = row0 + (c0 + pp) / G, hd = head * G + (c0 + pp) % G;
    float* out = a.part + (((uint64_t)row * a.hq + hd) * a.nsplit + z) * (D + kPartHead);
    if (a.nsplit > 1 && d == 0) {
      if (z == 0) out[2] = __builtin_bit_cast(float, split ? (tiles + per - 1) / per : kDone);
      out[0] = M;
      out[1] = lsum;
    }
    if (split) {
      out[kPartHead + d] = y;
    } else {
      float f;
      const float den = finish_sum(M, lsum, a.sink, hd, &f);
      ((T*)a.o.p)[(uint64_t)row * a.o.row + (uint64_t)hd * a.o.head + d] = (T)(ok && den != 0.0f ? y * f / den : 0.0f);
    }
  }
}

// Many rows (more than 16 pairs of one sequence and key head): a workgroup
// takes 64 NQ pairs, 16 NQ a wave, over the tiles they see, one at a time.
// Its waves turn the tile into operands in LDS (a wave the keys of 16 slots,
// or half of the values' dims), lane by lane as the MFMAs want them, so every
// read and write there is a lane's own 16 bytes; the next tile's record is
// loaded a tile ahead, and two sets of operands leave one barrier a tile. The
// vector units (softmax and parts) and the matrix cores bind about equally,
// so what counts is that a SIMD holds three or four such waves, of different
// workgroups, to overlap them (16 pairs a wave, not 32, for f32: 61 -> 55 us
// for 16 prompts of 12 heads of 64). bf16 outputs take a probability rounded once to
// bf16, and the denominator the sum of the rounded ones: an output's error is then as
// large again as its own rounding's. (A second part, as the few-row kernel takes,
// is 8 of 24 MFMAs a tile and 16 pairs at hd 128: 735 us for 546, 2 x 1000 rows
// over 30000 positions, 16 query and 4 key heads of 128.)
template <typename T, int D>
struct Many {
  // pairs a wave: the queries' parts and the outputs share its registers
  static constexpr int NQ = Parts<T>::q > 1 ? 1 : 2;
  // waves a SIMD that the registers are kept to
  static constexpr int waves = D == 128 ? 3 : 4;
  static constexpr int NPP = Parts<T>::q == 1 ? 1 : Parts<T>::p;
  static constexpr uint32_t pairs = 64 * NQ;
};

template <typename T, int D>
__global__ __launch_bounds__(256, (Many<T, D>::waves)) void k_kv4_many(Kv4Attend a, uint32_t vec) {
  constexpr int NP = Parts<T>::q, NPP = Many<T, D>::NPP, NQ = Many<T, D>::NQ;
  constexpr uint32_t PW = Many<T, D>::pairs;
  constexpr int KS = D / 32, OPS = D / 16;     // steps of a key operand, operands of a tile's keys (values)
  constexpr bool F32 = sizeof(T) == 4;
  constexpr uint32_t OR = D + 4;               // a row of outputs in LDS
  constexpr size_t LDS = std::max<size_t>(2 * 2 * OPS * 64 * 16, 4 * 16 * OR * 4);
  __shared__ __align__(16) char lds[LDS];
  __shared__ uint32_t flag[2][4];
  bf16x8_t(*ops)[2][OPS][64] = reinterpret_cast<bf16x8_t(*)[2][OPS][64]>(lds);   // [buffer][keys, values]
  const uint32_t tid = threadIdx.x, lane = tid & 63, m = lane & 15, j = lane >> 4;
  const uint32_t wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  // (key heads first: workgroups go round the eight XCDs, and a sequence's
  // parts, each longer than the next, must not all meet the same ones)
  const uint32_t head = blockIdx.x % a.c.heads, tile_i = blockIdx.x / a.c.heads, z = blockIdx.y, G = a.hq / a.c.heads;
  // the workgroup's sequence and its part of that sequence's pairs
  uint32_t i = 0, part_i = 0, before = 0;
  bool found = false;
#pragma unroll 1
  for (uint32_t b = 0; b < a.r.n && !found; b += 64) {
    uint32_t nt = 0;
    if (b + lane < a.r.n) {
      const uint32_t o0 = a.r.off[b + lane], o1 = a.r.off[b + lane + 1];
      const uint32_t pairs = o1 > o0 && o1 <= a.r.rows ? (o1 - o0) * G : 0;
      nt = pairs > kFewPairs ? (pairs + PW - 1) / PW : 0;
    }
    uint32_t sum = nt;
#pragma unroll 1
    for (int k = 1; k < 64; k <<= 1) {
      const uint32_t o = __shfl_up(sum, k, 64);
      if (lane >= (uint32_t)k) sum += o;
    }
    const unsigned long long hit = __ballot(before + sum > tile_i);
    if (hit) {
      const int f = __ffsll((long long)hit) - 1;
      i = b + f;
      // (a sequence's last rows see the most: they start first)
      part_i = before + __shfl(sum, f, 64) - 1 - tile_i;
      found = true;
    } else {
      before += __shfl(sum, 63, 64);
    }
  }
  if (!found) return;
  i = __builtin_amdgcn_readfirstlane(i);
  part_i = __builtin_amdgcn_readfirstlane(part_i);
  const uint32_t row0 = a.r.off[i], len = a.r.off[i + 1] - row0;
  const uint32_t q = a.r.seq ? a.r.seq[i] : i;
  const uint32_t pos = a.r.pos[i], last = pos + len - 1;
  const bool ok = has_place(a.c, q, pos);
  const uint32_t all = len * G, c0 = part_i * PW;   // (rows x query heads < 2^31)
  const View view(last, a.c.slots);
  const uint32_t t_lo = c0 / G, t_hi = (min(all, c0 + PW) - 1) / G;
  // before the ring wraps, slots past the last row's position hold nothing
  // that any of the pairs sees
  const bool flat = last < a.c.slots;
  const uint32_t seen = flat ? pos + t_hi + 1 : view.live;
  const uint32_t tiles = ok ? (seen + 31) / 32 : 0u;
  const uint32_t per = piece_tiles(tiles, a.nsplit, kManyTiles);
  const uint32_t t0 = z * per, t1 = min(tiles, t0 + per);
  if (z && t0 >= t1) return;
  const bool split = tiles > per;

  const uint8_t* base = record_of(a.c, ok ? q : 0, head, 0);
  // a wave's part of a record: the key codes of slots m and 16 + m, or the
  // value codes, and eight bytes with their scales; the same loads for both,
  // so that they stay in flight through a tile
  uint32_t rw[OPS], rs[2];
  const uint32_t half = wv & 1;
  const bool keys = wv < 2;
  const uint32_t krow = j * D / 128 * 16 + m;   // this lane's key scales, two bytes each
  const uint32_t w_at = (keys ? 0 : 16 * D) + lane * (D / 4);
  const uint32_t s_at = keys ? 32 * D + (krow * 2 & ~7u) : 33 * D + (m * D / 512 * 4 + j) * 8;
  auto load = [&](uint32_t tile) {
    const uint8_t* rec = base + (uint64_t)tile * (34 * D);
    load_words<D>(rw, rec + w_at);
    const uint2 t = *reinterpret_cast<const uint2*>(rec + s_at);
    rs[0] = t.x;
    rs[1] = t.y;
  };
  auto stage = [&](uint32_t tile, uint32_t buf) {
    bool bad;
    if (keys) {
      const uint32_t s0 = rs[0], s1 = rs[1], b8 = ((krow & 2 ? s1 : s0) >> ((krow & 1) * 16 + half * 8)) & 0xFF;
      const float ksc = __builtin_bit_cast(float, b8 << 23);
      bad = __any(b8 == 255);
#pragma unroll
      for (int d = 0; d < KS; d++) {
        const uint32_t w0 = rw[d], w1 = rw[KS + d], w = half ? w1 : w0;
        const u32x4_t o = {two_of<0>(w, ksc), two_of<1>(w, ksc), two_of<2>(w, ksc), two_of<3>(w, ksc)};
        ops[buf][0][half * KS + d][lane] = __builtin_bit_cast(bf16x8_t, o);
      }
    } else {
      bad = __any(has255(rs[0]) | has255(rs[1]));
      if (bad || tile * 32 + 32 > view.live) quiet_values(rs, tile, view.live, j);
      float vsc[8];
#pragma unroll
      for (int e = 0; e < 8; e++) vsc[e] = scale_of(rs[e / 4], e % 4);
      static_for<KS>([&](auto u_) {
        constexpr int u = decltype(u_)::value;
        if (half == u * 2 / KS)
          val_ops<D, u>(rw, vsc, ops[buf][1][2 * u][lane], ops[buf][1][2 * u + 1][lane]);
      });
    }
    if (lane == 0) flag[buf][wv] = bad;
  };
  if (t0 < t1) load(t0);   // (in flight while the queries are read)

  const float sc = a.scale * kLog2e;
  bf16x8_t qo[NQ][NP][KS];
  uint32_t ago[NQ];
#pragma unroll
  for (int n = 0; n < NQ; n++) {
    const uint32_t c = c0 + (wv * NQ + n) * 16 + m;
    const bool on = c < all;
    const uint32_t t = on ? c / G : t_lo, g = on ? c % G : 0;
    ago[n] = len - 1 - t;
    query_ops<T, D, NP>(a.q, row0 + t, head * G + g, j, on, vec, query_factor<T>(sc), qo[n]);
  }
  // the last slot that a pair of this wave sees, where the ring has not wrapped
  const uint32_t w0 = c0 + wv * NQ * 16;
  const uint32_t wave_hi = w0 < all ? pos + (min(all, w0 + NQ * 16) - 1) / G : 0;
  const float sf = score_factor<T>(sc);
  f32x4_t o[NQ][OPS], less[NQ];
  float mx[NQ], l[NQ];
  uint32_t nan[NQ];
#pragma unroll
  for (int n = 0; n < NQ; n++) {
    less[n] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int d = 0; d < OPS; d++) o[n][d] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
    mx[n] = -INFINITY;
    l[n] = 0.0f;
    nan[n] = 0;
  }
  uint32_t buf = 0;
  if (t0 < t1) stage(t0, 0);
  __syncthreads();
#pragma unroll 1
  for (uint32_t tile = t0; tile < t1; tile++) {
    const bool more = tile + 1 < t1;
    if (more) load(tile + 1);
    // (past every position of the wave's pairs: nothing to do)
    if (!flat || tile * 32 <= wave_hi) {
      const bool whole = view.whole(tile, len - 1 - t_lo);
      const bool bad_k = flag[buf][0] | flag[buf][1], bad = flag[buf][2] | flag[buf][3];
      // (f32 scores come out less their pair's maximum: the products start from it)
      f32x4_t s[NQ][2];
#pragma unroll
      for (int n = 0; n < NQ; n++) s[n][0] = s[n][1] = less[n];
#pragma unroll
      for (int d = 0; d < KS; d++)
#pragma unroll
        for (int h = 0; h < 2; h++) {
          const bf16x8_t ko = ops[buf][0][h * KS + d][lane];
#pragma unroll
          for (int u = 0; u < NP; u++)
#pragma unroll
            for (int n = 0; n < NQ; n++)
              s[n][h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ko, qo[n][u][d], s[n][h], 0, 0, 0);
        }
      bf16x8_t po[NQ][NPP];
      float x[NQ][8];
      bool raise = false;
      float top[NQ];
#pragma unroll
      for (int n = 0; n < NQ; n++)
#pragma unroll
        for (int e = 0; e < 8; e++) x[n][e] = s[n][e / 4][e % 4];
      if (bad_k) {
        // (such a key has made its own slot's scores anything)
        const uint32_t nk = nan_keys<D>(base + (uint64_t)tile * (34 * D), j);
#pragma unroll
        for (int e = 0; e < 8; e++)
#pragma unroll
          for (int n = 0; n < NQ; n++) x[n][e] = (nk >> e) & 1 ? __builtin_nanf("") : x[n][e];
      }
      if (!whole) {
#pragma unroll
        for (int e = 0; e < 8; e++) {
          const uint32_t slot = tile * 32 + 16 * (e / 4) + 4 * j + e % 4, back = view.back(slot);
          const bool live = slot < view.live;
#pragma unroll
          for (int n = 0; n < NQ; n++) x[n][e] = live && back >= ago[n] ? x[n][e] : -INFINITY;
        }
      }
      if (bad) {
#pragma unroll 1
        for (int n = 0; n < NQ; n++) {
          const uint32_t t = nan_blocks<D>(base + (uint64_t)tile * (34 * D), tile, view, n ? ago[NQ - 1] : ago[0], j);
          if (n == 0) nan[0] |= t;
          else nan[NQ - 1] |= t;
        }
      }
#pragma unroll
      for (int n = 0; n < NQ; n++) {
        top[n] = x[n][0];
#pragma unroll
        for (int e = 1; e < 8; e++) top[n] = fmaxf(top[n], x[n][e]);
        if constexpr (F32) raise |= top[n] > (mx[n] == -INFINITY ? mx[n] : kSlack);
        else raise |= top[n] * sf > mx[n] + kSlack;
      }
      if (__any(raise)) {
#pragma unroll
        for (int n = 0; n < NQ; n++) {
          const float was = mx[n] == -INFINITY ? 0.0f : mx[n];
          const float v = fmaxf(mx[n], F32 ? pair_max(top[n]) + was : pair_max(top[n]) * sf);
          const float f = v == mx[n] ? 1.0f : __builtin_amdgcn_exp2f(mx[n] - v);
          mx[n] = v;
          if constexpr (F32) {
            const float b = v == -INFINITY ? 0.0f : v;
#pragma unroll
            for (int e = 0; e < 8; e++) x[n][e] -= b - was;
            less[n] = f32x4_t{-b, -b, -b, -b};
          }
          l[n] *= f;
#pragma unroll
          for (int d = 0; d < OPS; d++) o[n][d] *= f;
        }
      }
#pragma unroll
      for (int n = 0; n < NQ; n++) {
        const float b = mx[n] == -INFINITY ? 0.0f : mx[n];
#pragma unroll
        for (int e = 0; e < 8; e++) x[n][e] = __builtin_amdgcn_exp2f(F32 ? x[n][e] : fmaf(x[n][e], sf, -b));
        split8_p(x[n], po[n]);
        if constexpr (NPP == 1) {
          const bf16x2_t one = {(__bf16)1.0f, (__bf16)1.0f};
#pragma unroll
          for (int e = 0; e < 8; e += 2)
            l[n] = __builtin_amdgcn_fdot2_f32_bf16(bf16x2_t{po[n][0][e], po[n][0][e + 1]}, one, l[n], false);
        } else {
#pragma unroll
          for (int e = 0; e < 8; e++) l[n] += x[n][e];
        }
      }
#pragma unroll
      for (int t = 0; t < OPS; t++) {
        const bf16x8_t vo = ops[buf][1][t][lane];
#pragma unroll
        for (int u = 0; u < NPP; u++)
#pragma unroll
          for (int n = 0; n < NQ; n++)
            o[n][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vo, po[n][u], o[n][t], 0, 0, 0);
      }
    }
    if (more) stage(tile + 1, buf ^ 1);
    __syncthreads();
    buf ^= 1;
  }
  // the outputs, 16 pairs at a time through the wave's part of LDS, so that a
  // store's lanes write whole rows
  float(*rows)[OR] = reinterpret_cast<float(*)[OR]>(lds + wv * (16 * OR * 4));
#pragma unroll
  for (int n = 0; n < NQ; n++) {
    const float ls = pair_sum(l[n]);
    const uint32_t nn = pair_or(nan[n]);
    float f = 1.0f, inv = 1.0f;
    const uint32_t c = c0 + (wv * NQ + n) * 16 + m;
    const bool on = c < all;
    const uint32_t row = on ? row0 + c / G : row0, hq = on ? head * G + c % G : 0;
    float* part = a.part + (((uint64_t)row * a.hq + hq) * a.nsplit + z) * (D + kPartHead);
    if (!split) {
      const float den = finish_sum(mx[n], ls, a.sink, hq, &f);
      inv = ok && den != 0.0f ? f / den : 0.0f;
    }
    if (a.nsplit > 1 && on && j == 0) {
      if (z == 0) part[2] = __builtin_bit_cast(float, split ? (tiles + per - 1) / per : kDone);
      part[0] = mx[n];
      part[1] = ls;
    }
#pragma unroll
    for (int i4 = 0; i4 < 4; i4++)
#pragma unroll
      for (int t = 0; t < OPS; t += 2) {
        const uint32_t d = j * (D / 4) + i4 * OPS + t;
        const bool bad = (nn >> (d / 32)) & 1;
        *reinterpret_cast<float2*>(&rows[m][d]) =
            make_float2(bad ? __builtin_nanf("") : o[n][t][i4] * inv, bad ? __builtin_nanf("") : o[n][t + 1][i4] * inv);
      }
    __builtin_amdgcn_wave_barrier();
    // where each pair's row goes, in elements (of the partials, or the outputs)
    const uint64_t to = split ? (uint64_t)(part - a.part) + kPartHead : (uint64_t)row * a.o.row + (uint64_t)hq * a.o.head;
    constexpr uint32_t LR = D / 8;   // lanes a row, eight outputs each
#pragma unroll
    for (uint32_t r = 0; r < 16; r += 64 / LR) {
      const uint32_t pp = r + lane / LR, d = lane % LR * 8;
      const uint64_t at = (uint64_t)(uint32_t)__shfl((uint32_t)(to >> 32), pp, 64) << 32 | (uint32_t)__shfl((uint32_t)to, pp, 64);
      const bool mine = __shfl((int)on, pp, 64);
      const f32x4_t y0 = *reinterpret_cast<const f32x4_t*>(&rows[pp][d]), y1 = *reinterpret_cast<const f32x4_t*>(&rows[pp][d + 4]);
      const float y[8] = {y0[0], y0[1], y0[2], y0[3], y1[0], y1[1], y1[2], y1[3]};
      if (mine) {
        if (split) store8(a.part + at + d, true, y);
        else store8((T*)a.o.p + at + d, vec, y);
      }
    }
    __builtin_amdgcn_wave_barrier();
  }
}

// The pieces of a (row, query head), a wave each: weights 2^(m_z - M), then
// the sink, then the division. D / 4 lanes take a piece's outputs, so several
// pieces are in flight at once.
template <typename T, int D>
__global__ __launch_bounds__(256) void k_kv4_join(Kv4Attend a) {
  constexpr uint32_t L = D / 4, GR = 64 / L;   // lanes a piece, pieces at once
  const uint32_t lane = threadIdx.x & 63;
  const uint64_t w = (uint64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const uint32_t row = (uint32_t)(w / a.hq), hd = (uint32_t)(w % a.hq);
  if (row >= a.r.rows) return;
  const float* part = a.part + ((uint64_t)row * a.hq + hd) * a.nsplit * (D + kPartHead);
  const uint32_t nz = __builtin_bit_cast(uint32_t, part[2]);
  // (a row that no sequence has: its words are whatever they are)
  if (a.r.off && (row < a.r.off[0] || row >= a.r.off[a.r.n])) return;
  if (nz > a.nsplit) return;
  float M = -INFINITY;
  for (uint32_t z = lane; z < nz; z += 64) M = fmaxf(M, part[z * (D + kPartHead)]);
  M = wmax(M);
  const uint32_t g = lane / L, d = lane % L * 4;
  float l = 0.0f;
  f32x4_t o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
  for (uint32_t z = g; z < nz; z += GR) {
    const float* p = part + z * (D + kPartHead);
    const f32x4_t y = *reinterpret_cast<const f32x4_t*>(p + kPartHead + d);
    const float m = p[0];
    const float f = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - M);
    l += p[1] * f;
    o += y * f;
  }
#pragma unroll
  for (uint32_t mk = L; mk < 64; mk <<= 1) {
    l += __shfl_xor(l, mk, 64);
#pragma unroll
    for (int e = 0; e < 4; e++) o[e] += __shfl_xor(o[e], mk, 64);
  }
  float f;
  const float den = finish_sum(M, l, a.sink, hd, &f);
  const float inv = nz && den != 0.0f ? f / den : 0.0f;
  T* out = (T*)a.o.p + (uint64_t)row * a.o.row + (uint64_t)hd * a.o.head + d;
  if (g == 0) {
#pragma unroll
    for (int e = 0; e < 4; e++) out[e] = (T)(nz ? o[e] * inv : 0.0f);
  }
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
  if (!c.data || !r.pos || c.slots == 0 || r.rows > kKv4MaxRows || (q && type != ET_F32)) return hipErrorInvalidValue;
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
  if (!c.data || !r.pos || c.slots == 0 || r.rows > kKv4MaxRows) return hipErrorInvalidValue;
  if (r.rows == 0 || r.n == 0) return hipSuccess;
  return by_type(type, c.hd, [&](auto t, auto d) -> hipError_t {
    using T = decltype(t);
    constexpr int D = decltype(d)::value;
    hipLaunchKernelGGL((k_kv4_read<T, D>), dim3((r.rows + 31) / 32, c.heads, 2), dim3(32 * D * sizeof(T) / 16), 0, st, c, r, k, v,
                       (uint32_t)(on16<T>(k) && on16<T>(v)));
    return hipGetLastError();
  });
}

uint64_t kv4_attend_groups(uint32_t heads, uint32_t n, uint32_t rows, bool ragged, uint32_t hq) {
  const uint64_t G = hq / heads;
  if (!ragged) return (uint64_t)n * heads * ((G + 15) / 16);
  return ((rows * G + 63) / 64 + n) * heads;   // (workgroups of 64 pairs or more)
}

// Pieces of the slots at most: as many as keep to three workgroups a CU, each
// sequence's tiles cut evenly by the kernels, which know its length (64 single
// rows of 12 heads, ragged to 2048 slots: 15 us whole, 24 in two pieces with
// the join; two pieces of 1024 rows over 30000 positions, 252 workgroups
// whole: 1050 us, in two 642, in three 537). A ragged call has a workgroup for
// each sequence and key head at least (64 sequences of four rows, 12 heads,
// 1900 positions: 58 us in eight pieces, 31 whole), and one for every 128
// pairs: f32 and f16 ones hold 64, but are as fast six a CU (1024 f32 rows
// of 12 heads over 30000 positions: 296 us so, 375 where 64 are counted).
uint32_t kv4_split(const Kv4& c, uint32_t n, uint32_t rows, bool ragged, uint32_t hq, uint64_t live) {
  const uint64_t slots = live ? std::min<uint64_t>(live, c.slots) : c.slots;
  const uint32_t tiles = (uint32_t)((slots + 31) / 32);
  const uint64_t G = hq / c.heads;
  const uint64_t parts = ragged ? std::max<uint64_t>(std::min(n, rows), (rows * G + 127) / 128) : n * ((G + 15) / 16);
  return (uint32_t)std::max<uint64_t>(
      1, std::min<uint64_t>({768 / std::max<uint64_t>(parts * c.heads, 1), 128, tiles / (ragged ? kManyTiles : kFewTiles)}));
}

hipError_t launch_kv4_attend(const Kv4Attend& a, int type, hipStream_t st) {
  if (!a.c.data || !a.r.pos || a.c.slots == 0 || a.c.heads == 0 || a.hq == 0 || a.hq % a.c.heads || a.nsplit == 0 || a.nsplit > 65535 || (a.nsplit > 1 && !a.part))
    return hipErrorInvalidValue;
  if (kv4_attend_groups(a.c.heads, a.r.n, a.r.rows, a.r.off != nullptr, a.hq) > kKv4MaxGroups) return hipErrorInvalidValue;
  if (a.r.rows == 0 || a.r.n == 0) return hipSuccess;
  return by_type(type, a.c.hd, [&](auto t, auto d) -> hipError_t {
    using T = decltype(t);
    constexpr int D = decltype(d)::value;
    const uint32_t vec = on16<T>(a.q) && on16<T>(a.o);
    const uint32_t G = a.hq / a.c.heads;
    // a pair's columns: one a part, where single rows leave the room
    constexpr int NC = sizeof(T) == 4 ? 4 : 2;
    const bool wide = !a.r.off && G * NC <= 16;
    const uint32_t ncol = a.r.off ? 1 : (G + 15) / 16;
    const dim3 grid(a.r.n * a.c.heads * ncol, a.nsplit);
    if (wide) hipLaunchKernelGGL((k_kv4_few<T, D, NC>), grid, dim3(256), 0, st, a, vec, 1u);
    else hipLaunchKernelGGL((k_kv4_few<T, D, 1>), grid, dim3(256), 0, st, a, vec, ncol);
    if (a.r.off) {
      constexpr uint32_t PW = Many<T, D>::pairs;
      const uint32_t gx = (uint32_t)(((uint64_t)a.r.rows * G + PW - 1) / PW) + a.r.n;
      hipLaunchKernelGGL((k_kv4_many<T, D>), dim3(gx * a.c.heads, a.nsplit), dim3(256), 0, st, a, vec);
    }
    if (a.nsplit > 1)
      hipLaunchKernelGGL((k_kv4_join<T, D>), dim3((uint32_t)(((uint64_t)a.r.rows * a.hq + 3) / 4)), dim3(256), 0, st, a);
    return hipGetLastError();
  });
}

}  // namespace ana
