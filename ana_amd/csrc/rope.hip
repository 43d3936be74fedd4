// Queries and keys of each head, RMS-normed and turned by their positions, in
// one pass (gfx950).
//
//   y = x n (1 + g),  n = 1 / sqrt(mean x^2 + eps)      (where there are gains)
//   a' = a cos t - b sin t,  b' = b cos t + a sin t,  t = p f_i
// for the pairs (a, b) of the head's first `rot` values.
//
// Bound by memory: every value is read and written once. A workgroup takes a
// few rows: their angles once into LDS, while its first loads are in flight,
// then the heads, a lane two pieces of 16 bytes that are each other's
// partners, so no value moves between lanes. (16384 rows of 32 + 8 heads of 128
// in bf16: 72 us, 4.7 TB/s, what a large copy reaches; 8384 of 12 + 12 heads of
// 64 in f32, normed: 26 us, 3.9 TB/s, one round of workgroups.)
#include <hip/hip_runtime.h>

#include <algorithm>

#include "mfma.h"
#include "rope.h"
#include "rows.h"

namespace ana {

namespace {

constexpr uint32_t kRopeRows = 16;   // rows a workgroup, at most

// cos and sin of p f. The angle in quarter turns is the exact product of 56
// bits times 2 / pi in twice 53, so that the part after the whole turns is
// right to f32's last bits at every position below 2^32, for frequencies
// up to 256 in size and some way past (in f32 the angle of
// position 10^6 is off by 0.03); then the series of sin and cos on a quarter
// turn about 0, cut where the next term is below 2^-28.
__device__ __forceinline__ float2 cos_sin(uint32_t p, float f) {
  constexpr double c0 = 0x1.45f306dc9c883p-1, c1 = -0x1.6b01ec5417056p-55;   // 2 / pi
  const double pd = p, fd = f;
  const double hi = pd * fd, lo = fma(pd, fd, -hi);
  const double t = hi * c0, tl = fma(hi, c0, -t) + (hi * c1 + lo * c0);
  const double n = __builtin_rint(t);
  const float a = (float)((t - n) + tl) * 1.57079632679489662f;
  const float z = a * a;
  float s = fmaf(z, 2.7557319e-6f, -1.9841270e-4f);
  s = fmaf(z, s, 8.3333333e-3f);
  s = fmaf(z, s, -1.6666667e-1f);
  s = fmaf(a * z, s, a);
  float c = fmaf(z, -2.7557319e-7f, 2.4801587e-5f);
  c = fmaf(z, c, -1.3888889e-3f);
  c = fmaf(z, c, 4.1666667e-2f);
  c = fmaf(z, c, -0.5f);
  c = fmaf(z, c, 1.0f);
  const double quarter = n - 4.0 * __builtin_floor(n * 0.25);   // 0 .. 3 (NaN for an angle that is not finite)
  const int k = (int)quarter;
  const float x = k & 1 ? s : c, y = k & 1 ? c : s;
  return make_float2(k == 1 || k == 2 ? -x : x, k >= 2 ? -y : y);
}

template <typename T, int E>
__device__ __forceinline__ void load_piece(const T* p, bool vec, float (&x)[E]) {
  typedef T vec_t __attribute__((ext_vector_type(E)));
  if (vec) {
    const vec_t v = *reinterpret_cast<const vec_t*>(p);
#pragma unroll
    for (int e = 0; e < E; e++) x[e] = (float)v[e];
  } else {
#pragma unroll
    for (int e = 0; e < E; e++) x[e] = (float)p[e];
  }
}
template <typename T, int E>
__device__ __forceinline__ void store_piece(T* p, bool vec, const float (&x)[E]) {
  typedef T vec_t __attribute__((ext_vector_type(E)));
  if (vec) {
    vec_t v;
#pragma unroll
    for (int e = 0; e < E; e++) v[e] = (T)x[e];
    *reinterpret_cast<vec_t*>(p) = v;
  } else {
#pragma unroll
    for (int e = 0; e < E; e++) p[e] = (T)x[e];
  }
}

// A workgroup's items are its rows' heads (queries, then keys), L lanes each,
// of which hd / (2 E) work; a thread takes U of them at a time.
template <typename T, int L, int U>
__global__ __launch_bounds__(256) void k_qk_rope(RopeArgs a, uint32_t R, uint32_t heads_y, uint32_t vec) {
  constexpr int E = 16 / sizeof(T);
  __shared__ float2 cs[kRopeRows * kRopeMaxHd / 2];
  __shared__ uint32_t pos_s[kRopeRows];
  __shared__ uint32_t state_s[kRopeRows];   // 0: no sequence's row, 1: with a position, 2: of a sequence that has none
  const uint32_t tid = threadIdx.x, sub = tid % L;
  const uint32_t row0 = blockIdx.x * R, rows = min(R, a.r.rows - row0);
  const uint32_t h0 = blockIdx.y * heads_y, H = min(heads_y, a.hq + a.hk - h0);
  const uint32_t half = a.rot / 2, items = rows * H;
  const bool works = sub < a.hd / (2 * E);
  // the lane's pieces of a head: dims d0 .. and d1 ..
  const uint32_t turned = a.rot / (2 * E);
  uint32_t d0 = sub * 2 * E, d1 = d0 + E;
  if (!a.near && sub < turned) {
    d0 = sub * E;
    d1 = d0 + half;
  }
  const bool turns = sub < turned;

  float x0[U][E], x1[U][E];
  // (rows that no sequence has are read too: they are the tensors' own)
  auto load = [&](uint32_t it, float (&y0)[E], float (&y1)[E]) {
    const uint32_t row = row0 + it / H, h = h0 + it % H;
    const bool is_q = h < a.hq;
    const Kv4Mat& m = is_q ? a.q : a.k;
    const T* p = (const T*)m.p + (uint64_t)row * m.row + (uint64_t)(is_q ? h : h - a.hq) * m.head;
    load_piece(p + d0, vec, y0);
    load_piece(p + d1, vec, y1);
  };
  uint32_t it = tid / L;
#pragma unroll
  for (int u = 0; u < U; u++)
    if (works && it + u * (256 / L) < items) load(it + u * (256 / L), x0[u], x1[u]);

  if (tid < 64) {
    const uint32_t i0 = a.r.off ? find_seq(a.r.off, a.r.n, row0) : 0;
    if (tid < rows) {
      const uint32_t row = row0 + tid;
      uint32_t i = row, o0 = row, o1 = row + 1;
      if (a.r.off) {
        i = find_from(a.r.off, a.r.n, row, i0);
        o0 = a.r.off[i];
        o1 = a.r.off[i + 1];
      }
      const bool on = row >= o0 && row < o1;
      const uint32_t p = on ? a.r.pos[i] : 0;
      pos_s[tid] = p + (row - o0);
      state_s[tid] = !on ? 0 : p < 0x80000000u ? 1 : 2;
    }
  }
  __syncthreads();
  for (uint32_t i = tid; i < rows * half; i += 256) cs[i] = cos_sin(pos_s[i / half], a.freq[i % half]);
  __syncthreads();

  for (;;) {
#pragma unroll
    for (int u = 0; u < U; u++) {
      const uint32_t at = it + u * (256 / L);
      const bool in = at < items;
      const uint32_t r = in ? at / H : 0, h = h0 + (in ? at % H : 0);
      const bool is_q = h < a.hq;
      const float* g = is_q ? a.gq : a.gk;
      float (&y0)[E] = x0[u], (&y1)[E] = x1[u];
      if (g) {
        float s = 0.0f;
        if (works && in) {
#pragma unroll
          for (int e = 0; e < E; e++) s = fmaf(y0[e], y0[e], s);
#pragma unroll
          for (int e = 0; e < E; e++) s = fmaf(y1[e], y1[e], s);
        }
#pragma unroll
        for (int m = 1; m < L; m <<= 1) s += __shfl_xor(s, m, 64);
        const float n = 1.0f / sqrtf(s / (float)a.hd + a.eps);
        if (works) {
#pragma unroll
          for (int e = 0; e < E; e++) {
            y0[e] = (y0[e] * n) * (1.0f + g[d0 + e]);
            y1[e] = (y1[e] * n) * (1.0f + g[d1 + e]);
          }
        }
      }
      const uint32_t st = state_s[r];
      if (!in || !works || st == 0) continue;
      if (turns) {
        const float2* w = cs + r * half + sub * E;
        if (a.near) {
#pragma unroll
          for (int e = 0; e < E; e += 2) {
            const float2 u0 = w[e / 2], u1 = w[E / 2 + e / 2];
            const float p0 = y0[e], q0 = y0[e + 1], p1 = y1[e], q1 = y1[e + 1];
            y0[e] = fmaf(p0, u0.x, -(q0 * u0.y));
            y0[e + 1] = fmaf(q0, u0.x, p0 * u0.y);
            y1[e] = fmaf(p1, u1.x, -(q1 * u1.y));
            y1[e + 1] = fmaf(q1, u1.x, p1 * u1.y);
          }
        } else {
#pragma unroll
          for (int e = 0; e < E; e++) {
            const float2 c = w[e];
            const float p0 = y0[e], q0 = y1[e];
            y0[e] = fmaf(p0, c.x, -(q0 * c.y));
            y1[e] = fmaf(q0, c.x, p0 * c.y);
          }
        }
      }
      if (st == 2) {
#pragma unroll
        for (int e = 0; e < E; e++) y0[e] = y1[e] = 0.0f;
      }
      const Kv4Mat& m = is_q ? a.qo : a.ko;
      T* p = (T*)m.p + (uint64_t)(row0 + r) * m.row + (uint64_t)(is_q ? h : h - a.hq) * m.head;
      store_piece(p + d0, vec, y0);
      store_piece(p + d1, vec, y1);
    }
    it += U * (256 / L);
    if (it - tid / L >= items) break;
#pragma unroll
    for (int u = 0; u < U; u++)
      if (works && it + u * (256 / L) < items) load(it + u * (256 / L), x0[u], x1[u]);
  }
}

template <typename T>
bool on16(const Kv4Mat& x) {
  return ((uintptr_t)x.p | (x.row * sizeof(T)) | (x.head * sizeof(T))) % 16 == 0;
}

}  // namespace

hipError_t launch_rope(const RopeArgs& a, int type, hipStream_t st) {
  if (!rope_fits(a.hd) || a.rot > a.hd || a.rot % 16 || (a.rot && !a.freq) || !a.r.pos || a.r.rows > kKv4MaxRows ||
      a.hq > 65535 || a.hk > 65535)
    return hipErrorInvalidValue;
  if (a.r.rows == 0 || a.r.n == 0 || a.hq + a.hk == 0) return hipSuccess;
  auto go = [&](auto t, auto l) -> hipError_t {
    using T = decltype(t);
    constexpr int L = decltype(l)::value, U = sizeof(T) == 4 ? 4 : 2;
    const uint32_t H = a.hq + a.hk, step = U * 256 / L;   // heads a workgroup takes at a time
    const uint32_t vec = on16<T>(a.q) && on16<T>(a.qo) && (!a.hk || (on16<T>(a.k) && on16<T>(a.ko)));
    // Rows a workgroup: as many as give each thread two turns, while there are two
    // workgroups a CU; single rows are cut into the heads of one turn. (And as many as
    // keep the grid's threads below 2^32.)
    uint32_t R = std::min(kRopeRows, std::max(1u, 2 * step / H)), hy = H;
    R = std::max(std::min(R, std::max(1u, a.r.rows / 512)), (a.r.rows + (1u << 23) - 1) >> 23);
    if (R == 1) hy = std::min(H, step);
    const dim3 grid((a.r.rows + R - 1) / R, (H + hy - 1) / hy);
    hipLaunchKernelGGL((k_qk_rope<T, L, U>), grid, dim3(256), 0, st, a, R, hy, vec);
    return hipGetLastError();
  };
  auto by_hd = [&](auto t) -> hipError_t {
    const uint32_t n = a.hd * sizeof(t) / 32;   // lanes that a head takes
    if (n <= 4) return go(t, std::integral_constant<int, 4>{});
    if (n <= 8) return go(t, std::integral_constant<int, 8>{});
    if constexpr (sizeof(t) == 4)
      if (n > 16) return go(t, std::integral_constant<int, 32>{});
    return go(t, std::integral_constant<int, 16>{});
  };
  switch (type) {
    case ET_F32: return by_hd(float{});
    case ET_BF16: return by_hd(__bf16{});
    case ET_F16: return by_hd(_Float16{});
    default: return hipErrorInvalidValue;
  }
}

}  // namespace ana
