// Keys and values held in 4 bits (MXFP4: E2M1 codes, an E8M0 scale a block of
// 32 values along a head): the cache's records and what the kernels take.
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>

namespace ana {

// A cache: per sequence and head, ceil(slots / 32) records of 34 hd bytes,
// 32 slots each. A record is laid out as the attention's lanes read it (lane
// 16 j + m of a wave), so that a wave loads one as whole consecutive pieces:
//   keys    [4 j][16 m][2 h][hd / 8 bytes]   slot 16 h + m, dims j hd / 4 ..
//   values  [4 j][16 m][8 e][hd / 32 bytes]  slot 16 (e / 4) + 4 j + e % 4, dims m hd / 16 ..
//   key scales    [hd / 32 blocks][16 m][2 h]
//   value scales  [hd / 32 blocks][4 j][8 e]
// A slot's codes and scales are whole bytes of its own, so two tokens that
// are written at once never share a byte.
struct Kv4 {
  uint8_t* data;
  uint64_t seq_bytes;   // from a sequence's records to the next one's (a multiple of 16)
  uint32_t seqs, slots, tiles, heads, hd;
};
__host__ __device__ inline uint32_t kv4_record(uint32_t hd) { return 34 * hd; }
inline uint64_t kv4_seq_bytes(uint32_t slots, uint32_t heads, uint32_t hd) {
  return (uint64_t)heads * (((uint64_t)slots + 31) / 32) * kv4_record(hd);
}

// The rows of a call: sequence i (cache place seq[i], or i) has rows off[i]
// .. off[i + 1] - 1 (or row i alone) at positions from pos[i].
struct Kv4Rows {
  const uint32_t *seq, *pos, *off;
  uint32_t n, rows;
};
// a tensor [rows][heads][hd]: strides in elements, hd consecutive
struct Kv4Mat {
  void* p;
  uint64_t row, head;
};

enum ElemType : int { ET_F32 = 0, ET_BF16 = 1, ET_F16 = 2 };

// A launch's threads along an axis are counted in 32 bits: the most rows (and
// sequences) of a call, and workgroups of the attention.
constexpr uint32_t kKv4MaxRows = 1u << 26, kKv4MaxGroups = (1u << 24) - 1;

// the head sizes and element types that the kernels take
inline bool kv4_fits(uint32_t hd) { return hd == 32 || hd == 64 || hd == 128; }

// k and v into the cache. With gk, k is qk-normed first, and with q (f32) the
// query rows of sequences with a place are normed in place with gq (one launch
// for a decoder layer).
hipError_t launch_kv4_write(const Kv4& c, const Kv4Rows& r, int type, const Kv4Mat& k, const Kv4Mat& v,
                            const float* gk, const float* gq, const Kv4Mat* q, uint32_t qheads, hipStream_t st);
// the values that the cache holds for the rows
hipError_t launch_kv4_read(const Kv4& c, const Kv4Rows& r, int type, const Kv4Mat& k, const Kv4Mat& v,
                           hipStream_t st);

constexpr uint32_t kKv4PartHead = 4;   // a partial result's words before its outputs

struct Kv4Attend {
  Kv4 c;
  Kv4Rows r;
  Kv4Mat q, o;
  uint32_t hq;
  float scale;
  const float* sink;   // [hq] or nullptr
  float* part;         // partials [rows][hq][nsplit][kKv4PartHead + hd], when nsplit > 1
  uint32_t nsplit;     // pieces that a sequence's slots are cut into at most
  // (set by the launches) a pair's places in `part` and the first of this
  // kernel's pieces; the groups of rows that share prefixes, whose pieces come
  // after the nsplit of a row's own
  uint32_t nz, z0;
  Kv4Rows pre;
};
// the pieces of a call (live: the most positions a sequence holds after it,
// as far as the caller knows; 0: the ring's slots), and the floats of
// partials they take
// (groups: the workgroups of its largest launch a piece, at most)
uint64_t kv4_attend_groups(uint32_t heads, uint32_t n, uint32_t rows, bool ragged, uint32_t hq);
uint32_t kv4_split(const Kv4& c, uint32_t n, uint32_t rows, bool ragged, uint32_t hq, uint64_t live);
inline uint64_t kv4_part_floats(uint32_t rows, uint32_t hq, uint32_t hd, uint32_t nsplit) {
  return nsplit > 1 ? (uint64_t)rows * hq * nsplit * (kKv4PartHead + hd) : 0;
}
hipError_t launch_kv4_attend(const Kv4Attend& a, int type, hipStream_t st);

// Attention where groups of rows also see a prefix that they share: group i of
// pre has rows off[i] .. off[i + 1] - 1 (off NULL: one group, of all rows), and
// they see the first pos[i] positions of its place in pc, as far as that ring
// holds them. part: kv4_part_floats of nsplit + psplit pieces.
uint64_t kv4_prefix_groups(uint32_t heads, uint32_t n, uint32_t rows, uint32_t hq);
uint32_t kv4_prefix_split(const Kv4& pc, uint32_t n, uint32_t rows, uint32_t hq, uint64_t live);
hipError_t launch_kv4_attend_shared(const Kv4Attend& a, const Kv4& pc, const Kv4Rows& pre, uint32_t psplit, int type,
                                    hipStream_t st);

}  // namespace ana
