// What the attention kernels share: the arguments, and the view of one block of one sequence.
#pragma once

#include "common.cuh"

namespace atlas {

constexpr int kAttnBlock = 128;  // rows of an entry of the block table
constexpr int kAttnMaxDim = 64;

struct Strides {
  int64_t outer, head, row;  // in elements; the last axis has unit stride
};

// q [outer, H, rows, D], k and v [outer, Hk, rows, D]; H / Hk query heads share a key head.
struct AttnArgs {
  const void *q, *k, *v, *o, *dout;  // o, dout: gradient only
  void *out, *dq, *dk, *dv;
  Strides sq, sk, sv, so, sdo, sdq, sdk, sdv;
  float* lse;    // [outer, H, rows]
  // Gradient only. CUDA cores: delta [outer, H, rows]. Tensor cores: for each head, negated, the
  // log-sum-exp in base 2 and delta of all sequences, each from a place that is a multiple of 16 bytes (seq_block's off;
  // vec_ld values a head), the largest |dout| of a sequence and key head as bits (fp16), and the counter of
  // work items.
  float *delta, *lse2, *delta2;
  int64_t vec_ld;
  uint32_t *amax, *counter;
  const int32_t *cu, *blocks;
  const int64_t* counts;
  int64_t outer, rows, B, cap;
  int H, Hk, D, packed;
  float scale;
};

// One entry of the block table: rows first .. first + 127 of sequence `seq`, whose rows are
// row0 .. row0 + len - 1 of outer index `outer`. Everything is cut to the tensors' extents, so that a
// table or prefix sums that do not belong to these tensors cannot lead outside them.
struct SeqBlock {
  int seq, first, len;
  int64_t row0, outer, off;
  bool on;     // an entry with a sequence
  bool spare;  // an entry behind the last
};

__device__ __forceinline__ SeqBlock seq_block(const AttnArgs& a, int64_t i) {
  SeqBlock s{};
  const int64_t n = a.counts[1];
  const int2 e = reinterpret_cast<const int2*>(a.blocks)[i];  // i < cap: both loads are under way at once
  s.spare = i >= n;
  if (s.spare) return s;
  if (e.x < 0 || e.x >= a.B || e.y < 0) return s;
  const int64_t c0 = a.cu[e.x], c1 = a.cu[e.x + 1];
  s.seq = e.x;
  s.first = e.y;
  s.row0 = a.packed ? c0 : 0;
  s.outer = a.packed ? 0 : e.x;
  if (s.row0 < 0 || s.row0 > a.rows || s.outer >= a.outer) return s;
  const int64_t len = c1 - c0, room = a.rows - s.row0;
  s.len = (int)(len < 0 ? 0 : len > room ? room : len);
  if (c0 < 0 || c0 + s.len > a.outer * a.rows) return s;
  s.off = (c0 + 4 * (int64_t)e.x + 3) & ~(int64_t)3;
  s.on = true;
  return s;
}

// Rows of no sequence that this block's CTA sets to zero: behind a padded sequence's end (its last
// block's), and behind the last sequence of a packed batch (shared out over the spare entries; the
// table always has one).
__device__ __forceinline__ bool idle_rows(const AttnArgs& a, const SeqBlock& s, int64_t i, int64_t* from, int64_t* to) {
  if (a.packed) {
    if (!s.spare) return false;
    const int64_t n = a.counts[1], parts = a.cap - n, part = i - n;
    int64_t end = a.cu[a.B];
    if (end < 0) end = 0;
    const int64_t left = a.rows - end;
    if (left <= 0) return false;
    *from = end + left * part / parts;
    *to = end + left * (part + 1) / parts;
    return *to > *from;
  }
  if (!s.on || s.first + kAttnBlock < s.len) return false;
  *from = s.len;
  *to = a.rows;
  return *to > *from;
}

// Sets a kernel's dynamic shared memory once per device (each launch of a short sequence would otherwise pay
// for it on the host).
template <typename K>
inline int attn_smem_once(K kernel, int bytes, bool (&done)[64]) {
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 0 && dev < 64 && done[dev]) return ATLAS_OK;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess)
    return fail(ATLAS_ERR_CUDA, "attention: shared memory attribute");
  if (dev >= 0 && dev < 64) done[dev] = true;
  return ATLAS_OK;
}

// Values a head of the padded vectors: every sequence's rows and up to 4 between two, and 128 that a
// tile may read behind the last.
inline int64_t attn_vec_ld(int64_t outer, int64_t rows, int64_t B) { return (outer * rows + 4 * B + 128 + 7) / 4 * 4; }

}  // namespace atlas
