// What the attention kernels share: the arguments, and the view of one block of one sequence.
#pragma once

#include "common.cuh"

namespace atlas {

constexpr int kAttnBlock = 128;  // rows of an entry of the block table
constexpr int kAttnMaxDim = 64;
constexpr int kAttnShort = 16;   // sequences whose gradient attn_delta_kernel makes whole
constexpr int kProbBits = 15;    // the fp16 gradient holds a probability times 2^15

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
  // vec_ld values a head), the counter of work items, and the blocks of more than kAttnShort rows, in no order:
  // sequence, first row, length, prefix sum. fp16 also: the squared norms of dout's rows (norm2, as lse2), and the
  // largest of a sequence and key head as bits, of its query heads' rows of dout (top_dout) and of its rows of v (top_v).
  float *delta, *lse2, *delta2, *norm2;
  int64_t vec_ld;
  uint32_t *top_dout, *top_v, *counter, *listed;
  int4* list;
  const int32_t *cu, *blocks;
  const int64_t* counts;
  int64_t outer, rows, B, cap;
  int H, Hk, D, packed;
  float scale;
};

// One entry of the block table: rows first .. first + 127 of sequence `seq`, whose rows are
// row0 .. row0 + len - 1 of outer index `outer`. Everything is cut to the tensors' extents, so that a
// table or prefix sums that do not belong to these tensors cannot lead outside them; a first row that is not a
// multiple of 128 is no entry (the gradient's bulk copies start there, which needs 16 bytes of alignment).
struct SeqBlock {
  int seq, first, len;
  int64_t row0, outer, off;
  bool on;     // an entry with a sequence
  bool spare;  // an entry behind the last
};

__device__ __forceinline__ int64_t seq_off(int seq, int c0) { return (c0 + 4 * (int64_t)seq + 3) & ~(int64_t)3; }

__device__ __forceinline__ SeqBlock seq_block(const AttnArgs& a, int64_t i) {
  SeqBlock s{};
  const int64_t n = a.counts[1];
  const int2 e = reinterpret_cast<const int2*>(a.blocks)[i];  // i < cap: both loads are under way at once
  s.spare = i >= n;
  if (s.spare) return s;
  if (e.x < 0 || e.x >= a.B || e.y < 0 || e.y % kAttnBlock) return s;
  const int64_t c0 = a.cu[e.x], c1 = a.cu[e.x + 1];
  s.seq = e.x;
  s.first = e.y;
  s.row0 = a.packed ? c0 : 0;
  s.outer = a.packed ? 0 : e.x;
  if (s.row0 < 0 || s.row0 > a.rows || s.outer >= a.outer) return s;
  const int64_t len = c1 - c0, room = a.rows - s.row0;
  s.len = (int)(len < 0 ? 0 : len > room ? room : len);
  if (c0 < 0 || c0 + s.len > a.outer * a.rows) return s;
  s.off = seq_off(e.x, (int)c0);
  s.on = true;
  return s;
}

// The last of sequences lo .. hi - 1 before which no more than g of a padded batch's idle rows lie, by a
// warp: 32 of them at a time.
__device__ __forceinline__ int64_t idle_seq(const AttnArgs& a, int64_t lo, int64_t hi, int64_t g, int lane) {
#pragma unroll 1
  while (hi - lo > 1) {
    const int64_t step = (hi - lo + 31) / 32, mid = lo + lane * step;
    const bool below = mid < hi && mid * a.rows - a.cu[mid] <= g;
    const int64_t at = lo + (31 - __clz(__ballot_sync(0xFFFFFFFFu, below) | 1u)) * step;
    lo = at;
    hi = at + step < hi ? at + step : hi;
  }
  return lo;
}

// The rows of no sequence - behind a padded sequence's end, or behind the last sequence of a packed batch -
// in order, shared out evenly over the spare entries of the table. The table has rows / 128 + B + 1 entries
// and a sequence takes at most len / 128 + 1 of them, so that a share is 128 rows or less. (Given to a
// sequence's own last entry, a batch of lengths 505 to 4040 spent 540 us in four CTAs that set thousands
// of rows to zero.)
struct IdleShare {
  int64_t all, left, from, end;  // rows; of no sequence; this share's, numbered
};
__device__ __forceinline__ IdleShare idle_share(const AttnArgs& a, int64_t i) {
  const int64_t n = a.counts[1], used = a.cu[a.B];
  IdleShare s;
  s.all = a.packed ? a.rows : a.outer * a.rows;
  s.left = used < 0 ? s.all : used < s.all ? s.all - used : 0;
  s.from = n < 0 || n > i ? s.left : s.left * (i - n) / (a.cap - n);
  s.end = n < 0 || n > i ? s.left : s.left * (i - n + 1) / (a.cap - n);
  return s;
}

// A lane's row of the share, number n0 + i of it (i < 32): false behind the share's end. For whole warps.
__device__ __forceinline__ bool idle_row(const AttnArgs& a, const IdleShare& s, int64_t n0, int i, int64_t* outer, int64_t* row) {
  const int lane = threadIdx.x % 32;
  const int64_t g0 = s.from + n0, g = g0 + i;
  if (g0 >= s.end) return false;
  int64_t b = 0, r = s.all - s.left + g;
  if (!a.packed) {  // before sequence b lie b * rows - cu[b] of them
    int64_t hi = idle_seq(a, 0, a.B, g0 + 31, lane) + 1;
    b = idle_seq(a, 0, hi, g0, lane);
#pragma unroll 1
    while (hi - b > 1) {
      const int64_t mid = (b + hi) >> 1;
      if (mid * a.rows - a.cu[mid] <= g) b = mid;
      else hi = mid;
    }
    r = g - b * a.rows + a.cu[b + 1];
  }
  *outer = b;
  *row = r;
  return g < s.end && r >= 0 && r < a.rows;
}

// The rows of spare entry i by a CTA of n threads: f(outer, row, sub) by 8 threads for each.
template <typename F>
__device__ __forceinline__ void idle_rows(const AttnArgs& a, int64_t i, int n, F f) {
  const IdleShare s = idle_share(a, i);
#pragma unroll 1
  for (int64_t at = threadIdx.x / 32 * 4; s.from + at < s.end; at += n / 8) {
    int64_t o = 0, r = 0;
    if (idle_row(a, s, at, threadIdx.x % 32 / 8, &o, &r)) f(o, r, threadIdx.x % 8);
  }
}

// The exponents of a row's weights are taken from a reference, and any reference gives the same quotient: it is the
// largest score known when it was chosen, so that a lone key's weight is 1 and nothing is lost to it. A tile's sum of
// weights above 2^room moves it. Before they meet the values the weights (or the values) are scaled by
// 2^-(room + b), b = ceil log2 of how many such sums a row has: all weights together are 1 at most then, and a sum of
// weighted values stays below the largest |v|. It is finite whenever the quotient is, which neither a reference left
// behind by rising scores nor a running maximum (n |v|) gives. Small values pay: what falls below the type's range by the
// scale is lost.
__device__ __forceinline__ int ceil_log2(int n) { return 32 - __clz(n - 1); }  // n >= 1
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// One row of a head set to zero by 8 lanes, 16 bytes at a time where it allows it.
__device__ __forceinline__ void zero_row(void* dst, const Strides& st, int size, int64_t outer, int head, int64_t row, int D, int sub) {
  char* p = reinterpret_cast<char*>(dst) + (outer * st.outer + head * st.head + row * st.row) * size;
  const int bytes = D * size;
  if ((((uintptr_t)p | (uintptr_t)bytes) & 15) == 0) {
    for (int d = sub * 16; d < bytes; d += 128) *reinterpret_cast<uint4*>(p + d) = make_uint4(0, 0, 0, 0);
  } else {
#pragma unroll 1
    for (int d = sub * size; d < bytes; d += 8 * size) {
      if (size == 4) *reinterpret_cast<uint32_t*>(p + d) = 0;
      else *reinterpret_cast<uint16_t*>(p + d) = 0;
    }
  }
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

// Entries of the block table that a batch needs.
__host__ __device__ inline int64_t attn_blocks(int64_t outer, int64_t rows, int64_t B) { return outer * rows / kAttnBlock + B + 1; }

// Values a head of the padded vectors: every sequence's rows and up to 4 between two, and 128 that a
// tile may read behind the last.
inline int64_t attn_vec_ld(int64_t outer, int64_t rows, int64_t B) { return (outer * rows + 4 * B + 128 + 7) / 4 * 4; }

}  // namespace atlas
