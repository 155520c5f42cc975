// Row maps of a batch built on the device from its sequences' lengths (atlas_seq_maps): prefix sums,
// the row and token id of every kept position, and the table of 128-row blocks that attention walks.
//
// With n_b the lengths, k_b = max(n_b - lead - trail, 0) the kept positions and
// t_b = max(1, ceil(n_b / 128)) the blocks of sequence b, everything is a search in prefix sums:
//   cu[b] = sum_{c<b} n_c;  output i belongs to the b with sum_{c<b} k_c <= i < sum_{c<=b} k_c.
// Nothing is computed beyond that: the floor is one launch and the 16 bytes a row written once. So
// the outputs, not the sequences, are what the CTAs share out (one long sequence is as even as many
// short ones), each thread writes two rows with one 16-byte store per array, and up to 1024
// sequences every CTA scans the lengths again for itself in shared memory (4 KB from L2) instead of
// waiting for a scan kernel. Above that two launches of one CTA per 1024 sequences (totals, then prefix sums)
// write to the workspace what the last one searches; its CTAs have long runs of outputs, so that the search
// for a run's first and last sequence (a warp's, 4 dependent reads for 65536) is paid once a CTA and not a thread. The
// kept positions' prefix sums of a run are then staged in shared memory; those of the blocks are not, and each entry of
// the block table searches the run's part of them in global memory.
#include "common.cuh"

namespace atlas {
namespace {

constexpr int kTile = 128;        // rows of a block
constexpr int kScan = 1024;       // sequences one CTA scans
constexpr int kThreads = 512;
constexpr int kRowsPerCta = 2 * kThreads;
constexpr int kStage = 1024;      // sequences whose prefix sums a CTA keeps in shared memory

struct MapArgs {
  const void* len;
  int len64;
  int64_t B, rows, stride, lead, trail;  // stride 0: packed
  const int64_t* seq;
  int32_t* cu;
  int64_t *slots, *tok;
  int32_t* blocks;
  int64_t cap;
  int64_t* counts;
  // More than 1024 sequences: totals of each 1024, and inclusive prefix sums [B].
  int64_t* total;
  int32_t *kept_end, *blk_end;
};

__device__ __forceinline__ int64_t raw_len(const MapArgs& a, int64_t b) {
  return a.len64 ? reinterpret_cast<const int64_t*>(a.len)[b] : (int64_t) reinterpret_cast<const int32_t*>(a.len)[b];
}

// A length outside [0, stride] (packed: [0, rows]) is cut to it and counted.
__device__ __forceinline__ int cut_len(const MapArgs& a, int64_t b, int* bad) {
  const int64_t n = raw_len(a, b), hi = a.stride ? a.stride : a.rows;
  const int64_t m = n < 0 ? 0 : (n > hi ? hi : n);
  *bad += m != n;
  return (int)m;
}
__device__ __forceinline__ int kept_of(const MapArgs& a, int n) {
  const int64_t k = (int64_t)n - a.lead - a.trail;
  return k > 0 ? (int)k : 0;
}
__device__ __forceinline__ int blocks_of(int n) { return n <= 0 ? 1 : (n + kTile - 1) / kTile; }

__device__ __forceinline__ int64_t warp_sum64(int64_t v) {
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  return v;
}

// Sum over the block (every thread gets it); `red` holds one slot per warp.
__device__ int64_t block_sum64(int64_t v, int64_t* red) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  v = warp_sum64(v);
  __syncthreads();
  if (lane == 0) red[w] = v;
  __syncthreads();
  return warp_sum64(lane < (int)blockDim.x / 32 ? red[lane] : 0);
}

// Inclusive scan over the block of one int per thread plus `base`; `red` holds one slot per warp.
__device__ int block_scan(int v, int base, int* red) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  int x = v;
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xFFFFFFFFu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();
  if (lane == 31) red[w] = x;
  __syncthreads();
  for (int i = 0; i < w; ++i) base += red[i];
  return base + x;
}

// First index in [lo, hi) whose inclusive prefix sum is above i.
__device__ __forceinline__ int upper(const int32_t* end, int lo, int hi, int i) {
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (end[mid] > i) hi = mid;
    else lo = mid + 1;
  }
  return lo;
}

// The same by a warp: 32 probes a step, so that 65536 sequences take 4 dependent reads and not 16.
__device__ __forceinline__ int upper_warp(const int32_t* end, int lo, int hi, int i) {
  const int lane = threadIdx.x & 31;
  while (lo < hi) {
    const int step = (hi - lo + 31) / 32, at = lo + lane * step;
    // probes at the last element of each of 32 parts
    const int probe = at + step - 1 < hi ? at + step - 1 : hi - 1;
    const uint32_t above = __ballot_sync(0xFFFFFFFFu, at >= hi || end[probe] > i);
    const int part = __ffs(above) - 1;  // the first part whose last element is above i
    if (above == 0) return hi;
    const int from = lo + part * step;
    if (from >= hi) return hi;
    if (step == 1) return from;
    lo = from;
    hi = from + step < hi ? from + step : hi;
  }
  return lo;
}

// The outputs of this CTA, an even share of each kind, from the inclusive prefix sums of kept positions and
// blocks. NARROW: those are in global memory, and four warps first look for the sequences of the share's
// first and last outputs.
template <bool NARROW>
__device__ void fill(const MapArgs& a, const int32_t* kept_end, const int32_t* blk_end, const int32_t* cu) {
  __shared__ int s_range[4];
  __shared__ int32_t s_end[NARROW ? kStage : 1], s_first[NARROW ? kStage : 1];
  const int B = (int)a.B;
  const int total = kept_end[B - 1], nblk = blk_end[B - 1];
  const int64_t rper = (a.rows + 2 * gridDim.x - 1) / (2 * gridDim.x) * 2, row0 = blockIdx.x * rper;
  const int64_t row1 = row0 + rper < a.rows ? row0 + rper : a.rows;
  const int64_t bper = (a.cap + gridDim.x - 1) / gridDim.x, blk0 = blockIdx.x * bper;
  const int64_t blk1 = blk0 + bper < a.cap ? blk0 + bper : a.cap;
  int lo = 0, hi = B, blo = 0, bhi = B;
  if (NARROW) {
    const int w = threadIdx.x >> 5;
    if (w < 4) {
      const bool last = w & 1, rows = w < 2;
      const int n = rows ? total : nblk;
      int64_t i = rows ? (last ? row1 - 1 : row0) : (last ? blk1 - 1 : blk0);
      if (i > n - 1) i = n - 1;
      const int at = n ? upper_warp(rows ? kept_end : blk_end, 0, B, (int)(i < 0 ? 0 : i)) : 0;
      if ((threadIdx.x & 31) == 0) s_range[w] = at;
    }
    __syncthreads();
    lo = s_range[0];
    hi = s_range[1] + 1;
    blo = s_range[2];
    bhi = s_range[3] + 1;
    if (hi - lo <= kStage) {  // the share's part of the prefix sums in shared memory, indexed from lo
      for (int i = threadIdx.x; i < hi - lo; i += kThreads) {
        s_end[i] = kept_end[lo + i];
        s_first[i] = lo + i ? kept_end[lo + i - 1] : 0;
      }
      __syncthreads();
    }
  }
  const bool staged = NARROW && hi - lo <= kStage;
  for (int64_t i0 = row0 + threadIdx.x * 2; i0 < row1; i0 += 2 * kThreads) {
    int64_t s[2], t[2];
    int b = i0 >= total ? B : staged ? lo + upper(s_end, 0, hi - lo, (int)i0) : upper(kept_end, lo, hi, (int)i0);
    for (int e = 0; e < 2; ++e) {
      const int64_t i = i0 + e;
      if (i >= total) {
        s[e] = t[e] = -1;
        continue;
      }
      if (staged) {
        if (s_end[b - lo] <= i) b = lo + upper(s_end, b + 1 - lo, hi - lo, (int)i);
      } else if (kept_end[b] <= i) {
        b = upper(kept_end, b + 1, hi, (int)i);
      }
      const int64_t p = i - (staged ? s_first[b - lo] : b ? kept_end[b - 1] : 0);
      s[e] = (a.stride ? b * a.stride : (int64_t)cu[b]) + a.lead + p;
      t[e] = (a.seq ? a.seq[b] : (int64_t)b) * 1024 + p;  // core.pack_tok
    }
    if (i0 + 1 < a.rows) {
      *reinterpret_cast<longlong2*>(a.slots + i0) = make_longlong2(s[0], s[1]);
      *reinterpret_cast<longlong2*>(a.tok + i0) = make_longlong2(t[0], t[1]);
    } else {
      a.slots[i0] = s[0];
      a.tok[i0] = t[0];
    }
  }
  for (int64_t i = blk0 + threadIdx.x; i < blk1; i += kThreads) {
    int2 e = make_int2(-1, -1);
    if (i < nblk) {
      const int b = upper(blk_end, blo, bhi, (int)i);
      e = make_int2(b, ((int)i - (b ? blk_end[b - 1] : 0)) * kTile);
    }
    reinterpret_cast<int2*>(a.blocks)[i] = e;
  }
}

// One launch: every CTA scans all (at most 1024) lengths, two a thread. 109 sequences in 32918 rows: 4.9 us.
__global__ void __launch_bounds__(kThreads) maps_small_kernel(const MapArgs a) {
  __shared__ int32_t s_kept[kScan], s_blk[kScan], s_cu[kScan + 1];
  __shared__ int64_t red64[kThreads / 32];
  __shared__ int red[kThreads / 32];
  const int B = (int)a.B;
  const int b0 = 2 * threadIdx.x;
  int bad = 0;
  int n0 = b0 < B ? cut_len(a, b0, &bad) : 0;
  int n1 = b0 + 1 < B ? cut_len(a, b0 + 1, &bad) : 0;
  const int64_t sum = block_sum64((int64_t)n0 + n1, red64);
  int64_t nbad = block_sum64(bad, red64);
  if (sum > a.rows) {  // the sequences do not fit: no map at all rather than one that is wrong
    n0 = n1 = 0;
    nbad += 1;
  }
  const int k0 = b0 < B ? kept_of(a, n0) : 0, k1 = b0 + 1 < B ? kept_of(a, n1) : 0;
  const int t0 = b0 < B ? blocks_of(n0) : 0, t1 = b0 + 1 < B ? blocks_of(n1) : 0;
  const int ec = block_scan(n0 + n1, 0, red), ek = block_scan(k0 + k1, 0, red), et = block_scan(t0 + t1, 0, red);
  if (b0 < B) {
    s_cu[b0] = ec - n1 - n0;
    s_kept[b0] = ek - k1;
    s_blk[b0] = et - t1;
  }
  if (b0 + 1 < B) {
    s_cu[b0 + 1] = ec - n1;
    s_kept[b0 + 1] = ek;
    s_blk[b0 + 1] = et;
  }
  if (blockIdx.x == 0) {
    if (b0 < B) a.cu[b0] = ec - n1 - n0;
    if (b0 + 1 < B) a.cu[b0 + 1] = ec - n1;
    if (b0 == B - 1 || b0 + 1 == B - 1) {
      a.cu[B] = ec;
      a.counts[0] = ek;
      a.counts[1] = et;
      a.counts[2] = nbad;
    }
  }
  __syncthreads();
  fill<false>(a, s_kept, s_blk, s_cu);
}

// Three launches (65536 sequences of 1 to 64 rows: 3.8, 5.6 and 15.6 us, 36 MB written), the first: rows, kept
// positions, blocks and misfits of each 1024 sequences.
__global__ void __launch_bounds__(kScan) maps_total_kernel(const MapArgs a) {
  __shared__ int64_t red64[kScan / 32];
  const int64_t b = (int64_t)blockIdx.x * kScan + threadIdx.x;
  int bad = 0;
  const int n = b < a.B ? cut_len(a, b, &bad) : 0;
  const int64_t t[4] = {block_sum64(n, red64), block_sum64(b < a.B ? kept_of(a, n) : 0, red64),
                        block_sum64(b < a.B ? blocks_of(n) : 0, red64), block_sum64(bad, red64)};
  if (threadIdx.x < 4) a.total[blockIdx.x * 4 + threadIdx.x] = t[threadIdx.x];
}

// The second: the totals before a CTA's own sequences, and the scan of those.
__global__ void __launch_bounds__(kScan) maps_scan_kernel(const MapArgs a) {
  __shared__ int64_t red64[kScan / 32];
  __shared__ int red[kScan / 32];
  int64_t all = 0, nbad = 0, pc = 0, pk = 0, pt = 0;
  for (int64_t c = threadIdx.x; c < gridDim.x; c += kScan) {
    const int64_t* t = a.total + c * 4;
    all += t[0];
    nbad += t[3];
    if (c < blockIdx.x) {
      pc += t[0];
      pk += t[1];
      pt += t[2];
    }
  }
  all = block_sum64(all, red64);
  nbad = block_sum64(nbad, red64);
  pc = block_sum64(pc, red64);
  pk = block_sum64(pk, red64);
  pt = block_sum64(pt, red64);
  const int64_t first = (int64_t)blockIdx.x * kScan, b = first + threadIdx.x;
  const bool on = b < a.B, fits = all <= a.rows;
  if (!fits) {  // no map at all: every sequence empty, which still has one block
    pc = pk = 0;
    pt = first;
    nbad += 1;
  }
  int ignore = 0;
  const int n = on && fits ? cut_len(a, b, &ignore) : 0;
  const int ec = block_scan(n, (int)pc, red);
  const int ek = block_scan(on ? kept_of(a, n) : 0, (int)pk, red);
  const int et = block_scan(on ? blocks_of(n) : 0, (int)pt, red);
  if (!on) return;
  a.cu[b] = ec - n;
  a.kept_end[b] = ek;
  a.blk_end[b] = et;
  if (b == a.B - 1) {
    a.cu[a.B] = ec;
    a.counts[0] = ek;
    a.counts[1] = et;
    a.counts[2] = nbad;
  }
}

__global__ void __launch_bounds__(kThreads) maps_fill_kernel(const MapArgs a) {
  fill<true>(a, a.kept_end, a.blk_end, a.cu);
}

}  // namespace
}  // namespace atlas

using namespace atlas;

extern "C" int64_t atlas_seq_maps_ws_bytes(int64_t B) {
  return B > kScan ? 8 * B + 32 * ((B + kScan - 1) / kScan) : 0;
}

extern "C" int atlas_seq_maps(const void* lengths, int lengths_i64, int64_t B, int64_t rows, int64_t stride, int64_t lead,
                              int64_t trail, const int64_t* seq, int32_t* cu, int64_t* slots, int64_t* tok,
                              int32_t* blocks, int64_t* counts, void* ws, int64_t ws_bytes, void* stream) {
  ATLAS_REQUIRE(B >= 1 && rows >= 1 && rows < (1LL << 31) - 1 && B < (1LL << 30), "seq_maps: bad shape (B=%lld, rows=%lld)",
                (long long)B, (long long)rows);
  ATLAS_REQUIRE(stride >= 0 && lead >= 0 && trail >= 0 && lead < (1LL << 31) && trail < (1LL << 31),
                "seq_maps: stride, lead and trail must not be negative");
  ATLAS_REQUIRE(stride == 0 || stride <= rows / B, "seq_maps: %lld sequences of stride %lld do not fit %lld rows",
                (long long)B, (long long)stride, (long long)rows);
  ATLAS_REQUIRE(lengths && cu && slots && tok && blocks && counts, "seq_maps: null pointer");
  ATLAS_REQUIRE(((uintptr_t)slots | (uintptr_t)tok) % 16 == 0 && (uintptr_t)blocks % 8 == 0,
                "seq_maps: slots and tok must be 16-byte aligned, blocks 8-byte aligned");
  ATLAS_REQUIRE(ws_bytes >= atlas_seq_maps_ws_bytes(B) && (ws || B <= kScan), "seq_maps: workspace too small");
  ATLAS_REQUIRE((uintptr_t)ws % 8 == 0, "seq_maps: the workspace must be 8-byte aligned");
  MapArgs a{lengths, lengths_i64, B, rows, stride, lead, trail, seq, cu, slots, tok, blocks, rows / kTile + B + 1, counts,
            (int64_t*)ws, nullptr, nullptr};
  cudaStream_t st = (cudaStream_t)stream;
  // 1024 outputs a CTA while there are few, else an even share of a grid that is resident at once
  const int64_t want = (rows + kRowsPerCta - 1) / kRowsPerCta, most = 4 * num_sms();
  const unsigned grid = (unsigned)(want < most ? want : most);
  if (B <= kScan) {
    maps_small_kernel<<<grid, kThreads, 0, st>>>(a);
  } else {
    const unsigned parts = (unsigned)((B + kScan - 1) / kScan);
    a.kept_end = (int32_t*)(a.total + 4 * parts);
    a.blk_end = a.kept_end + B;
    maps_total_kernel<<<parts, kScan, 0, st>>>(a);
    maps_scan_kernel<<<parts, kScan, 0, st>>>(a);
    maps_fill_kernel<<<grid, kThreads, 0, st>>>(a);
  }
  return check_launch("seq_maps");
}
