// Log probabilities of given tokens with entropy, ranks and the most likely alternatives, and the
// gradient into the logits (atlas_token_logprobs, atlas_token_logprobs_grad).
//
// Per row x[0..V), M a running maximum:
//   Z = sum e^(x - M),  T = sum e^(x - M) (x - M),  lse = M + log Z,
//   entropy = log Z - T / Z,  logprob_j = (x[t_j] - M) - log Z,
//   rank_j = 1 + #{v : x_v > x[t_j]},  top = the n largest, ties to the lowest index,
//   dx_v = p_v (-sum_j g_j - g_H (log p_v + entropy)) + sum_{j : t_j = v} g_j.
// One read of the row: a larger maximum rescales Z and T (T <- e^(M-M') (T + Z (M - M'))). The
// difference x - M is taken before the factor log2 e, so that logits at the type's lowest value stay
// finite, and T holds the distances from the maximum, so that a sharp row's small entropy is no
// difference of large numbers. Sums are fp32. A term is ex2 of the rounded product d log2 e, off by |d| 2^-24 and 2 units
// of the last place: of Z that is sum p |d| 2^-24, at most (entropy + log Z) 2^-24, the size of the rounding that lse itself
// takes: the shorter form is enough.
//
// Rows: a row whose logits are all -inf has lse = -inf, log probability -inf, entropy 0 and a zero
// gradient; a NaN or +inf makes the row's numbers NaN (NaN counts as the largest among the
// alternatives). A token outside [0, V) stands for "none": log probability 0, rank 0, no gradient.
#include <cooperative_groups.h>

#include "common.cuh"

namespace atlas {
namespace {

namespace cg = cooperative_groups;

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kNegInf = -__builtin_inff();
constexpr int kMaxTop = 32;     // alternatives: one per lane of a warp
constexpr int kMaxGiven = 64;   // tokens per row
constexpr uint32_t kFull = 0xFFFFFFFFu;

struct LpArgs {
  const void* x;
  int64_t N, V, ld;
  const int64_t* tok;
  int J, top;
  float* logprob;
  int32_t* rank;
  float *entropy, *lse;
  int64_t* top_id;
  float* top_logprob;
};

__device__ __forceinline__ float ex2(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

// Two fp32 values as one operand of the packed fp32 instructions.
using f32x2 = unsigned long long;
__device__ __forceinline__ f32x2 pair(float a, float b) {
  f32x2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpair(f32x2 v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
  f32x2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// Order of the alternatives as an unsigned integer: -0 as +0, NaN above all, never 0.
__device__ __forceinline__ uint32_t order_key(float v) {
  if (v != v) return 0xFFFFFFFFu;
  const uint32_t u = __float_as_uint(v + 0.0f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
  if (k == 0xFFFFFFFFu) return __int_as_float(0x7FC00000);
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7FFFFFFFu) : ~k);
}

// Running statistics of a part of a row.
struct Stat {
  float M, Z, T;
};
__device__ __forceinline__ float ref_of(float M) { return M == kNegInf ? 0.f : M; }
__device__ __forceinline__ void raise_to(Stat& s, float M) {  // M >= s.M
  if (s.M != kNegInf) {
    const float d = s.M - M, f = ex2(d * kLog2e);
    s.T = f > 0.f ? f * (s.T + s.Z * d) : f * s.Z;  // f = 0: T vanishes (f Z keeps a NaN)
    s.Z *= f;
  }
  s.M = M;
}
__device__ __forceinline__ void add_term(Stat& s, float x, float ref) {
  const float d = x - ref, e = ex2(d * kLog2e);
  s.Z += e;
  s.T = fmaf(e, fmaxf(d, -1000.f), s.T);  // d = -inf: its term is 0
}
__device__ __forceinline__ Stat join(Stat a, Stat b) {
  const float M = fmaxf(a.M, b.M);
  if (M != kNegInf) {
    raise_to(a, M);
    raise_to(b, M);
  }
  return Stat{M, a.Z + b.Z, a.T + b.T};
}
__device__ __forceinline__ Stat warp_join(Stat s) {
#pragma unroll
  for (int o = 16; o; o >>= 1)
    s = join(s, Stat{__shfl_xor_sync(kFull, s.M, o), __shfl_xor_sync(kFull, s.Z, o), __shfl_xor_sync(kFull, s.T, o)});
  return s;
}
// (log Z, lse, entropy) of a finished row
__device__ __forceinline__ void finish(const Stat& s, float* lz, float* lse, float* ent) {
  *lz = logf(s.Z);
  if (s.M == kNegInf && s.Z == 0.f) {  // every logit -inf
    *lse = kNegInf;
    *ent = 0.f;
  } else {
    *lse = ref_of(s.M) + *lz;
    *ent = *lz - s.T / s.Z;
  }
}
__device__ __forceinline__ float logprob_of(float x, const Stat& s, float lz, float lse) {
  return lse == kNegInf ? kNegInf : (x - ref_of(s.M)) - lz;
}

// ------------------------------------------------------------------------------------ short rows
// V <= 32 NE: a warp keeps a whole row in registers (v = lane + 32 e). The alternatives are n rounds
// of two warp reductions (largest key, then lowest index among its holders). 30973 x 33 bf16: 9 us without
// alternatives, 16 with five (2 MB: the reductions, one after the other, are what it takes); 8191 x 33 fp32 with 20
// tokens 5.5 us.
template <int DT, int NE>
__global__ void __launch_bounds__(256) logprobs_short_kernel(const LpArgs a) {
  using T = typename Elem<DT>::T;
  const int lane = threadIdx.x & 31;
  const int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (row >= a.N) return;
  const int V = (int)a.V;
  const T* xr = reinterpret_cast<const T*>(a.x) + row * a.ld;
  float x[NE];
  float mx = kNegInf;
#pragma unroll
  for (int e = 0; e < NE; ++e) {
    const int v = lane + 32 * e;
    x[e] = v < V ? Elem<DT>::f(xr[v]) : kNegInf;
    mx = fmaxf(mx, x[e]);
  }
  Stat s{mx, 0.f, 0.f};
#pragma unroll
  for (int o = 16; o; o >>= 1) s.M = fmaxf(s.M, __shfl_xor_sync(kFull, s.M, o));
  const float ref = ref_of(s.M);
#pragma unroll
  for (int e = 0; e < NE; ++e) add_term(s, x[e], ref);
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    s.Z += __shfl_xor_sync(kFull, s.Z, o);
    s.T += __shfl_xor_sync(kFull, s.T, o);
  }
  float lz, lse, ent;
  finish(s, &lz, &lse, &ent);
  if (lane == 0) {
    a.lse[row] = lse;
    a.entropy[row] = ent;
  }
  for (int j0 = 0; j0 < a.J; j0 += 32) {
    const int nj = min(32, a.J - j0);
    const int64_t t = lane < nj ? a.tok[row * a.J + j0 + lane] : -1;
    const bool on = t >= 0 && t < V;
    const float xt = on ? Elem<DT>::f(xr[t]) : 0.f;
    int rank = 0;
    for (int j = 0; j < nj; ++j) {
      const float b = __shfl_sync(kFull, xt, j);
      int c = 0;
#pragma unroll
      for (int e = 0; e < NE; ++e) c += __popc(__ballot_sync(kFull, x[e] > b));
      if (lane == j) rank = c + 1;
    }
    if (lane < nj) {
      a.logprob[row * a.J + j0 + lane] = on ? logprob_of(xt, s, lz, lse) : 0.f;
      a.rank[row * a.J + j0 + lane] = on ? rank : 0;
    }
  }
  if (a.top) {
    uint32_t key[NE];
#pragma unroll
    for (int e = 0; e < NE; ++e) key[e] = lane + 32 * e < V ? order_key(x[e]) : 0u;
    int my_id = 0;
    float my_x = 0.f;
    for (int i = 0; i < a.top; ++i) {
      uint32_t best = 0;
#pragma unroll
      for (int e = 0; e < NE; ++e) best = max(best, key[e]);
      best = __reduce_max_sync(kFull, best);
      uint32_t id = 0xFFFFFFFFu;
#pragma unroll
      for (int e = NE - 1; e >= 0; --e)
        if (key[e] == best) id = lane + 32 * e;
      id = __reduce_min_sync(kFull, id);
#pragma unroll
      for (int e = 0; e < NE; ++e)
        if (id == (uint32_t)(lane + 32 * e)) key[e] = 0u;
      if (lane == i) {
        my_id = (int)id;
        my_x = key_value(best);
      }
    }
    if (lane < a.top) {
      a.top_id[row * a.top + lane] = my_id;
      a.top_logprob[row * a.top + lane] = logprob_of(my_x, s, lz, lse);
    }
  }
}

// ------------------------------------------------------------------------------------- long rows
// A cluster of CL CTAs shares one row (CL = 1 where there are rows enough to fill the GPU), each CTA
// streams its part with 16-byte loads. Alternatives: each warp keeps its 32 best so far as 64-bit
// keys (order << 32 | ~index), sorted over the lanes; what beats the n-th of them is collected in
// shared memory, and every 32 of those are sorted (bitonic) and merged into the list.
// Threads of a CTA: 128 where rows fill the GPU (4095 x 50003 bf16: 98 us, 256 threads 104, 512 144: a row's
// start and end overlap with other rows), 512 where a cluster shares one row (65537 bf16: 14 us, 128 20). With
// alternatives registers are kept to 64, so that 8 CTAs or 2 fit an SM: with 20 of them 950 x 74074 bf16 took 197 us without that, 145
// with it (25 rows: 35 and 27; one row of 65537: 17 and 19).
constexpr int long_threads(int CL) { return CL == 1 ? 128 : 512; }
constexpr int long_ctas(int CL, bool top) { return !top ? 0 : CL == 1 ? 8 : 2; }
constexpr int kLongUnroll = 2;

__device__ __forceinline__ uint64_t shfl_xor64(uint64_t v, int o) { return __shfl_xor_sync(kFull, v, o); }

// Largest first over the lanes, from any bitonic sequence.
__device__ __forceinline__ uint64_t bitonic_merge(uint64_t v, int lane) {
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    const uint64_t w = shfl_xor64(v, o);
    v = ((lane & o) == 0) == (v > w) ? v : w;
  }
  return v;
}
template <typename K>
__device__ __forceinline__ K warp_sort_desc(K v, int lane) {
#pragma unroll
  for (int k = 2; k <= 32; k <<= 1)
#pragma unroll
    for (int o = k >> 1; o; o >>= 1) {
      const K w = __shfl_xor_sync(kFull, v, o);
      const bool first = ((lane & o) == 0) == ((lane & k) == 0);
      v = first == (v > w) ? v : w;
    }
  return v;
}
// The 32 largest of two lists that are sorted largest first.
__device__ __forceinline__ uint64_t merge_lists(uint64_t a, uint64_t b, int lane) {
  const uint64_t r = __shfl_sync(kFull, b, 31 - lane);
  return bitonic_merge(a > r ? a : r, lane);
}

// A warp's alternatives, in shared memory, and their code out of line: few values of a row get there, and in
// registers, with a copy in every vector's code, they made kernels of 95 to 130 KB.
struct TopState {
  uint64_t list[32];  // largest first, one a lane
  uint64_t buf[64];   // waiting
  uint64_t bar;       // the n-th entry: what must be beaten
  int held;           // entries waiting
};

__device__ __forceinline__ uint64_t full_key(uint32_t k, uint32_t id) { return ((uint64_t)k << 32) | (uint32_t)~id; }

// 16 bytes of a row as the kernels look at them: the largest, and how many are above a given value. For
// 16-bit types both two values at a time (max passes over a NaN, a comparison with one is false).
template <int DT>
struct Vec {
  using T = typename Elem<DT>::T;
  static constexpr int N = 16 / sizeof(T);
  uint4 raw;
  __device__ __forceinline__ float at(int i) const { return Elem<DT>::f(reinterpret_cast<const T*>(&raw)[i]); }
  __device__ __forceinline__ float top() const {
    if constexpr (DT == ATLAS_F32) {
      return fmaxf(fmaxf(at(0), at(1)), fmaxf(at(2), at(3)));
    } else if constexpr (DT == ATLAS_BF16) {
      const auto* w = reinterpret_cast<const __nv_bfloat162*>(&raw);
      const __nv_bfloat162 m = __hmax2(__hmax2(w[0], w[1]), __hmax2(w[2], w[3]));
      return fmaxf(__low2float(m), __high2float(m));
    } else {
      const auto* w = reinterpret_cast<const __half2*>(&raw);
      const __half2 m = __hmax2(__hmax2(w[0], w[1]), __hmax2(w[2], w[3]));
      return fmaxf(__low2float(m), __high2float(m));
    }
  }
  // x: a value of the row's type
  __device__ __forceinline__ int above(float x) const {
    if constexpr (DT == ATLAS_F32) {
      return (at(0) > x) + (at(1) > x) + (at(2) > x) + (at(3) > x);
    } else if constexpr (DT == ATLAS_BF16) {
      const auto* w = reinterpret_cast<const __nv_bfloat162*>(&raw);
      const __nv_bfloat162 b = __float2bfloat162_rn(x);
      const __nv_bfloat162 n = __hadd2(__hadd2(__hgt2(w[0], b), __hgt2(w[1], b)), __hadd2(__hgt2(w[2], b), __hgt2(w[3], b)));
      return (int)(__low2float(n) + __high2float(n));
    } else {
      const auto* w = reinterpret_cast<const __half2*>(&raw);
      const __half2 b = __float2half2_rn(x);
      const __half2 n = __hadd2(__hadd2(__hgt2(w[0], b), __hgt2(w[1], b)), __hadd2(__hgt2(w[2], b), __hgt2(w[3], b)));
      return (int)(__low2float(n) + __high2float(n));
    }
  }
  __device__ static __forceinline__ uint4 lowest() {  // -inf throughout
    const uint32_t u = DT == ATLAS_F32 ? 0xFF800000u : DT == ATLAS_BF16 ? 0xFF80FF80u : 0xFC00FC00u;
    return make_uint4(u, u, u, u);
  }
};

// Sorts 32 of the waiting entries and merges them into the list.
__device__ __noinline__ void top_flush(TopState& s, int n, int lane) {
  const int held = s.held;
  const uint64_t v = lane < held ? s.buf[lane] : 0;
  const uint64_t rest = lane + 32 < held ? s.buf[lane + 32] : 0;
  const uint64_t list = merge_lists(s.list[lane], warp_sort_desc(v, lane), lane);
  const uint64_t nth = __shfl_sync(kFull, list, n - 1), bar = s.bar;
  __syncwarp();
  s.list[lane] = list;
  s.buf[lane] = rest;
  if (lane == 0) {
    s.held = max(0, held - 32);
    if (nth > bar) s.bar = nth;
  }
  __syncwarp();
}

// Offers the first `count` values of each lane's vector, columns v .. (`on`: there are any), and returns the
// order key that a value has to reach from now on. mx is the largest value that the lane has met: the n-th
// largest of those is a bar too, since n entries are as large. It starts the bar, and raises it at every call
// where few are wanted and a sort of 32 costs less than the values that would come without it (950 x 74074
// bf16: 5 alternatives 103 us, 115 with the start alone; 20: 167 and 145).
constexpr int kRaiseTop = 8;
template <int DT>
__device__ __noinline__ uint32_t top_offer(TopState& s, uint4 raw, int count, bool on, uint32_t v, float mx, int n, int lane) {
  using T = typename Elem<DT>::T;
  uint64_t bar = s.bar;
  int held = s.held;
  if (bar == 0 || n <= kRaiseTop) {
    const uint32_t largest = order_key(mx);
    const uint32_t nth = n == 1 ? __reduce_max_sync(kFull, largest) : __shfl_sync(kFull, warp_sort_desc(largest, lane), n - 1);
    const uint64_t below = ((uint64_t)nth << 32) - 1;
    if (below > bar) {
      bar = below;
      __syncwarp();
      if (lane == 0) s.bar = bar;
    }
  }
  uint32_t mine = 0;  // which of the lane's values reach the bar
#pragma unroll
  for (int i = 0; i < 16 / (int)sizeof(T); ++i) {
    const float x = Elem<DT>::f(reinterpret_cast<const T*>(&raw)[i]);
    mine |= (uint32_t)(on && i < count && order_key(x) >= (uint32_t)(bar >> 32)) << i;
  }
#pragma unroll 1
  for (uint32_t left = __reduce_or_sync(kFull, mine); left; left &= left - 1) {
    const int i = __ffs(left) - 1;
    constexpr int per = 4 / sizeof(T);
    const int w = i / per;
    const uint32_t word = w < 2 ? (w == 0 ? raw.x : raw.y) : w == 2 ? raw.z : raw.w;
    float x;
    if constexpr (DT == ATLAS_F32) x = __uint_as_float(word);
    else if constexpr (DT == ATLAS_BF16) x = __uint_as_float(i & 1 ? word & 0xFFFF0000u : word << 16);
    else x = __half2float(__ushort_as_half((unsigned short)(i & 1 ? word >> 16 : word & 0xFFFFu)));
    const uint64_t key = on ? full_key(order_key(x), v + i) : 0;
    const bool in = key > bar;
    const uint32_t m = __ballot_sync(kFull, in);
    if (!m) continue;
    if (in) s.buf[held + __popc(m & ((1u << lane) - 1))] = key;
    held += __popc(m);
    __syncwarp();
    if (held >= 32) {
      if (lane == 0) s.held = held;
      __syncwarp();
      top_flush(s, n, lane);
      held -= 32;
      bar = s.bar;
    }
  }
  __syncwarp();
  if (lane == 0) s.held = held;
  __syncwarp();
  return (uint32_t)(bar >> 32);
}

// A warp's view of them while it streams its part of a row.
struct Top {
  TopState* s;
  uint32_t bar;  // order key
  int n;
};

template <int G>
struct Given {
  float x[G];
  int c[G];
};

// The columns v .. of one vector of this lane (`on`: there is one; the others are all -inf).
template <int DT, int G, bool STATS, bool TOP>
__device__ __forceinline__ void take(const Vec<DT>& q, bool on, uint32_t v, int lane, Stat& s, Given<G>& g, Top& top) {
  constexpr int N = Vec<DT>::N;
  if (STATS) {
    const float mx = q.top();
    if (TOP) {
      // NaN sorts first: the maximum passes over it, so it is looked for apart
      bool any = false;
#pragma unroll
      for (int i = 0; i < N; ++i) any |= q.at(i) != q.at(i);
      any |= order_key(mx) >= top.bar;
      if (__any_sync(kFull, on && any)) top.bar = top_offer<DT>(*top.s, q.raw, N, on, v, fmaxf(s.M, mx), top.n, lane);
    }
    if (mx > s.M) raise_to(s, mx);
    const float ref = ref_of(s.M);
    const f32x2 nref = pair(-ref, -ref), l2 = pair(kLog2e, kLog2e);
    f32x2 z = 0, t = 0;
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      float d0, d1, e0, e1;
      const f32x2 d = add2(pair(q.at(i), q.at(i + 1)), nref);
      unpair(mul2(d, l2), e0, e1);
      unpair(d, d0, d1);
      const f32x2 e = pair(ex2(e0), ex2(e1));
      z = add2(z, e);
      t = fma2(e, pair(fmaxf(d0, -1000.f), fmaxf(d1, -1000.f)), t);  // d = -inf: its term is 0
    }
    float z0, z1, t0, t1;
    unpair(z, z0, z1);
    unpair(t, t0, t1);
    s.Z += z0 + z1;
    s.T += t0 + t1;
  }
#pragma unroll
  for (int k = 0; k < G; ++k) g.c[k] += q.above(g.x[k]);
}

// One single column for each lane of a warp.
template <int DT, int G, bool STATS, bool TOP>
__device__ __forceinline__ void take_one(float x, bool on, uint32_t v, int lane, Stat& s, Given<G>& g, Top& top) {
  if (STATS) {
    if (TOP) {
      uint4 raw = make_uint4(__float_as_uint(x), 0, 0, 0);
      if (DT == ATLAS_BF16) raw.x >>= 16;
      if (DT == ATLAS_F16) raw.x = __half_as_ushort(__float2half_rn(x));  // exact: x is one
      top.bar = top_offer<DT>(*top.s, raw, 1, on, v, fmaxf(s.M, x), top.n, lane);
    }
    if (x > s.M) raise_to(s, x);
    add_term(s, x, ref_of(s.M));
  }
#pragma unroll
  for (int k = 0; k < G; ++k) g.c[k] += x > g.x[k];
}

template <int DT, int G, int NT, bool STATS, bool TOP>
__device__ __forceinline__ void stream_row(const typename Elem<DT>::T* xr, int c0, int c1, Stat& s, Given<G>& g, Top& top) {
  using T = typename Elem<DT>::T;
  constexpr int VEC = 16 / sizeof(T), U = kLongUnroll;
  const int lane = threadIdx.x & 31;
  // columns up to the first 16-byte boundary and behind the last: one each for the lanes of warp 0
  const int mis = (int)((reinterpret_cast<uintptr_t>(xr + c0) & 15) / sizeof(T));
  const int head = min(c1 - c0, mis ? VEC - mis : 0);
  const int nvec = (c1 - c0 - head) / VEC;
  const int b0 = c0 + head, t0 = b0 + nvec * VEC;
  if (threadIdx.x < 32) {
    const int v = lane < head ? c0 + lane : t0 + lane - head;
    const bool on = v < c1;
    take_one<DT, G, STATS, TOP>(on ? Elem<DT>::f(xr[v]) : kNegInf, on, v, lane, s, g, top);
  }
  // U vectors of a thread are under way while the U before them are worked on
  const uint4* xv = reinterpret_cast<const uint4*>(xr + b0);
  Vec<DT> q[2][U];
  auto fetch = [&](int i0, Vec<DT>(&r)[U]) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u * NT + (int)threadIdx.x;
      r[u].raw = i < nvec ? __ldg(xv + i) : Vec<DT>::lowest();
    }
  };
  auto work = [&](int i0, const Vec<DT>(&r)[U]) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u * NT + (int)threadIdx.x;
      if (i0 + u * NT + (int)(threadIdx.x & ~31u) >= nvec) break;  // the whole warp is behind the end
      take<DT, G, STATS, TOP>(r[u], i < nvec, b0 + i * VEC, lane, s, g, top);
    }
  };
  constexpr int STEP = U * NT;
  fetch(0, q[0]);
  for (int i0 = 0; i0 < nvec; i0 += 2 * STEP) {
    fetch(i0 + STEP, q[1]);
    work(i0, q[0]);
    fetch(i0 + 2 * STEP, q[0]);
    work(i0 + STEP, q[1]);
  }
}

template <int NT>
struct LongSmem {
  TopState top[NT / 32];
  uint64_t list[32];
  Stat warp[NT / 32], cta;
  int cnt[kMaxGiven];
};

template <int DT, int G, int CL, bool TOP>
__global__ void __launch_bounds__(long_threads(CL), long_ctas(CL, TOP)) logprobs_long_kernel(const LpArgs a) {
  using T = typename Elem<DT>::T;
  constexpr int NT = long_threads(CL), NW = NT / 32;
  __shared__ LongSmem<NT> sm;
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int64_t row = blockIdx.x / CL;
  const int part = blockIdx.x % CL;
  const int V = (int)a.V;
  const T* xr = reinterpret_cast<const T*>(a.x) + row * a.ld;
  const int c0 = (int)((int64_t)V * part / CL), c1 = (int)((int64_t)V * (part + 1) / CL);
  Stat s{kNegInf, 0.f, 0.f};
  Top top{&sm.top[w], 0, max(a.top, 1)};
  if (TOP) {
    sm.top[w].list[lane] = 0;
    if (lane == 0) sm.top[w].bar = sm.top[w].held = 0;
  }
  if (threadIdx.x < kMaxGiven) sm.cnt[threadIdx.x] = 0;
  __syncthreads();
  for (int j0 = 0; j0 == 0 || j0 < a.J; j0 += G) {
    Given<G> g;
#pragma unroll
    for (int k = 0; k < G; ++k) {
      const int64_t t = j0 + k < a.J ? a.tok[row * a.J + j0 + k] : -1;
      g.x[k] = t >= 0 && t < V ? Elem<DT>::f(xr[t]) : -kNegInf;
      g.c[k] = 0;
    }
    if (j0 == 0) stream_row<DT, G, NT, true, TOP>(xr, c0, c1, s, g, top);
    else stream_row<DT, G, NT, false, false>(xr, c0, c1, s, g, top);
#pragma unroll
    for (int k = 0; k < G; ++k) {
      const int c = __reduce_add_sync(kFull, g.c[k]);
      if (lane == 0 && j0 + k < a.J) atomicAdd(&sm.cnt[j0 + k], c);  // integers: any order
    }
  }
  s = warp_join(s);
  if (lane == 0) sm.warp[w] = s;
  if (TOP) {
    while (sm.top[w].held > 0) top_flush(sm.top[w], top.n, lane);
  }
  __syncthreads();
  for (int o = NW / 2; TOP && o; o >>= 1) {
    if (w < o) sm.top[w].list[lane] = merge_lists(sm.top[w].list[lane], sm.top[w + o].list[lane], lane);
    __syncthreads();
  }
  if (w == 0) {
    s = lane < NW ? sm.warp[lane] : Stat{kNegInf, 0.f, 0.f};
    s = warp_join(s);
    if (lane == 0) sm.cta = s;
    sm.list[lane] = TOP ? sm.top[0].list[lane] : 0;
  }
  cg::cluster_group cl = cg::this_cluster();
  if (CL > 1) cl.sync();
  if (CL > 1 && TOP && part == 0) {  // the parts' lists, merged by a tree of warps
    if (w < CL) sm.top[w].list[lane] = cl.map_shared_rank(&sm, w < CL ? w : 0)->list[lane];
    __syncthreads();
    for (int o = CL / 2; o; o >>= 1) {
      if (w < o) sm.top[w].list[lane] = merge_lists(sm.top[w].list[lane], sm.top[w + o].list[lane], lane);
      __syncthreads();
    }
  }
  if (part == 0 && w == 0) {
    const uint64_t list = CL > 1 ? sm.top[0].list[lane] : sm.list[lane];
    if (CL > 1) {
      s = lane < CL ? cl.map_shared_rank(&sm, lane < CL ? lane : 0)->cta : Stat{kNegInf, 0.f, 0.f};
      s = warp_join(s);
    }
    float lz, lse, ent;
    finish(s, &lz, &lse, &ent);
    if (lane == 0) {
      a.lse[row] = lse;
      a.entropy[row] = ent;
    }
    for (int j = lane; j < a.J; j += 32) {
      const int64_t t = a.tok[row * a.J + j];
      const bool on = t >= 0 && t < V;
      int c = 1;
      if (CL > 1)
        for (int r = 0; r < CL; ++r) c += cl.map_shared_rank(&sm, r)->cnt[j];
      else
        c += sm.cnt[j];
      a.logprob[row * a.J + j] = on ? logprob_of(Elem<DT>::f(xr[t]), s, lz, lse) : 0.f;
      a.rank[row * a.J + j] = on ? c : 0;
    }
    if (TOP && lane < a.top) {
      a.top_id[row * a.top + lane] = (int64_t)(uint32_t)~(uint32_t)list;
      a.top_logprob[row * a.top + lane] = logprob_of(key_value((uint32_t)(list >> 32)), s, lz, lse);
    }
  }
  if (CL > 1) cl.sync();  // no CTA leaves while its shared memory may be read
}

// -------------------------------------------------------------------------------------- gradient
struct GradArgs {
  const void* x;
  int64_t N, V, ld;
  const int64_t* tok;
  int J;
  const float *lse, *entropy, *g_logprob, *g_entropy;  // either g may be null
  void* dx;
  int64_t ldd;
};

template <int DT>
__device__ __forceinline__ void put(typename Elem<DT>::T* p, float v);
template <>
__device__ __forceinline__ void put<ATLAS_F32>(float* p, float v) { *p = v; }
template <>
__device__ __forceinline__ void put<ATLAS_BF16>(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ void put<ATLAS_F16>(__half* p, float v) { *p = __float2half_rn(v); }

// What a row's gradient needs: y = log p = (x - m) - lz, dx = p (a - b y).
struct RowGrad {
  float m, lz, a, b;
  bool none;  // no logit above -inf: zero gradient
};
// lse alone gives log p = x - lse an error of half a step of lse: beyond this the row's maximum and
// log Z are taken again, apart (2^-24 64 = 4e-6 of p).
constexpr float kLseFar = 64.f;
__device__ __forceinline__ RowGrad row_grad(const GradArgs& a, int64_t row, float gsum) {
  const float lse = a.lse[row], gh = a.g_entropy ? a.g_entropy[row] : 0.f;
  return RowGrad{lse, 0.f, -gsum - (a.g_entropy ? gh * a.entropy[row] : 0.f), gh, lse == kNegInf};
}
__device__ __forceinline__ bool is_far(const RowGrad& r) { return !r.none && fabsf(r.m) > kLseFar; }
__device__ __forceinline__ float grad_of(const RowGrad& r, float x) {
  const float y = (x - r.m) - r.lz, p = ex2(y * kLog2e);
  return r.none ? 0.f : p * fmaf(-r.b, fmaxf(y, -1000.f), r.a);
}

// V <= 32 NE: one warp per row. 30973 x 33 bf16: 7.6 us.
template <int DT, int NE>
__global__ void __launch_bounds__(256) logprobs_grad_short_kernel(const GradArgs a) {
  using T = typename Elem<DT>::T;
  const int lane = threadIdx.x & 31;
  const int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (row >= a.N) return;
  const int V = (int)a.V;
  const T* xr = reinterpret_cast<const T*>(a.x) + row * a.ld;
  T* dr = reinterpret_cast<T*>(a.dx) + row * a.ldd;
  float x[NE], d[NE];
#pragma unroll
  for (int e = 0; e < NE; ++e) {
    const int v = lane + 32 * e;
    x[e] = v < V ? Elem<DT>::f(xr[v]) : kNegInf;
    d[e] = 0.f;
  }
  float gsum = 0.f;
  for (int j0 = 0; a.g_logprob && j0 < a.J; j0 += 32) {
    const int nj = min(32, a.J - j0);
    int64_t t = lane < nj ? a.tok[row * a.J + j0 + lane] : -1;
    if (t < 0 || t >= V) t = -1;
    const float g = t >= 0 ? a.g_logprob[row * a.J + j0 + lane] : 0.f;
    for (int j = 0; j < nj; ++j) {
      const float gj = __shfl_sync(kFull, g, j);
      const int tj = __shfl_sync(kFull, (int)t, j);
      gsum += gj;
#pragma unroll
      for (int e = 0; e < NE; ++e)
        if (tj == lane + 32 * e) d[e] += gj;
    }
  }
  RowGrad r = row_grad(a, row, gsum);
  if (is_far(r)) {
    Stat s{kNegInf, 0.f, 0.f};
#pragma unroll
    for (int e = 0; e < NE; ++e) s.M = fmaxf(s.M, x[e]);
#pragma unroll
    for (int o = 16; o; o >>= 1) s.M = fmaxf(s.M, __shfl_xor_sync(kFull, s.M, o));
#pragma unroll
    for (int e = 0; e < NE; ++e) s.Z += ex2((x[e] - ref_of(s.M)) * kLog2e);
#pragma unroll
    for (int o = 16; o; o >>= 1) s.Z += __shfl_xor_sync(kFull, s.Z, o);
    r.m = ref_of(s.M);
    r.lz = logf(s.Z);
  }
#pragma unroll
  for (int e = 0; e < NE; ++e) {
    const int v = lane + 32 * e;
    if (v < V) put<DT>(dr + v, r.none ? 0.f : grad_of(r, x[e]) + d[e]);
  }
}

// Longer rows: grid (parts, rows); a CTA writes its part of the row, then the threads that hold the
// first occurrence of a token in that part write that column again with the sum of its tokens' terms.
// 4095 x 50003 bf16: 147 us, 5.6 TB/s, 0.85 of a copy's rate.
constexpr int kGradThreads = 256;

template <int DT>
__global__ void __launch_bounds__(kGradThreads) logprobs_grad_long_kernel(const GradArgs a, int part_cols) {
  using T = typename Elem<DT>::T;
  constexpr int VEC = 16 / sizeof(T);
  __shared__ int s_tok[kMaxGiven];
  __shared__ float s_g[kMaxGiven];
  __shared__ Stat s_stat[kGradThreads / 32];
  const int V = (int)a.V;
  for (int64_t row = blockIdx.y; row < a.N; row += gridDim.y) {
    const T* xr = reinterpret_cast<const T*>(a.x) + row * a.ld;
    T* dr = reinterpret_cast<T*>(a.dx) + row * a.ldd;
    const int J = a.g_logprob ? a.J : 0;
    __syncthreads();
    if (threadIdx.x < J) {
      const int64_t t = a.tok[row * a.J + threadIdx.x];
      const bool on = t >= 0 && t < V;
      s_tok[threadIdx.x] = on ? (int)t : -1;
      s_g[threadIdx.x] = on ? a.g_logprob[row * a.J + threadIdx.x] : 0.f;
    }
    __syncthreads();
    float gsum = 0.f;
    for (int j = 0; j < J; ++j) gsum += s_g[j];
    RowGrad r = row_grad(a, row, gsum);
    if (is_far(r)) {
      Stat s{kNegInf, 0.f, 0.f};
      for (int v = threadIdx.x; v < V; v += kGradThreads) {
        const float x = Elem<DT>::f(xr[v]);
        if (x > s.M) raise_to(s, x);
        add_term(s, x, ref_of(s.M));
      }
      s = warp_join(s);
      if ((threadIdx.x & 31) == 0) s_stat[threadIdx.x >> 5] = s;
      __syncthreads();
      s = s_stat[0];
      for (int i = 1; i < kGradThreads / 32; ++i) s = join(s, s_stat[i]);
      r.m = ref_of(s.M);
      r.lz = logf(s.Z);
    }
    const int c0 = blockIdx.x * part_cols, c1 = min(V, c0 + part_cols);
    // 16-byte accesses where the two rows are aligned alike, else single ones
    const int mis = (int)((reinterpret_cast<uintptr_t>(xr + c0) & 15) / sizeof(T));
    const bool alike = ((reinterpret_cast<uintptr_t>(xr + c0) ^ reinterpret_cast<uintptr_t>(dr + c0)) & 15) == 0;
    const int head = alike ? min(c1 - c0, mis ? VEC - mis : 0) : c1 - c0;
    const int nvec = (c1 - c0 - head) / VEC, b0 = c0 + head, t0 = b0 + nvec * VEC;
    for (int v = c0 + threadIdx.x; v < b0; v += kGradThreads) put<DT>(dr + v, grad_of(r, Elem<DT>::f(xr[v])));
    for (int v = t0 + threadIdx.x; v < c1; v += kGradThreads) put<DT>(dr + v, grad_of(r, Elem<DT>::f(xr[v])));
    const f32x2 nm = pair(-r.m, -r.m), nlz = pair(-r.lz, -r.lz), l2 = pair(kLog2e, kLog2e), ga = pair(r.a, r.a), gb = pair(-r.b, -r.b);
    constexpr int U = 4;
    for (int i0 = threadIdx.x; i0 < nvec; i0 += U * kGradThreads) {
      uint4 raw[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (i0 + u * kGradThreads < nvec) raw[u] = __ldcs(reinterpret_cast<const uint4*>(xr + b0) + i0 + u * kGradThreads);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (i0 + u * kGradThreads >= nvec) break;
        const T* e = reinterpret_cast<const T*>(&raw[u]);
        uint4 out;
        T* o = reinterpret_cast<T*>(&out);
#pragma unroll
        for (int k = 0; k < VEC; k += 2) {
          float y0, y1, p0, p1;
          const f32x2 y = add2(add2(pair(Elem<DT>::f(e[k]), Elem<DT>::f(e[k + 1])), nm), nlz);
          unpair(mul2(y, l2), p0, p1);
          unpair(y, y0, y1);
          unpair(mul2(pair(ex2(p0), ex2(p1)), fma2(gb, pair(fmaxf(y0, -1000.f), fmaxf(y1, -1000.f)), ga)), p0, p1);
          put<DT>(o + k, r.none ? 0.f : p0);
          put<DT>(o + k + 1, r.none ? 0.f : p1);
        }
        __stcs(reinterpret_cast<uint4*>(dr + b0) + i0 + u * kGradThreads, out);
      }
    }
    __syncthreads();
    if (threadIdx.x < J) {
      const int t = s_tok[threadIdx.x];
      bool first = t >= c0 && t < c1 && !r.none;
      float g = 0.f;
      for (int j = 0; j < J; ++j)
        if (s_tok[j] == t) {
          if (j < (int)threadIdx.x) first = false;
          g += s_g[j];
        }
      if (first) put<DT>(dr + t, grad_of(r, Elem<DT>::f(xr[t])) + g);
    }
  }
}

template <int DT, int CL, bool TOP>
void launch_long(const cudaLaunchConfig_t& cfg, const LpArgs& a) {
  if (a.J <= 1) cudaLaunchKernelEx(&cfg, logprobs_long_kernel<DT, 1, CL, TOP>, a);
  else cudaLaunchKernelEx(&cfg, logprobs_long_kernel<DT, 8, CL, TOP>, a);
}

template <int DT>
int launch_fwd(const LpArgs& a, cudaStream_t st) {
  const unsigned warps = (unsigned)((a.N + 7) / 8);
  if (a.V <= 64) logprobs_short_kernel<DT, 2><<<warps, 256, 0, st>>>(a);
  else if (a.V <= 256) logprobs_short_kernel<DT, 8><<<warps, 256, 0, st>>>(a);
  else if (a.V <= 1024) logprobs_short_kernel<DT, 32><<<warps, 256, 0, st>>>(a);
  else {
    // few rows: eight CTAs to a row, joined over the cluster's shared memory
    const bool split = a.N < num_sms() && a.V >= 8192;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = 8;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.gridDim = dim3((unsigned)(split ? a.N * 8 : a.N));
    cfg.blockDim = dim3(long_threads(split ? 8 : 1));
    cfg.stream = st;
    cfg.attrs = at;
    cfg.numAttrs = split ? 1 : 0;
    if (split) a.top ? launch_long<DT, 8, true>(cfg, a) : launch_long<DT, 8, false>(cfg, a);
    else a.top ? launch_long<DT, 1, true>(cfg, a) : launch_long<DT, 1, false>(cfg, a);
  }
  return check_launch("token_logprobs");
}

template <int DT>
int launch_grad(const GradArgs& a, cudaStream_t st) {
  const unsigned warps = (unsigned)((a.N + 7) / 8);
  if (a.V <= 64) logprobs_grad_short_kernel<DT, 2><<<warps, 256, 0, st>>>(a);
  else if (a.V <= 256) logprobs_grad_short_kernel<DT, 8><<<warps, 256, 0, st>>>(a);
  else {
    // at most 16384 columns a CTA, fewer (down to 2048) where the rows alone leave SMs idle
    int64_t part = a.V * a.N / (4 * num_sms()) / 2048 * 2048;
    part = part < 2048 ? 2048 : part > 16384 ? 16384 : part;
    logprobs_grad_long_kernel<DT><<<dim3((unsigned)((a.V + part - 1) / part), (unsigned)(a.N < 65535 ? a.N : 65535)),
                                    kGradThreads, 0, st>>>(a, (int)part);
  }
  return check_launch("token_logprobs_grad");
}

}  // namespace
}  // namespace atlas

using namespace atlas;

extern "C" int atlas_token_logprobs(const void* logits, int dtype, int64_t N, int64_t V, int64_t ld, const int64_t* tokens,
                                    int64_t J, int64_t top, float* logprob, int32_t* rank, float* entropy, float* lse,
                                    int64_t* top_id, float* top_logprob, void* stream) {
  ATLAS_REQUIRE(N >= 0 && V >= 1 && V < (1LL << 30) && N < (1LL << 27) && ld >= V, "token_logprobs: bad shape");
  ATLAS_REQUIRE(J >= 0 && J <= kMaxGiven, "token_logprobs: at most %d tokens a row", kMaxGiven);
  ATLAS_REQUIRE(top >= 0 && top <= kMaxTop && top <= V, "token_logprobs: top must be in [0, min(%d, V)]", kMaxTop);
  if (N == 0) return ATLAS_OK;
  ATLAS_REQUIRE(logits && entropy && lse && (!J || (tokens && logprob && rank)) && (!top || (top_id && top_logprob)),
                "token_logprobs: null pointer");
  const LpArgs a{logits, N, V, ld, tokens, (int)J, (int)top, logprob, rank, entropy, lse, top_id, top_logprob};
  cudaStream_t st = (cudaStream_t)stream;
  switch (dtype) {
    case ATLAS_F32: return launch_fwd<ATLAS_F32>(a, st);
    case ATLAS_BF16: return launch_fwd<ATLAS_BF16>(a, st);
    case ATLAS_F16: return launch_fwd<ATLAS_F16>(a, st);
    default: return fail(ATLAS_ERR_ARG, "token_logprobs: unknown dtype %d", dtype);
  }
}

extern "C" int atlas_token_logprobs_grad(const void* logits, int dtype, int64_t N, int64_t V, int64_t ld,
                                         const int64_t* tokens, int64_t J, const float* lse, const float* entropy,
                                         const float* g_logprob, const float* g_entropy, void* dlogits, int64_t ldd,
                                         void* stream) {
  ATLAS_REQUIRE(N >= 0 && V >= 1 && V < (1LL << 30) && N < (1LL << 27) && ld >= V && ldd >= V,
                "token_logprobs_grad: bad shape");
  ATLAS_REQUIRE(J >= 0 && J <= kMaxGiven, "token_logprobs_grad: at most %d tokens a row", kMaxGiven);
  if (N == 0) return ATLAS_OK;
  ATLAS_REQUIRE(logits && lse && dlogits && (!g_entropy || entropy) && (!(J && g_logprob) || tokens),
                "token_logprobs_grad: null pointer");
  const GradArgs a{logits, N, V, ld, tokens, (int)J, lse, entropy, J ? g_logprob : nullptr, g_entropy, dlogits, ldd};
  cudaStream_t st = (cudaStream_t)stream;
  switch (dtype) {
    case ATLAS_F32: return launch_grad<ATLAS_F32>(a, st);
    case ATLAS_BF16: return launch_grad<ATLAS_BF16>(a, st);
    case ATLAS_F16: return launch_grad<ATLAS_F16>(a, st);
    default: return fail(ATLAS_ERR_ARG, "token_logprobs_grad: unknown dtype %d", dtype);
  }
}
