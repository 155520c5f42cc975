// Attention over the valid rows and its gradient on CUDA cores: fp32 tensors, and 16-bit ones whose
// strides or width TMA cannot address (the tensor-core kernels take the others).
//
//   S = scale q k^T,  lse = log sum exp S,  out = exp(S - lse) v
//   delta = sum_d dout out,  P = exp(S - lse),  dS = P (dout v^T - delta)
//   dv = P^T dout,  dk = scale dS^T q,  dq = scale dS k
//
// 64 x 64 tiles, 256 threads, each with 4 rows (ty + 16 i) and 4 columns (tx + 16 j) of a tile of
// scores; operands lie in shared memory as fp32 rows of DP + 4 words, read as float4 along the head
// dimension (the 16 tx of a half warp hit distinct banks, the ty broadcast). The next tile's rows are in
// registers on their way while this one is worked on. Scores are in base 2 (the queries carry scale log2 e). The
// exponents' reference comes from the maximum of a row's first tile, with room for 2^8 above it (attn.cuh), and only a
// sum beyond that (or no reference yet: scores of -inf so far) raises it and rescales. The gradient is two kernels, one CTA per key
// tile (dk, dv; all query heads of its key head, one after the other) and one per query tile (dq): scores are
// computed twice, but no sum crosses CTAs, so every result is the same from run to run. 40 sequences of 32 to 402 rows, 20 heads of 16,
// fp32: 194 us forward (3 GFLOP, 0.21 of the FMA rate: the tiles' shared-memory reads and the exponentials' issue).
#include "attn.cuh"

namespace atlas {
namespace {

constexpr int BT = 64;       // rows of a tile
constexpr int PP = 80;       // row pitch of a tile of scores: the two ty of a warp in different bank halves
constexpr int kThreads = 256;
constexpr int kRoom = 8;       // bits that scores may rise above the first tile's before its reference is raised
constexpr int kIdleHeads = 4;  // heads of a CTA that sets rows to zero: its time is the look-up's, 2.5 us
constexpr float kNegInf = -__builtin_inff();

template <int DT>
__device__ __forceinline__ void put(typename Elem<DT>::T* p, float v);
template <>
__device__ __forceinline__ void put<ATLAS_F32>(float* p, float v) { *p = v; }
template <>
__device__ __forceinline__ void put<ATLAS_BF16>(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ void put<ATLAS_F16>(__half* p, float v) { *p = __float2half_rn(v); }

__device__ __forceinline__ float ex2(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// Rows first .. first + 63 of a head, four columns at a time: from memory into registers (zero behind `len` and
// behind D), and from there into shared memory. `vec`: fp32 rows that 16-byte loads may read.
template <int DT, int DP>
struct Tile {
  float4 r[DP / 16];
  __device__ __forceinline__ void fetch(const void* src, const Strides& st, int64_t outer, int head, int64_t row0, int first,
                                        int len, int D, bool vec) {
    using T = typename Elem<DT>::T;
    const T* p = reinterpret_cast<const T*>(src) + outer * st.outer + head * st.head + row0 * st.row;
#pragma unroll
    for (int k = 0; k < DP / 16; ++k) {
      const int i = threadIdx.x + k * kThreads, x = first + i / (DP / 4), d = i % (DP / 4) * 4;
      r[k] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (x < len && d < D) {
        const T* q = p + (int64_t)x * st.row + d;
        if (DT == ATLAS_F32 && vec) {
          r[k] = __ldg(reinterpret_cast<const float4*>(q));
        } else {
          r[k].x = Elem<DT>::f(q[0]);
          if (d + 1 < D) r[k].y = Elem<DT>::f(q[1]);
          if (d + 2 < D) r[k].z = Elem<DT>::f(q[2]);
          if (d + 3 < D) r[k].w = Elem<DT>::f(q[3]);
        }
      }
    }
  }
  __device__ __forceinline__ void put(float* dst, float mul) const {
#pragma unroll
    for (int k = 0; k < DP / 16; ++k) {
      const int i = threadIdx.x + k * kThreads;
      *reinterpret_cast<float4*>(dst + i / (DP / 4) * (DP + 4) + i % (DP / 4) * 4) =
          make_float4(r[k].x * mul, r[k].y * mul, r[k].z * mul, r[k].w * mul);
    }
  }
};

// c[i][j] = sum_d a[ty + 16 i][d] b[tx + 16 j][d]
template <int DP>
__device__ __forceinline__ void mm_rows(const float* a, const float* b, int ty, int tx, float (&c)[4][4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) c[i][j] = 0.f;
#pragma unroll 2
  for (int d = 0; d < DP; d += 4) {
    float4 x[4], y[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[i] = *reinterpret_cast<const float4*>(a + (ty + 16 * i) * (DP + 4) + d);
      y[i] = *reinterpret_cast<const float4*>(b + (tx + 16 * i) * (DP + 4) + d);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        c[i][j] = fmaf(x[i].x, y[j].x, c[i][j]);
        c[i][j] = fmaf(x[i].y, y[j].y, c[i][j]);
        c[i][j] = fmaf(x[i].z, y[j].z, c[i][j]);
        c[i][j] = fmaf(x[i].w, y[j].w, c[i][j]);
      }
  }
}

// acc[i][c] += sum_n p[ty + 16 i][n] v[n][tx C + c]
template <int DP>
__device__ __forceinline__ void mm_cols(const float* p, const float* v, int ty, int tx, float (&acc)[4][DP / 16]) {
  constexpr int C = DP / 16;
#pragma unroll 2
  for (int n = 0; n < BT; n += 4) {
    float4 x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = *reinterpret_cast<const float4*>(p + (ty + 16 * i) * PP + n);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      float y[C];
#pragma unroll
      for (int c = 0; c < C; ++c) y[c] = v[(n + k) * (DP + 4) + tx * C + c];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float w = k == 0 ? x[i].x : k == 1 ? x[i].y : k == 2 ? x[i].z : x[i].w;
#pragma unroll
        for (int c = 0; c < C; ++c) acc[i][c] = fmaf(w, y[c], acc[i][c]);
      }
    }
  }
}

__device__ __forceinline__ float row_max(float v) {
#pragma unroll
  for (int o = 8; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xFFFFFFFFu, v, o));
  return v;
}
__device__ __forceinline__ float row_sum(float v) {
#pragma unroll
  for (int o = 8; o; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  return v;
}

template <int DT, int DP>
__device__ __forceinline__ void store_tile(void* dst, const Strides& st, int64_t outer, int head, int64_t row0, int first, int len,
                                           int D, int ty, int tx, const float (&acc)[4][DP / 16], const float (&mul)[4]) {
  using T = typename Elem<DT>::T;
  constexpr int C = DP / 16;
  T* p = reinterpret_cast<T*>(dst) + outer * st.outer + head * st.head + row0 * st.row;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = first + ty + 16 * i;
    if (r >= len) continue;
#pragma unroll
    for (int c = 0; c < C; ++c)
      if (tx * C + c < D) put<DT>(p + (int64_t)r * st.row + tx * C + c, acc[i][c] * mul[i]);
  }
}

// Short sequences: thread (r, c) makes the score of query r and key c, then 4 columns of a row r of a result.
struct alignas(16) ShortSmem {  // rows are read and written as float4
  float k[kAttnShort][68], v[kAttnShort][68], q[kAttnShort][68], g[kAttnShort][68], p[kAttnShort][20], ds[kAttnShort][20];
};

__device__ __forceinline__ float4& row_of(float (&tile)[kAttnShort][68], int row, int col) {
  return *reinterpret_cast<float4*>(&tile[row][col]);
}
__device__ __forceinline__ void add4(float4& acc, float w, const float4& x) {
  acc.x = fmaf(w, x.x, acc.x);
  acc.y = fmaf(w, x.y, acc.y);
  acc.z = fmaf(w, x.z, acc.z);
  acc.w = fmaf(w, x.w, acc.w);
}
// Columns 4 c .. of row r of a head; vec: rows of whole 16-byte pieces, so that D is a multiple of 4.
template <int DT>
__device__ __forceinline__ float4 short_load(const void* src, const Strides& st, const SeqBlock& b, int head, int r, int c, int D, bool vec) {
  using T = typename Elem<DT>::T;
  const T* p = reinterpret_cast<const T*>(src) + b.outer * st.outer + head * st.head + (b.row0 + r) * st.row + 4 * c;
  float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
  if (r >= b.len) return x;
  if (vec) {
    if (4 * c < D) {
      alignas(16) T w[4];
      if (sizeof(T) == 4) *reinterpret_cast<uint4*>(w) = __ldg(reinterpret_cast<const uint4*>(p));
      else *reinterpret_cast<uint2*>(w) = __ldg(reinterpret_cast<const uint2*>(p));
      x = make_float4(Elem<DT>::f(w[0]), Elem<DT>::f(w[1]), Elem<DT>::f(w[2]), Elem<DT>::f(w[3]));
    }
  } else {
    if (4 * c < D) x.x = Elem<DT>::f(p[0]);
    if (4 * c + 1 < D) x.y = Elem<DT>::f(p[1]);
    if (4 * c + 2 < D) x.z = Elem<DT>::f(p[2]);
    if (4 * c + 3 < D) x.w = Elem<DT>::f(p[3]);
  }
  return x;
}
template <int DT>
__device__ __forceinline__ void short_store(void* dst, const Strides& st, const SeqBlock& b, int head, int r, int c, int D, const float4& x,
                                            float f) {
  using T = typename Elem<DT>::T;
  T* p = reinterpret_cast<T*>(dst) + b.outer * st.outer + head * st.head + (b.row0 + r) * st.row + 4 * c;
  const float w[4] = {x.x * f, x.y * f, x.z * f, x.w * f};
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (r < b.len && 4 * c + e < D) put<DT>(p + e, w[e]);
}

// ---------------------------------------------------------------------------------------- forward
// A short sequence and head: 64 x 64 tiles would be empty for the most part (140 fp32 sequences of 1 to 3 rows, 40 heads
// of 64: 204 us by those, 62 by this).
template <int DT>
__device__ __noinline__ void short_out(const AttnArgs& a, SeqBlock b, int head, ShortSmem& s, bool vec) {
  const int r = threadIdx.x / kAttnShort, c = threadIdx.x % kAttnShort, len = b.len, kh = head / (a.H / a.Hk);
  row_of(s.q, r, 4 * c) = short_load<DT>(a.q, a.sq, b, head, r, c, a.D, vec);
  row_of(s.k, r, 4 * c) = short_load<DT>(a.k, a.sk, b, kh, r, c, a.D, vec);
  row_of(s.v, r, 4 * c) = short_load<DT>(a.v, a.sv, b, kh, r, c, a.D, vec);
  __syncthreads();
  float x = kNegInf;
  if (r < len && c < len) {
    float sc = 0.f;
#pragma unroll 4
    for (int d = 0; d < a.D; d += 4) {
      const float4 u = row_of(s.q, r, d), w = row_of(s.k, c, d);
      sc = fmaf(u.x, w.x, fmaf(u.y, w.y, fmaf(u.z, w.z, fmaf(u.w, w.w, sc))));
    }
    x = sc * (a.scale * kLog2e);
  }
  float m = x;
#pragma unroll
  for (int o = kAttnShort / 2; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
  const float ref = m == kNegInf ? 0.f : m, p = ex2(x - ref);
  float sum = p;
#pragma unroll
  for (int o = kAttnShort / 2; o; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
  s.p[r][c] = p / sum;  // before the values are summed: no sum above the largest of them
  __syncwarp();  // a row's scores are of one half of a warp
  float4 out = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int j = 0; j < len; ++j) add4(out, s.p[r][j], row_of(s.v, j, 4 * c));
  short_store<DT>(a.out, a.so, b, head, r, c, a.D, out, 1.f);
  if (c == 0 && r < len) a.lse[(b.outer * a.H + head) * a.rows + b.row0 + r] = (ref + log2f(sum)) * kLn2;
}

template <int DT, int DP>
__global__ void __launch_bounds__(kThreads, DP == 64 ? 2 : 3) attn_fwd_simt_kernel(const __grid_constant__ AttnArgs a, int vec) {
  extern __shared__ float sm[];
  constexpr int TILE = BT * (DP + 4);
  float *sq = sm, *sk = sm + TILE, *sv = sm + 2 * TILE, *sp = sm + 3 * TILE;
  const int head = blockIdx.y, tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int64_t bi = blockIdx.x >> 1;
  const SeqBlock s = seq_block(a, bi);
  if (s.spare) {
    if (blockIdx.x & 1 || head % kIdleHeads) return;
    idle_rows(a, bi, kThreads, [&](int64_t o, int64_t r, int sub) {
      for (int h = head; h < min(head + kIdleHeads, a.H); ++h) {
        zero_row(a.out, a.so, sizeof(typename Elem<DT>::T), o, h, r, a.D, sub);
        if (sub == 0) a.lse[(o * a.H + h) * a.rows + r] = 0.f;
      }
    });
    return;
  }
  const int first = s.first + (blockIdx.x & 1) * BT;
  if (!s.on || first >= s.len) return;
  if (s.len <= kAttnShort) {
    short_out<DT>(a, s, head, *reinterpret_cast<ShortSmem*>(sm), vec);
    return;
  }
  const int kh = head / (a.H / a.Hk);
  // a thread's sum is that of 4 of a tile's 64 columns
  const float v_scale = pow2(-kRoom - 4 - ceil_log2((s.len + BT - 1) / BT));
  Tile<DT, DP> tk, tv;
  tk.fetch(a.q, a.sq, s.outer, head, s.row0, first, s.len, a.D, vec);
  tk.put(sq, a.scale * kLog2e);
  tk.fetch(a.k, a.sk, s.outer, kh, s.row0, 0, s.len, a.D, vec);
  tv.fetch(a.v, a.sv, s.outer, kh, s.row0, 0, s.len, a.D, vec);
  float m[4], l[4], acc[4][DP / 16];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    m[i] = kNegInf;
    l[i] = 0.f;
#pragma unroll
    for (int c = 0; c < DP / 16; ++c) acc[i][c] = 0.f;
  }
  for (int n0 = 0; n0 < s.len; n0 += BT) {
    __syncthreads();
    tk.put(sk, 1.f);
    tv.put(sv, v_scale);
    __syncthreads();
    if (n0 + BT < s.len) {
      tk.fetch(a.k, a.sk, s.outer, kh, s.row0, n0 + BT, s.len, a.D, vec);
      tv.fetch(a.v, a.sv, s.outer, kh, s.row0, n0 + BT, s.len, a.D, vec);
    }
    float c[4][4];
    mm_rows<DP>(sq, sk, ty, tx, c);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (n0 + tx + 16 * j >= s.len) c[i][j] = kNegInf;
    auto highest = [&](int i) { return row_max(fmaxf(fmaxf(c[i][0], c[i][1]), fmaxf(c[i][2], c[i][3]))); };
    if (n0 == 0) {
#pragma unroll
      for (int i = 0; i < 4; ++i) m[i] = highest(i);
    }
    float e[4][4], sum[4];
    bool bad = false;
    auto powers = [&] {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float ref = m[i] == kNegInf ? 0.f : m[i];
#pragma unroll
        for (int j = 0; j < 4; ++j) e[i][j] = ex2(c[i][j] - ref);
        sum[i] = (e[i][0] + e[i][1]) + (e[i][2] + e[i][3]);
        bad |= m[i] == kNegInf || !(sum[i] <= (float)(1 << kRoom));
      }
    };
    powers();
    if (n0 > 0 && __any_sync(0xFFFFFFFFu, bad)) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float to = fmaxf(m[i], highest(i)), f = m[i] == to || m[i] == kNegInf ? 1.f : ex2(m[i] - to);
        m[i] = to;
        l[i] *= f;
#pragma unroll
        for (int d = 0; d < DP / 16; ++d) acc[i][d] *= f;
      }
      powers();
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      l[i] += sum[i];
#pragma unroll
      for (int j = 0; j < 4; ++j) sp[(ty + 16 * i) * PP + tx + 16 * j] = e[i][j];
    }
    __syncwarp();  // a warp's rows of sp are its own
    mm_cols<DP>(sp, sv, ty, tx, acc);
  }
  float inv[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    l[i] = row_sum(l[i]);
    inv[i] = 1.f / (l[i] * v_scale);
    const int r = first + ty + 16 * i;
    if (tx == 0 && r < s.len) a.lse[(s.outer * a.H + head) * a.rows + s.row0 + r] = ((m[i] == kNegInf ? 0.f : m[i]) + log2f(l[i])) * kLn2;
  }
  store_tile<DT, DP>(a.out, a.so, s.outer, head, s.row0, first, s.len, a.D, ty, tx, acc, inv);
}

// --------------------------------------------------------------------------------------- gradient
// KEYS: this CTA's rows are keys (dk, dv), the loop runs over the queries of every query head of the
// key head; otherwise its rows are queries (dq) and the loop runs over the keys.
template <int DT, int DP, bool KEYS>
__global__ void __launch_bounds__(kThreads, 2) attn_bwd_simt_kernel(const AttnArgs a, int vec) {
  extern __shared__ float sm[];
  constexpr int TILE = BT * (DP + 4);
  // rows of this CTA: k and v (KEYS) or q and dout; of the loop: the other two
  float *s0 = sm, *s1 = sm + TILE, *t0 = sm + 2 * TILE, *t1 = sm + 3 * TILE, *sp = sm + 4 * TILE, *sd = sp + BT * PP,
        *s_lse = sd + BT * PP, *s_delta = s_lse + BT;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4, group = a.H / a.Hk;
  const int64_t bi = blockIdx.x >> 1;
  const SeqBlock s = seq_block(a, bi);
  if (s.spare) {
    if (blockIdx.x & 1 || blockIdx.y % kIdleHeads) return;
    idle_rows(a, bi, kThreads, [&](int64_t o, int64_t r, int sub) {
      constexpr int size = sizeof(typename Elem<DT>::T);
      for (int h = blockIdx.y; h < min((int)blockIdx.y + kIdleHeads, (int)gridDim.y); ++h) {
        zero_row(KEYS ? a.dk : a.dq, KEYS ? a.sdk : a.sdq, size, o, h, r, a.D, sub);
        if (KEYS) zero_row(a.dv, a.sdv, size, o, h, r, a.D, sub);
      }
    });
    return;
  }
  const int first = s.first + (blockIdx.x & 1) * BT;
  if (!s.on || first >= s.len || s.len <= kAttnShort) return;
  const int kh = KEYS ? blockIdx.y : blockIdx.y / group;
  // the queries' scores in base 2: the factor goes to the tile of queries or keys that stays
  Tile<DT, DP> ta, tb;
  ta.fetch(KEYS ? a.k : a.q, KEYS ? a.sk : a.sq, s.outer, blockIdx.y, s.row0, first, s.len, a.D, vec);
  tb.fetch(KEYS ? a.v : a.dout, KEYS ? a.sv : a.sdo, s.outer, blockIdx.y, s.row0, first, s.len, a.D, vec);
  ta.put(s0, a.scale * kLog2e);
  tb.put(s1, 1.f);
  auto fetch = [&](int h, int n0) {
    ta.fetch(KEYS ? a.q : a.k, KEYS ? a.sq : a.sk, s.outer, KEYS ? h : kh, s.row0, n0, s.len, a.D, vec);
    tb.fetch(KEYS ? a.dout : a.v, KEYS ? a.sdo : a.sv, s.outer, KEYS ? h : kh, s.row0, n0, s.len, a.D, vec);
  };
  fetch(kh * group, 0);
  float g0[4][DP / 16], g1[4][DP / 16];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int c = 0; c < DP / 16; ++c) g0[i][c] = g1[i][c] = 0.f;
  for (int h = KEYS ? kh * group : (int)blockIdx.y; h < (KEYS ? (kh + 1) * group : (int)blockIdx.y + 1); ++h) {
    const float* lse = a.lse + (s.outer * a.H + h) * a.rows + s.row0;
    const float* delta = a.delta + (s.outer * a.H + h) * a.rows + s.row0;
    for (int n0 = 0; n0 < s.len; n0 += BT) {
      __syncthreads();
      ta.put(t0, 1.f);
      tb.put(t1, 1.f);
      const int q0 = KEYS ? n0 : first;
      if (threadIdx.x < BT) {
        const bool on = q0 + (int)threadIdx.x < s.len;
        s_lse[threadIdx.x] = on ? lse[q0 + threadIdx.x] * kLog2e : 0.f;
        s_delta[threadIdx.x] = on ? delta[q0 + threadIdx.x] : 0.f;
      }
      __syncthreads();
      if (n0 + BT < s.len) fetch(h, n0 + BT);
      else if (KEYS && h + 1 < (kh + 1) * group) fetch(h + 1, 0);
      float c[4][4], d[4][4];
      mm_rows<DP>(s0, t0, ty, tx, c);
      mm_rows<DP>(s1, t1, ty, tx, d);
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int qi = KEYS ? tx + 16 * j : ty + 16 * i;
          const bool on = first + ty + 16 * i < s.len && n0 + tx + 16 * j < s.len;
          const float p = on ? ex2(c[i][j] - s_lse[qi]) : 0.f;
          sp[(ty + 16 * i) * PP + tx + 16 * j] = p;
          sd[(ty + 16 * i) * PP + tx + 16 * j] = on ? p * (d[i][j] - s_delta[qi]) : 0.f;
        }
      __syncwarp();
      if (KEYS) mm_cols<DP>(sp, t1, ty, tx, g1);
      mm_cols<DP>(sd, t0, ty, tx, g0);
    }
  }
  const float sc[4] = {a.scale, a.scale, a.scale, a.scale}, one[4] = {1.f, 1.f, 1.f, 1.f};
  if (KEYS) {
    store_tile<DT, DP>(a.dk, a.sdk, s.outer, kh, s.row0, first, s.len, a.D, ty, tx, g0, sc);
    store_tile<DT, DP>(a.dv, a.sdv, s.outer, kh, s.row0, first, s.len, a.D, ty, tx, g1, one);
  } else {
    store_tile<DT, DP>(a.dq, a.sdq, s.outer, blockIdx.y, s.row0, first, s.len, a.D, ty, tx, g0, sc);
  }
}

// The gradient of a sequence of up to kAttnShort rows and one key head: thread (r, c) makes the score of
// query r and key c, then 4 columns of row r of dq, dk and dv. Tiles of 64 and 128 rows would be empty for the
// most part: 288 pairs of rows with 10 heads took 90 us in the tensor-core kernel's items, 3 us each. Over few keys
// dP and delta lie close together as well, and the rounding of a 16-bit out would be the gradients' largest
// error (bf16, D = 8, relative norm of dq 5.4e-3 at 2 keys, 4.3e-3 at 4, 3.6e-3 at 16; the rounding of the
// result alone is 1.7e-3): here delta is sum_j P_j dP_j, and dS stays in 32 bits.
template <int DT, bool VEC>
__device__ __forceinline__ void short_grad(const AttnArgs& a, const SeqBlock& b, int kh, ShortSmem& s) {
  using T = typename Elem<DT>::T;
  static_assert(kThreads == kAttnShort * kAttnShort && kAttnMaxDim == 4 * kAttnShort, "a thread per pair of rows");
  const int r = threadIdx.x / kAttnShort, c = threadIdx.x % kAttnShort, len = b.len, group = a.H / a.Hk;
  auto load = [&](const void* src, const Strides& st, int head) { return short_load<DT>(src, st, b, head, r, c, a.D, VEC); };
  auto store = [&](void* dst, const Strides& st, int head, const float4& x, float f) { short_store<DT>(dst, st, b, head, r, c, a.D, x, f); };
  const bool on = r < len && c < len;
  const float* lses = a.lse + b.outer * a.H * a.rows + b.row0 + r;
  int h = kh * group;
  row_of(s.k, r, 4 * c) = load(a.k, a.sk, kh);
  row_of(s.v, r, 4 * c) = load(a.v, a.sv, kh);
  float4 q = load(a.q, a.sq, h), g = load(a.dout, a.sdo, h), dk = make_float4(0.f, 0.f, 0.f, 0.f), dv = dk;
  float lse = on ? lses[h * a.rows] : 0.f;
#pragma unroll 1
  for (int left = group; left; --left, ++h) {
    row_of(s.q, r, 4 * c) = q;
    row_of(s.g, r, 4 * c) = g;
    __syncthreads();
    float p = 0.f, dp = 0.f, sc = 0.f;
    if (on) {
#pragma unroll 4
      for (int d = 0; d < a.D; d += 4) {
        const float4 x = row_of(s.q, r, d), y = row_of(s.k, c, d), w = row_of(s.g, r, d), z = row_of(s.v, c, d);
        sc = fmaf(x.x, y.x, fmaf(x.y, y.y, fmaf(x.z, y.z, fmaf(x.w, y.w, sc))));
        dp = fmaf(w.x, z.x, fmaf(w.y, z.y, fmaf(w.z, z.z, fmaf(w.w, z.w, dp))));
      }
      p = ex2((sc * a.scale - lse) * kLog2e);
    }
    if (left > 1) {  // the next head's rows are on their way
      q = load(a.q, a.sq, h + 1);
      g = load(a.dout, a.sdo, h + 1);
      lse = on ? lses[(h + 1) * a.rows] : 0.f;
    }
    float delta = p * dp;
#pragma unroll
    for (int m = kAttnShort / 2; m; m >>= 1) delta += __shfl_xor_sync(0xFFFFFFFFu, delta, m);
    s.p[r][c] = p;
    s.ds[r][c] = on ? p * (dp - delta) : 0.f;
    __syncthreads();
    float4 dq = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int j = 0; j < len; ++j) {
      add4(dq, s.ds[r][j], row_of(s.k, j, 4 * c));
      add4(dk, s.ds[j][r], row_of(s.q, j, 4 * c));
      add4(dv, s.p[j][r], row_of(s.g, j, 4 * c));
    }
    store(a.dq, a.sdq, h, dq, a.scale);
    __syncthreads();
  }
  store(a.dk, a.sdk, kh, dk, a.scale);
  store(a.dv, a.sdv, kh, dv, 1.f);
}

// 16 bytes, or one element, of a row: what a lane of the functions below reads of it.
template <int DT, bool VEC>
struct RowPart {
  using T = typename Elem<DT>::T;
  static constexpr int E = VEC ? 16 / sizeof(T) : 1;    // elements per load
  static constexpr int G = VEC ? kAttnMaxDim / E : 32;  // lanes per row
  static constexpr int PER = kThreads / G;              // rows at a time
};

__device__ __forceinline__ float sum_lanes(float v, int n) {
  for (int m = n / 2; m; m >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, m);
  return v;
}
// The largest of a warp's values (none negative; NaN is the largest) into *to, as bits, so that the order does not matter.
__device__ __forceinline__ void raise_top(uint32_t* to, float v) {
  const uint32_t u = __reduce_max_sync(0xFFFFFFFFu, __float_as_uint(fabsf(v)));
  if ((threadIdx.x & 31) == 0) atomicMax(to, u);
}

// delta = sum_d dout out of the rows of a block and head, G lanes to a row: 8 lanes with 16-byte loads where
// rows are aligned for them (VEC), else a warp. fp16: the squared norms of dout's rows as well.
template <int DT, bool VEC>
__device__ __forceinline__ void delta_rows(const AttnArgs& a, const SeqBlock& s, int head) {
  using T = typename Elem<DT>::T;
  constexpr int E = RowPart<DT, VEC>::E, G = RowPart<DT, VEC>::G, PER = RowPart<DT, VEC>::PER;
  constexpr bool NORM = DT == ATLAS_F16;
  const int sub = threadIdx.x % G;
  const T* o = reinterpret_cast<const T*>(a.o) + s.outer * a.so.outer + head * a.so.head + s.row0 * a.so.row;
  const T* g = reinterpret_cast<const T*>(a.dout) + s.outer * a.sdo.outer + head * a.sdo.head + s.row0 * a.sdo.row;
  const int64_t vec_at = head * a.vec_ld + s.off, row_at = (s.outer * a.H + head) * a.rows + s.row0;
  float top = 0.f;
  constexpr int U = VEC ? 4 : 1;  // rows of a thread whose loads are under way at once
#pragma unroll 1
  for (int k0 = 0; k0 < kAttnBlock / PER; k0 += U) {
    const int r0 = s.first + k0 * PER + (int)threadIdx.x / G;
    float v[U] = {}, n2[U] = {}, lse[U] = {};
    uint4 x[U], y[U];
    auto product = [&](int u, T a0, T b0) {
      const float w = Elem<DT>::f(b0);
      v[u] = fmaf(Elem<DT>::f(a0), w, v[u]);
      if (NORM) n2[u] = fmaf(w, w, n2[u]);
    };
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int r = r0 + u * PER;
      const bool on = r < s.len;
      if (VEC) {
        x[u] = y[u] = make_uint4(0, 0, 0, 0);
        if (on && sub * E < a.D) {
          x[u] = __ldg(reinterpret_cast<const uint4*>(o + (int64_t)r * a.so.row + sub * E));
          y[u] = __ldg(reinterpret_cast<const uint4*>(g + (int64_t)r * a.sdo.row + sub * E));
        }
      } else if (on) {
        for (int d = sub; d < a.D; d += G) product(u, o[(int64_t)r * a.so.row + d], g[(int64_t)r * a.sdo.row + d]);
      }
      if (a.lse2 && sub == 0 && on) lse[u] = a.lse[row_at + r];
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int r = r0 + u * PER;
      if (VEC) {
#pragma unroll
        for (int e = 0; e < E; ++e) product(u, reinterpret_cast<const T*>(&x[u])[e], reinterpret_cast<const T*>(&y[u])[e]);
      }
      v[u] = sum_lanes(v[u], G);
      if (NORM) n2[u] = sum_lanes(n2[u], G);
      if (sub == 0 && r < s.len) {
        if (a.lse2) {
          a.lse2[vec_at + r] = fmaf(lse[u], -kLog2e, NORM ? (float)kProbBits : 0.f);
          a.delta2[vec_at + r] = -v[u];
          if (NORM) a.norm2[vec_at + r] = n2[u];
        } else {
          a.delta[row_at + r] = v[u];
        }
      }
      if (NORM) top = n2[u] > top || n2[u] != n2[u] ? n2[u] : top;
    }
  }
  if (NORM && a.lse2) raise_top(a.top_dout + (int64_t)s.seq * a.Hk + head / (a.H / a.Hk), top);
}

// The largest squared norm of rows first .. of a key head's v (fp16; see dS_scale in attn_tc.cu). Out of line: it takes
// only what it needs, so that the kernel's arguments stay where they are.
template <int DT, bool VEC>
__device__ __noinline__ void value_norms(const typename Elem<DT>::T* v, int64_t stride, int first, int len, int D, uint32_t* to) {
  using T = typename Elem<DT>::T;
  constexpr int E = RowPart<DT, VEC>::E, G = RowPart<DT, VEC>::G, PER = RowPart<DT, VEC>::PER;
  const int sub = threadIdx.x % G;
  float top = 0.f;
#pragma unroll 4
  for (int k = 0; k < kAttnBlock / PER; ++k) {
    const int r = first + k * PER + (int)threadIdx.x / G;
    float n2 = 0.f;
    if (r < len) {
      if (VEC) {
        if (sub * E < D) {
          const uint4 x = __ldg(reinterpret_cast<const uint4*>(v + (int64_t)r * stride + sub * E));
#pragma unroll
          for (int e = 0; e < E; ++e) {
            const float w = Elem<DT>::f(reinterpret_cast<const T*>(&x)[e]);
            n2 = fmaf(w, w, n2);
          }
        }
      } else {
        for (int d = sub; d < D; d += G) {
          const float w = Elem<DT>::f(v[(int64_t)r * stride + d]);
          n2 = fmaf(w, w, n2);
        }
      }
    }
    n2 = sum_lanes(n2, G);
    top = n2 > top || n2 != n2 ? n2 : top;
  }
  raise_top(to, top);
}

// Before the gradient's kernels: delta, and the gradients of short sequences; for the tensor-core kernel also
// the list of its blocks, and zero to the rows that it does not write. bf16: 160 MB of out and dout in 39 us,
// 4.1 TB/s (fp16, with the norms of dout's and v's rows, 75 us); what bounds it is the latency of a CTA's loads, two for its entry, then four rows of a thread at once.
template <int DT, bool VEC>
__global__ void __launch_bounds__(kThreads, 4) attn_delta_kernel(const AttnArgs a) {
  __shared__ ShortSmem sm;
  const SeqBlock s = seq_block(a, blockIdx.x);
  const int head = blockIdx.y;
  if (!s.on) {
    if (s.spare && a.lse2 && head % kIdleHeads == 0)
      idle_rows(a, blockIdx.x, kThreads, [&](int64_t o, int64_t r, int sub) {
        constexpr int size = sizeof(typename Elem<DT>::T);
        for (int h = head; h < min(head + kIdleHeads, a.H); ++h) {
          zero_row(a.dq, a.sdq, size, o, h, r, a.D, sub);
          if (h < a.Hk) {
            zero_row(a.dk, a.sdk, size, o, h, r, a.D, sub);
            zero_row(a.dv, a.sdv, size, o, h, r, a.D, sub);
          }
        }
      });
  } else if (s.len > kAttnShort) {
    if (a.lse2 && head == 0 && threadIdx.x == 0 && s.first < s.len) {
      const uint32_t i = atomicAdd(a.listed, 1u);
      if (i < attn_blocks(a.outer, a.rows, a.B)) a.list[i] = make_int4(s.seq, s.first, s.len, a.cu[s.seq]);
    }
    delta_rows<DT, VEC>(a, s, head);
    if (DT == ATLAS_F16 && a.lse2 && head < a.Hk)
      value_norms<DT, VEC>(reinterpret_cast<const typename Elem<DT>::T*>(a.v) + s.outer * a.sv.outer + head * a.sv.head + s.row0 * a.sv.row,
                           a.sv.row, s.first, s.len, a.D, a.top_v + (int64_t)s.seq * a.Hk + head);
  } else if (s.first == 0 && head < a.Hk) {
    short_grad<DT, VEC>(a, s, head, sm);
  }
}

}  // namespace

namespace {
bool rows_of_16(const void* p, const Strides& s, int esize) {
  const int64_t m = 16 / esize;
  return (uintptr_t)p % 16 == 0 && s.row % m == 0 && s.head % m == 0 && s.outer % m == 0;
}
// Whether every row that the kernels load is made of whole 16-byte pieces (fp32).
int vec_rows(const AttnArgs& a, int dtype, bool grad) {
  return dtype == ATLAS_F32 && a.D % 4 == 0 && rows_of_16(a.q, a.sq, 4) && rows_of_16(a.k, a.sk, 4) && rows_of_16(a.v, a.sv, 4) &&
         (!grad || rows_of_16(a.dout, a.sdo, 4));
}
template <int DT>
void launch_delta(const AttnArgs& a, cudaStream_t st) {
  const int size = DT == ATLAS_F32 ? 4 : 2;
  const dim3 grid((unsigned)a.cap, a.H);
  if (a.D * size % 16 == 0 && rows_of_16(a.o, a.so, size) && rows_of_16(a.dout, a.sdo, size) && rows_of_16(a.q, a.sq, size) &&
      rows_of_16(a.k, a.sk, size) && rows_of_16(a.v, a.sv, size))
    attn_delta_kernel<DT, true><<<grid, kThreads, 0, st>>>(a);
  else
    attn_delta_kernel<DT, false><<<grid, kThreads, 0, st>>>(a);
}
}  // namespace

int attn_delta(const AttnArgs& a, int dtype, cudaStream_t st) {
  if (dtype == ATLAS_F32) launch_delta<ATLAS_F32>(a, st);
  else if (dtype == ATLAS_BF16) launch_delta<ATLAS_BF16>(a, st);
  else launch_delta<ATLAS_F16>(a, st);
  return check_launch("attention_grad");
}

namespace {

template <int DT, int DP>
int fwd(const AttnArgs& a, cudaStream_t st) {
  const int bytes = (3 * BT * (DP + 4) + BT * PP) * 4;
  static_assert((3 * BT * (DP + 4) + BT * PP) * 4 >= sizeof(ShortSmem), "short sequences use the same memory");
  static bool done[64] = {};
  if (int rc = attn_smem_once(attn_fwd_simt_kernel<DT, DP>, bytes, done)) return rc;
  attn_fwd_simt_kernel<DT, DP><<<dim3((unsigned)(2 * a.cap), a.H), kThreads, bytes, st>>>(a, vec_rows(a, DT, false));
  return check_launch("attention");
}

template <int DT, int DP>
int bwd(const AttnArgs& a, cudaStream_t st) {
  const int bytes = (4 * BT * (DP + 4) + 2 * BT * PP + 2 * BT) * 4;
  static bool done[2][64] = {};
  if (int rc = attn_smem_once(attn_bwd_simt_kernel<DT, DP, true>, bytes, done[0])) return rc;
  if (int rc = attn_smem_once(attn_bwd_simt_kernel<DT, DP, false>, bytes, done[1])) return rc;
  if (int rc = attn_delta(a, DT, st)) return rc;
  const int vec = vec_rows(a, DT, true);
  attn_bwd_simt_kernel<DT, DP, true><<<dim3((unsigned)(2 * a.cap), a.Hk), kThreads, bytes, st>>>(a, vec);
  attn_bwd_simt_kernel<DT, DP, false><<<dim3((unsigned)(2 * a.cap), a.H), kThreads, bytes, st>>>(a, vec);
  return check_launch("attention_grad");
}

template <int DT>
int dispatch(const AttnArgs& a, bool grad, cudaStream_t st) {
  if (a.D <= 16) return grad ? bwd<DT, 16>(a, st) : fwd<DT, 16>(a, st);
  if (a.D <= 32) return grad ? bwd<DT, 32>(a, st) : fwd<DT, 32>(a, st);
  return grad ? bwd<DT, 64>(a, st) : fwd<DT, 64>(a, st);
}

}  // namespace

int attn_simt(const AttnArgs& a, int dtype, bool grad, cudaStream_t st) {
  switch (dtype) {
    case ATLAS_F32: return dispatch<ATLAS_F32>(a, grad, st);
    case ATLAS_BF16: return dispatch<ATLAS_BF16>(a, grad, st);
    default: return dispatch<ATLAS_F16>(a, grad, st);
  }
}

}  // namespace atlas
