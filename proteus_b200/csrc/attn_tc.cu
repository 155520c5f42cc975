// Attention over the valid rows and its gradient on tcgen05 tensor cores, for bf16 and fp16 tensors
// whose strides TMA can address (head dimension up to 64; narrower heads are zero-filled to 64 by the
// TMA box, which costs nothing that bounds these kernels).
//
//   S = scale q k^T,  lse = log sum exp S,  out = exp(S - lse) v
//   delta = sum_d dout out,  P = exp(S - lse),  dS = P (dout v^T - delta)
//   dv = P^T dout,  dk = scale dS^T q,  dq = scale dS k
//
// What bounds them: an SM computes 16 exponentials a clock against 128 x 64 x 2 tensor operations, so a
// 128 x 128 tile of scores costs 1024 clocks of exponentials and 256 to 512 of products. The products
// therefore only have to stay out of the way: operands come by TMA as 128-byte-swizzled rows, scores and
// probabilities live in TMEM (P is written over S as 16-bit and is the next product's A operand
// from there), one thread per row of scores needs no shuffles, and two CTAs per SM alternate.
//
// Rows behind a sequence's end: their columns of S are masked, products stop at the next multiple of
// 16, and the rows up to there are set to zero in shared memory where they are summed over, since
// 0 x NaN is NaN.
//
// Every wait is bounded (see tc.cuh); a wait that gives up records its code and the CTA leaves.
#include "attn.cuh"
#include "tc.cuh"

namespace atlas {

int attn_delta(const AttnArgs& a, int dtype, cudaStream_t st);

namespace {
using namespace tc;

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kNegInf = -__builtin_inff();
constexpr int BM = 128;                     // rows of a CTA
constexpr uint32_t kTile = BM * 128;        // bytes of 128 rows of 64 elements

__device__ __forceinline__ float ex2(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

template <int DT>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  uint32_t r;
  if (DT == ATLAS_BF16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// Zero rows [from, to) of one head (16-bit elements).
__device__ void zero_rows16(void* dst, const Strides& st, int64_t outer, int head, int64_t from, int64_t to, int D) {
  uint16_t* p = reinterpret_cast<uint16_t*>(dst) + outer * st.outer + head * st.head;
  const int64_t n = (to - from) * D;
  for (int64_t i = threadIdx.x; i < n; i += blockDim.x) p[(from + i / D) * st.row + i % D] = 0;
}

// One row of 64 accumulators, times `mul`, as D 16-bit elements; `vec`: 16-byte stores are aligned.
template <int DT>
__device__ __forceinline__ void store_row(void* dst, const float (&acc)[64], float mul, int D, bool vec) {
  if (vec) {
#pragma unroll
    for (int d = 0; d < 64; d += 8)
      if (d < D) {
        uint4 w;
        w.x = pack2<DT>(acc[d] * mul, acc[d + 1] * mul);
        w.y = pack2<DT>(acc[d + 2] * mul, acc[d + 3] * mul);
        w.z = pack2<DT>(acc[d + 4] * mul, acc[d + 5] * mul);
        w.w = pack2<DT>(acc[d + 6] * mul, acc[d + 7] * mul);
        *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(dst) + d) = w;
      }
  } else {
#pragma unroll
    for (int d = 0; d < 64; ++d)
      if (d < D) reinterpret_cast<uint16_t*>(dst)[d] = (uint16_t)pack2<DT>(acc[d] * mul, 0.f);
  }
}

// Zero the rows [from, to) of a tile of 128-byte rows, by the 32 lanes of a warp, and make the tensor
// core see it.
__device__ __forceinline__ void zero_tile_rows(uint8_t* tile, int from, int to, int lane) {
  for (int i = from * 8 + lane; i < to * 8; i += 32) reinterpret_cast<uint4*>(tile)[i] = make_uint4(0, 0, 0, 0);
  fence_async_smem();
  __syncwarp();
}

__device__ __forceinline__ int up16(int n) { return (n + 15) & ~15; }

// ---------------------------------------------------------------------------------------- forward
// Warps 0-3: softmax, one thread per query; warp 4: TMA; warp 5: products and TMEM.
// TMEM: two buffers of 128 columns. S(i) fills buffer i & 1, P(i) overwrites its columns 0-63 as 16-bit,
// P(i) v lands in its columns 64-127. The softmax warps fold P(i-1) v into registers between the
// maximum of S(i) and its exponentials: the product has had that long to finish, and S(i+1)
// can be computed during the exponentials.
constexpr int kFwdThreads = 192;

struct FwdSmem {
  uint8_t q[kTile], k[2][kTile], v[2][kTile];
  uint64_t q_full, k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2], p_full[2], o_full[2], s_free[2];
  uint32_t tmem;
};

template <int DT>
__global__ void __launch_bounds__(kFwdThreads, 2)
attn_fwd_tc_kernel(const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mk,
                   const __grid_constant__ CUtensorMap mv, const AttnArgs a, int vec) {
  extern __shared__ uint8_t raw[];
  FwdSmem& s = *reinterpret_cast<FwdSmem*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  const int head = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const SeqBlock b = seq_block(a, blockIdx.x);
  int64_t z0, z1;
  if (idle_rows(a, b, blockIdx.x, &z0, &z1)) {
    zero_rows16(a.out, a.so, b.outer, head, z0, z1, a.D);
    float* l = a.lse + (b.outer * a.H + head) * a.rows;
    for (int64_t r = z0 + threadIdx.x; r < z1; r += kFwdThreads) l[r] = 0.f;
  }
  if (!b.on || b.first >= b.len) return;
  const int kh = head / (a.H / a.Hk), n = (b.len + BM - 1) / BM;
  const int live = min(4, (b.len - b.first + 31) / 32);  // softmax warps that have a row
  if (threadIdx.x == 0) {
    mbar_init(&s.q_full, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s.k_full[i], 1);
      mbar_init(&s.k_empty[i], 1);
      mbar_init(&s.v_full[i], 1);
      mbar_init(&s.v_empty[i], 1);
      mbar_init(&s.s_full[i], 1);
      mbar_init(&s.o_full[i], 1);
      mbar_init(&s.p_full[i], live * 32);
      mbar_init(&s.s_free[i], live * 32);
    }
    fence_barrier_init();
  }
  if (warp == 5) tmem_alloc(&s.tmem, 256);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s.tmem;

  if (warp == 4) {
    if (lane == 0) {
      const int r0 = (int)b.row0, o = (int)b.outer;
      mbar_arrive_expect_tx(&s.q_full, kTile);
      tma_load_4d(s.q, &mq, 0, r0 + b.first, head, o, &s.q_full);
      for (int i = 0; i < n; ++i) {
        const int st = i & 1;
        const uint32_t ph = ((i >> 1) & 1) ^ 1;
        if (i >= 2 && !mbar_wait(&s.k_empty[st], ph, 201)) break;
        mbar_arrive_expect_tx(&s.k_full[st], kTile);
        tma_load_4d(s.k[st], &mk, 0, r0 + i * BM, kh, o, &s.k_full[st]);
        if (i >= 2 && !mbar_wait(&s.v_empty[st], ph, 202)) break;
        mbar_arrive_expect_tx(&s.v_full[st], kTile);
        tma_load_4d(s.v[st], &mv, 0, r0 + i * BM, kh, o, &s.v_full[st]);
      }
    }
  } else if (warp == 5) {
    const uint32_t base = DT == ATLAS_BF16 ? idesc_bf16_f32(BM, 0) : idesc_f16_f32(BM, 0);
    const uint32_t id_pv = base | kMnB | (64u >> 3) << 17;
    // S(i) = q k(i)^T into buffer i & 1
    auto scores = [&](int i) {
      if (!mbar_wait(&s.k_full[i & 1], (i >> 1) & 1, 203)) return false;
      tc_fence_after();
      if (lane == 0) {
        const uint32_t id = base | (uint32_t)(up16(min(BM, b.len - i * BM)) >> 3) << 17;
        const uint32_t q = smem_u32(s.q), k = smem_u32(s.k[i & 1]);
#pragma unroll
        for (int kk = 0; kk < 4; ++kk)
          mma_f16(tmem + (i & 1) * 128, sdesc_k_sw128(q + kk * 32), sdesc_k_sw128(k + kk * 32), id, kk > 0);
        mma_commit(&s.k_empty[i & 1]);
        mma_commit(&s.s_full[i & 1]);
      }
      __syncwarp();
      return true;
    };
    bool ok = mbar_wait(&s.q_full, 0, 204) && scores(0) && (n < 2 || scores(1));
    for (int i = 0; ok && i < n; ++i) {
      const int bf = i & 1, cols = min(BM, b.len - i * BM);
      const uint32_t ph = (i >> 1) & 1;
      if (!mbar_wait(&s.v_full[bf], ph, 205)) break;
      if (cols & 15) zero_tile_rows(s.v[bf], cols, up16(cols), lane);
      if (!mbar_wait(&s.p_full[bf], ph, 206)) break;
      tc_fence_after();
      if (lane == 0) {
        const uint32_t v = smem_u32(s.v[bf]);
        for (int kk = 0; kk < up16(cols) / 16; ++kk)
          mma_f16_ts(tmem + bf * 128 + 64, tmem + bf * 128 + kk * 8, sdesc_mn_sw128(v + kk * 2048), id_pv, kk > 0);
        mma_commit(&s.v_empty[bf]);
        mma_commit(&s.o_full[bf]);
      }
      __syncwarp();
      if (i + 2 < n) ok = mbar_wait(&s.s_free[bf], ph, 207) && scores(i + 2);
    }
  } else if (warp < live) {
    const uint32_t lanes = tmem + ((uint32_t)(warp * 32) << 16);
    const float c = a.scale * kLog2e;
    float o[64], m = kNegInf, l = 0.f, fold = 1.f;
#pragma unroll
    for (int d = 0; d < 64; ++d) o[d] = 0.f;
    auto take_o = [&](int i) {  // o <- o fold + P(i) v
      if (!mbar_wait(&s.o_full[i & 1], (i >> 1) & 1, 208)) return false;
      tc_fence_after();
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t r[32];
        tmem_ld32(lanes + (i & 1) * 128 + 64 + h * 32, r);
        tmem_ld_wait();
#pragma unroll
        for (int d = 0; d < 32; ++d) o[h * 32 + d] = fmaf(o[h * 32 + d], fold, __uint_as_float(r[d]));
      }
      tc_fence_before();
      mbar_arrive(&s.s_free[i & 1]);
      return true;
    };
    bool ok = true;
    for (int i = 0; i < n; ++i) {
      const int cols = min(BM, b.len - i * BM);
      const uint32_t buf = lanes + (i & 1) * 128;
      ok = mbar_wait(&s.s_full[i & 1], (i >> 1) & 1, 209);
      if (!ok) break;
      tc_fence_after();
      float mx = kNegInf;
#pragma unroll
      for (int h = 0; h < 4; ++h)
        if (h * 32 < cols) {
          uint32_t r[32];
          tmem_ld32(buf + h * 32, r);
          tmem_ld_wait();
          if (h * 32 + 32 <= cols) {
#pragma unroll
            for (int j = 0; j < 32; ++j) mx = fmaxf(mx, __uint_as_float(r[j]));
          } else {
#pragma unroll
            for (int j = 0; j < 32; ++j) mx = fmaxf(mx, h * 32 + j < cols ? __uint_as_float(r[j]) : kNegInf);
          }
        }
      mx = fmaxf(m, mx);
      const float ref = mx == kNegInf ? 0.f : mx * c;
      const float f = m == kNegInf ? 0.f : ex2(fmaf(m, c, -ref));
      if (i > 0) {
        ok = take_o(i - 1);
        if (!ok) break;
      }
      fold = f;
      m = mx;
      float sum = 0.f;
#pragma unroll
      for (int h = 0; h < 4; ++h)
        if (h * 32 < cols) {
          uint32_t r[32], p[16];
          tmem_ld32(buf + h * 32, r);
          tmem_ld_wait();
          if (h * 32 + 32 > cols) {
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (h * 32 + j >= cols) r[j] = 0xFF800000u;  // -inf
          }
#pragma unroll
          for (int j = 0; j < 32; j += 2) {
            const float x = ex2(fmaf(__uint_as_float(r[j]), c, -ref)), y = ex2(fmaf(__uint_as_float(r[j + 1]), c, -ref));
            sum += x + y;
            p[j / 2] = pack2<DT>(x, y);
          }
          tmem_st16(buf + h * 16, p);
        }
      l = fmaf(l, f, sum);
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(&s.p_full[i & 1]);
    }
    if (ok) ok = take_o(n - 1);
    const int row = b.first + warp * 32 + lane;
    if (ok && row < b.len) {
      a.lse[(b.outer * a.H + head) * a.rows + b.row0 + row] = ((m == kNegInf ? 0.f : m * c) + log2f(l)) * kLn2;
      uint16_t* dst = reinterpret_cast<uint16_t*>(a.out) + b.outer * a.so.outer + head * a.so.head + (b.row0 + row) * a.so.row;
      store_row<DT>(dst, o, 1.f / l, a.D, vec);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 5) {
    tc_fence_after();
    tmem_dealloc(tmem, 256);
  }
}

// --------------------------------------------------------------------------------------- gradient
// One launch: CTAs with blockIdx.y < Hk own 128 keys (dk, dv; they loop over the queries of every
// query head of the key head), the others 128 queries (dq; they loop over the keys). Scores are
// computed in both, but no sum crosses CTAs. The CTA's two tiles A0, A1 (k, v or q, dout) stay in shared
// memory, tiles of 64 rows B0, B1 (q, dout or k, v) come in turn:
//   S = A0 B0^T, dP = A1 B1^T, and with P, dS written over them as 16-bit A operands
//   keys: dv += P B1, dk += dS B0;  queries: dq += dS B0.
// Warps 0-7: two threads per row, 32 columns each; warp 8: TMA, and for keys the log-sum-exp and
// delta of the 64 queries; warp 9: products and TMEM (S, dP, and two sums of 64 columns each).
constexpr int kBwdThreads = 320;
constexpr int BN = 64;
constexpr uint32_t kHalf = BN * 128;

struct BwdSmem {
  uint8_t a0[kTile], a1[kTile], b0[2][kHalf], b1[2][kHalf];
  float lse[2][BN], delta[2][BN];  // keys: per loop tile; lse in base 2
  uint64_t a_full, b_full[2], b_empty[2], s_full, p_full, acc_full;
  uint32_t tmem;
};

// dS of fp16 gradients is held in fp16, whose range ends at 6e-8: it is scaled by the power of two that
// brings the largest |dout| of its sequence and key head to 2^-4, which leaves room for |v| summed over
// the head dimension up to 2^19, and dk, dq are scaled back in fp32.
__device__ __forceinline__ float gain_of(uint32_t amax_bits) {
  const int e = (int)(amax_bits >> 23);
  return e == 0 || e >= 250 ? 1.f : __uint_as_float((uint32_t)(250 - e) << 23);
}

template <int DT>
__global__ void __launch_bounds__(kBwdThreads, 2)
attn_bwd_tc_kernel(const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mk,
                   const __grid_constant__ CUtensorMap mv, const __grid_constant__ CUtensorMap mdo, const AttnArgs a, int vec) {
  extern __shared__ uint8_t raw[];
  BwdSmem& s = *reinterpret_cast<BwdSmem*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, group = a.H / a.Hk;
  const bool keys = (int)blockIdx.y < a.Hk;
  const int head = keys ? (int)blockIdx.y : (int)blockIdx.y - a.Hk;  // the CTA's own head
  const SeqBlock b = seq_block(a, blockIdx.x);
  int64_t z0, z1;
  if (idle_rows(a, b, blockIdx.x, &z0, &z1)) {
    if (keys) {
      zero_rows16(a.dk, a.sdk, b.outer, head, z0, z1, a.D);
      zero_rows16(a.dv, a.sdv, b.outer, head, z0, z1, a.D);
    } else {
      zero_rows16(a.dq, a.sdq, b.outer, head, z0, z1, a.D);
    }
  }
  if (!b.on || b.first >= b.len) return;
  const int per = (b.len + BN - 1) / BN;       // loop tiles of one head
  const int n = keys ? per * group : per;
  const int live = min(4, (b.len - b.first + 31) / 32);  // lane quarters that have a row
  if (threadIdx.x == 0) {
    mbar_init(&s.a_full, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s.b_full[i], 33);
      mbar_init(&s.b_empty[i], 1);
    }
    mbar_init(&s.s_full, 1);
    mbar_init(&s.p_full, live * 64);
    mbar_init(&s.acc_full, 1);
    fence_barrier_init();
  }
  if (warp == 9) tmem_alloc(&s.tmem, 256);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s.tmem;
  const int64_t vec0 = b.outer * a.H * a.rows + b.row0;  // lse and delta of query head h: + h rows

  if (warp == 8) {
    const int r0 = (int)b.row0, o = (int)b.outer, kh = keys ? head : head / group;
    if (lane == 0) {
      mbar_arrive_expect_tx(&s.a_full, 2 * kTile);
      for (int half = 0; half < 2; ++half) {  // boxes of 64 rows
        tma_load_4d(s.a0 + half * kHalf, keys ? &mk : &mq, 0, r0 + b.first + half * BN, head, o, &s.a_full);
        tma_load_4d(s.a1 + half * kHalf, keys ? &mv : &mdo, 0, r0 + b.first + half * BN, head, o, &s.a_full);
      }
    }
    for (int i = 0; i < n; ++i) {
      const int st = i & 1, row = (i % per) * BN, h = keys ? head * group + i / per : kh;
      if (i >= 2 && !mbar_wait(&s.b_empty[st], ((i >> 1) & 1) ^ 1, 211)) break;
      if (lane == 0) {
        mbar_arrive_expect_tx(&s.b_full[st], 2 * kHalf);
        tma_load_4d(s.b0[st], keys ? &mq : &mk, 0, r0 + row, h, o, &s.b_full[st]);
        tma_load_4d(s.b1[st], keys ? &mdo : &mv, 0, r0 + row, h, o, &s.b_full[st]);
      }
      if (keys) {
        for (int j = lane; j < BN; j += 32) {
          const bool on = row + j < b.len;
          const int64_t at = vec0 + (int64_t)h * a.rows + row + j;
          s.lse[st][j] = on ? a.lse[at] * kLog2e : 0.f;
          s.delta[st][j] = on ? a.delta[at] : 0.f;
        }
      }
      mbar_arrive(&s.b_full[st]);
    }
  } else if (warp == 9) {
    const uint32_t base = DT == ATLAS_BF16 ? idesc_bf16_f32(BM, 0) : idesc_f16_f32(BM, 0);
    const uint32_t id_sum = base | kMnB | (64u >> 3) << 17;
    const uint32_t a0 = smem_u32(s.a0), a1 = smem_u32(s.a1);
    bool ok = mbar_wait(&s.a_full, 0, 212);
    for (int i = 0; ok && i < n; ++i) {
      const int st = i & 1, cols = min(BN, b.len - (i % per) * BN), c16 = up16(cols);
      // S(i) overwrites P(i-1) and dS(i-1): the products that read them must be done
      if (i && !mbar_wait(&s.b_empty[st ^ 1], ((i - 1) >> 1) & 1, 218)) break;
      if (!mbar_wait(&s.b_full[st], (i >> 1) & 1, 213)) break;
      if (cols & 15) {
        zero_tile_rows(s.b0[st], cols, c16, lane);
        if (keys) zero_tile_rows(s.b1[st], cols, c16, lane);
      }
      tc_fence_after();
      const uint32_t b0 = smem_u32(s.b0[st]), b1 = smem_u32(s.b1[st]);
      if (lane == 0) {
        const uint32_t id = base | (uint32_t)(c16 >> 3) << 17;
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) mma_f16(tmem, sdesc_k_sw128(a0 + kk * 32), sdesc_k_sw128(b0 + kk * 32), id, kk > 0);
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) mma_f16(tmem + 64, sdesc_k_sw128(a1 + kk * 32), sdesc_k_sw128(b1 + kk * 32), id, kk > 0);
        mma_commit(&s.s_full);
      }
      __syncwarp();
      if (!mbar_wait(&s.p_full, i & 1, 214)) break;
      tc_fence_after();
      if (lane == 0) {
        // P and dS are 16-bit over the first half of each thread's own 32 columns of S and dP: the K
        // elements 0-31 in columns 0-15, 32-63 in columns 32-47
        for (int kk = 0; kk < c16 / 16; ++kk) {
          const uint32_t col = (kk >> 1) * 32 + (kk & 1) * 8;
          if (keys) mma_f16_ts(tmem + 128, tmem + col, sdesc_mn_sw128(b1 + kk * 2048), id_sum, i > 0 || kk > 0);
          mma_f16_ts(tmem + 192, tmem + 64 + col, sdesc_mn_sw128(b0 + kk * 2048), id_sum, i > 0 || kk > 0);
        }
        mma_commit(&s.b_empty[st]);
        if (i == n - 1) mma_commit(&s.acc_full);
      }
      __syncwarp();
    }
  } else if ((warp & 3) < live) {
    const int quarter = warp & 3, half = warp >> 2;  // columns 32 half .. of every loop tile
    const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16);
    const int row = b.first + quarter * 32 + lane;
    const float c = a.scale * kLog2e;
    const float gain = DT == ATLAS_F16 ? gain_of(a.amax[(int64_t)b.seq * a.Hk + (keys ? head : head / group)]) : 1.f;
    float lse = 0.f, delta = 0.f;
    if (!keys && row < b.len) {
      lse = a.lse[vec0 + (int64_t)head * a.rows + row] * kLog2e;
      delta = a.delta[vec0 + (int64_t)head * a.rows + row];
    }
    bool ok = true;
    for (int i = 0; i < n; ++i) {
      const int st = i & 1, left = min(BN, b.len - (i % per) * BN) - half * 32;  // columns of this thread's part
      ok = mbar_wait(&s.s_full, i & 1, 215);
      if (!ok) break;
      tc_fence_after();
      if (keys) {  // written by warp 8 before b_full, which the products waited for; seen here by its own wait
        ok = mbar_wait(&s.b_full[st], (i >> 1) & 1, 216);
        if (!ok) break;
      }
      if (left > 0) {
        uint32_t x[32], y[32];
        tmem_ld32(lanes + half * 32, x);
        tmem_ld32(lanes + 64 + half * 32, y);
        tmem_ld_wait();
        uint32_t p[16], d[16];
#pragma unroll
        for (int j = 0; j < 32; j += 2) {
          float w[2], g[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float l = keys ? s.lse[st][half * 32 + j + e] : lse, dl = keys ? s.delta[st][half * 32 + j + e] : delta;
            w[e] = ex2(fmaf(__uint_as_float(x[j + e]), c, -l));
            g[e] = (DT == ATLAS_F16 ? w[e] * gain : w[e]) * (__uint_as_float(y[j + e]) - dl);
            if (j + e >= left) w[e] = g[e] = 0.f;
          }
          p[j / 2] = pack2<DT>(w[0], w[1]);
          d[j / 2] = pack2<DT>(g[0], g[1]);
        }
        if (keys) tmem_st16(lanes + half * 32, p);
        tmem_st16(lanes + 64 + half * 32, d);
        tmem_st_wait();
      }
      tc_fence_before();
      mbar_arrive(&s.p_full);
    }
    if (ok) ok = mbar_wait(&s.acc_full, 0, 217);
    tc_fence_after();
    // keys: warps 0-3 write dv, 4-7 dk; queries: warps 4-7 write dq
    if (ok && (keys || half)) {
      float acc[64];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t r[32];
        tmem_ld32(lanes + 128 + half * 64 + h * 32, r);
        tmem_ld_wait();
#pragma unroll
        for (int d = 0; d < 32; ++d) acc[h * 32 + d] = __uint_as_float(r[d]);
      }
      if (row < b.len) {
        void* out = !half ? a.dv : keys ? a.dk : a.dq;
        const Strides& so = !half ? a.sdv : keys ? a.sdk : a.sdq;
        uint16_t* dst = reinterpret_cast<uint16_t*>(out) + b.outer * so.outer + head * so.head + (b.row0 + row) * so.row;
        store_row<DT>(dst, acc, half ? a.scale / gain : 1.f, a.D, vec);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem, 256);
  }
}

// ------------------------------------------------------------------------------------------- host
// [outer, heads, rows, D] as a 4-D map of boxes of `box_rows` rows x 64 elements; columns from D on read as 0.
int make_map(CUtensorMap* map, const void* base, int dtype, const Strides& st, int64_t outer, int64_t heads, int64_t rows, int D,
             int box_rows) {
  using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                              const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
  static Encode encode = [] {
    void* fn = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      fn = nullptr;
    return reinterpret_cast<Encode>(fn);
  }();
  if (!encode) return fail(ATLAS_ERR_CUDA, "cuTensorMapEncodeTiled entry point unavailable");
  // the stride of an axis with one element is never used, but has to be a valid one
  const cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)rows, (cuuint64_t)heads, (cuuint64_t)outer};
  const cuuint64_t strides[3] = {rows > 1 ? (cuuint64_t)st.row * 2 : 128, heads > 1 ? (cuuint64_t)st.head * 2 : 128,
                                 outer > 1 ? (cuuint64_t)st.outer * 2 : 128};
  const cuuint32_t box[4] = {64, (cuuint32_t)box_rows, 1, 1}, step[4] = {1, 1, 1, 1};
  const CUresult r = encode(map, dtype == ATLAS_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
                            const_cast<void*>(base), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? ATLAS_OK : fail(ATLAS_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", (int)r);
}

bool stride_ok(int64_t s, int64_t extent) { return extent <= 1 || (s > 0 && s % 8 == 0 && s < (1LL << 38)); }
bool map_ok(const void* p, const Strides& s, int64_t outer, int64_t heads, int64_t rows) {
  return (uintptr_t)p % 16 == 0 && stride_ok(s.row, rows) && stride_ok(s.head, heads) && stride_ok(s.outer, outer);
}

template <int DT>
int fwd(const AttnArgs& a, cudaStream_t st) {
  CUtensorMap mq, mk, mv;
  if (int rc = make_map(&mq, a.q, DT, a.sq, a.outer, a.H, a.rows, a.D, BM)) return rc;
  if (int rc = make_map(&mk, a.k, DT, a.sk, a.outer, a.Hk, a.rows, a.D, BM)) return rc;
  if (int rc = make_map(&mv, a.v, DT, a.sv, a.outer, a.Hk, a.rows, a.D, BM)) return rc;
  const int bytes = sizeof(FwdSmem) + 1024;
  if (cudaFuncSetAttribute(attn_fwd_tc_kernel<DT>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess)
    return fail(ATLAS_ERR_CUDA, "attention: shared memory attribute");
  const int vec = a.D % 8 == 0 && map_ok(a.out, a.so, a.outer, a.H, a.rows);
  attn_fwd_tc_kernel<DT><<<dim3((unsigned)a.cap, a.H), kFwdThreads, bytes, st>>>(mq, mk, mv, a, vec);
  return check_launch("attention");
}

template <int DT>
int bwd(const AttnArgs& a, cudaStream_t st) {
  CUtensorMap mq, mk, mv, mdo;
  if (int rc = make_map(&mq, a.q, DT, a.sq, a.outer, a.H, a.rows, a.D, BN)) return rc;
  if (int rc = make_map(&mk, a.k, DT, a.sk, a.outer, a.Hk, a.rows, a.D, BN)) return rc;
  if (int rc = make_map(&mv, a.v, DT, a.sv, a.outer, a.Hk, a.rows, a.D, BN)) return rc;
  if (int rc = make_map(&mdo, a.dout, DT, a.sdo, a.outer, a.H, a.rows, a.D, BN)) return rc;
  const int bytes = sizeof(BwdSmem) + 1024;
  if (cudaFuncSetAttribute(attn_bwd_tc_kernel<DT>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess)
    return fail(ATLAS_ERR_CUDA, "attention_grad: shared memory attribute");
  const int vec = a.D % 8 == 0 && map_ok(a.dq, a.sdq, a.outer, a.H, a.rows) && map_ok(a.dk, a.sdk, a.outer, a.Hk, a.rows) &&
                  map_ok(a.dv, a.sdv, a.outer, a.Hk, a.rows);
  if (DT == ATLAS_F16 && cudaMemsetAsync(a.amax, 0, (size_t)(a.B * a.Hk) * 4, st) != cudaSuccess)
    return fail(ATLAS_ERR_CUDA, "attention_grad: clearing the workspace failed");
  if (int rc = attn_delta(a, DT, st)) return rc;
  attn_bwd_tc_kernel<DT><<<dim3((unsigned)a.cap, a.Hk + a.H), kBwdThreads, bytes, st>>>(mq, mk, mv, mdo, a, vec);
  return check_launch("attention_grad");
}

}  // namespace

// Whether the tensor-core kernels take these tensors: 16-bit, every stride a multiple of 16 bytes (a
// positive one: an expanded axis has none that TMA accepts), a positive scale (the row maximum is
// taken before the scale).
bool attn_tc_takes(const AttnArgs& a, int dtype, bool grad) {
  if (dtype == ATLAS_F32 || !(a.scale > 0.f)) return false;
  if (grad && (a.H + a.Hk > 65535 || !map_ok(a.dout, a.sdo, a.outer, a.H, a.rows))) return false;
  return map_ok(a.q, a.sq, a.outer, a.H, a.rows) && map_ok(a.k, a.sk, a.outer, a.Hk, a.rows) &&
         map_ok(a.v, a.sv, a.outer, a.Hk, a.rows);
}

int attn_tc(const AttnArgs& a, int dtype, bool grad, cudaStream_t st) {
  if (grad) return dtype == ATLAS_BF16 ? bwd<ATLAS_BF16>(a, st) : bwd<ATLAS_F16>(a, st);
  return dtype == ATLAS_BF16 ? fwd<ATLAS_BF16>(a, st) : fwd<ATLAS_F16>(a, st);
}

// Status word of this file's bounded waits (see atlas_device_status).
int attn_device_status(int* v, int reset) {
  if (cudaMemcpyFromSymbol(v, g_device_status, sizeof(int)) != cudaSuccess) return ATLAS_ERR_CUDA;
  const int z = 0;
  if (reset && cudaMemcpyToSymbol(g_device_status, &z, sizeof(int)) != cudaSuccess) return ATLAS_ERR_CUDA;
  return ATLAS_OK;
}

}  // namespace atlas
