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

// ------------------------------------------------------------------------------------------- host
// [outer, heads, rows, D] as a 4-D map of boxes of 128 rows x 64 elements; columns from D on read as 0.
int make_map(CUtensorMap* map, const void* base, int dtype, const Strides& st, int64_t outer, int64_t heads, int64_t rows, int D) {
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
  const cuuint32_t box[4] = {64, BM, 1, 1}, step[4] = {1, 1, 1, 1};
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
  if (int rc = make_map(&mq, a.q, DT, a.sq, a.outer, a.H, a.rows, a.D)) return rc;
  if (int rc = make_map(&mk, a.k, DT, a.sk, a.outer, a.Hk, a.rows, a.D)) return rc;
  if (int rc = make_map(&mv, a.v, DT, a.sv, a.outer, a.Hk, a.rows, a.D)) return rc;
  const int bytes = sizeof(FwdSmem) + 1024;
  if (cudaFuncSetAttribute(attn_fwd_tc_kernel<DT>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess)
    return fail(ATLAS_ERR_CUDA, "attention: shared memory attribute");
  const int vec = a.D % 8 == 0 && map_ok(a.out, a.so, a.outer, a.H, a.rows);
  attn_fwd_tc_kernel<DT><<<dim3((unsigned)a.cap, a.H), kFwdThreads, bytes, st>>>(mq, mk, mv, a, vec);
  return check_launch("attention");
}

}  // namespace

// Whether the tensor-core kernels take these tensors: 16-bit, every stride a multiple of 16 bytes (a
// positive one: an expanded axis has none that TMA accepts), a positive scale (the row maximum is
// taken before the scale).
bool attn_tc_takes(const AttnArgs& a, int dtype, bool grad) {
  if (dtype == ATLAS_F32 || !(a.scale > 0.f) || grad) return false;
  return map_ok(a.q, a.sq, a.outer, a.H, a.rows) && map_ok(a.k, a.sk, a.outer, a.Hk, a.rows) &&
         map_ok(a.v, a.sv, a.outer, a.Hk, a.rows);
}

int attn_tc(const AttnArgs& a, int dtype, bool grad, cudaStream_t st) {
  (void)grad;
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
