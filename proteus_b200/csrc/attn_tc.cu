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
// from there), and one thread per row of scores needs no shuffles.
//
// Rows behind a sequence's end: their columns of S are masked, products stop at the next multiple of
// 16, and the rows up to there are set to zero in shared memory where they are summed over, since
// 0 x NaN is NaN.
//
// What is rounded to 16 bits, and why: P before it meets v or dout, and dS before it meets q, since both are operands
// of a 16-bit product (dS before it meets k is held as two such values, see the gradient below). Their sums (l, the
// outputs, dq, dk, dv), the scores, the log-sum-exp and delta are fp32. An operand that is off by up to half a step,
// 2^-8 (bf16) or 2^-11 (fp16), independently for each key, moves a result by as much of its norm as the result's own
// rounding does, so that the two together are 1.4 times the one that no kernel avoids (bf16: 2.4e-3 of the norm for
// 1.7e-3). A second product with what the rounding left over takes that away, for half as many tensor operations again
// and a second value written to TMEM; fp32 tensors keep 24 bits throughout. Exponentials are ex2 of a score in
// base 2: the factor log2 e goes into the score's scale, which rounds it once, 2^-24 of the score.
//
// Every wait is bounded (see tc.cuh); a wait that gives up records its code and the CTA leaves, behind what it
// still has under way (last_phases).
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
__device__ __forceinline__ void load_pairs(f32x2 (&v)[2], const float* p) {
  const ulonglong2 w = *reinterpret_cast<const ulonglong2*>(p);
  v[0] = w.x;
  v[1] = w.y;
}

// Moves registers between warpgroups (see the kernels' shares).
template <int N>
__device__ __forceinline__ void regs_inc() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void regs_dec() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

template <int DT>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  uint32_t r;
  if (DT == ATLAS_BF16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// Packed 16-bit elements of a row, of which `n` (or more, or none) exist, where 16-byte stores do not fit.
struct Packed16 {
  uint32_t w[8];
};
__device__ __noinline__ void store16_single(uint16_t* dst, Packed16 v, int n) {
#pragma unroll
  for (int e = 0; e < 16; ++e)
    if (e < n) dst[e] = (uint16_t)(v.w[e / 2] >> (16 * (e & 1)));
}

// Zero the rows [from, to) of a tile of 128-byte rows, by the 32 lanes of a warp, and make the tensor
// core see it.
__device__ __forceinline__ void zero_tile_rows(uint8_t* tile, int from, int to, int lane) {
  for (int i = from * 8 + lane; i < to * 8; i += 32) reinterpret_cast<uint4*>(tile)[i] = make_uint4(0, 0, 0, 0);
  fence_async_smem();
  __syncwarp();
}

// Waits, with a limit, for the phases that `n` arrivals in turn on a ring of barriers end: a CTA's memory is
// not another's before its copies have landed in it and its products have reported there.
__device__ __forceinline__ void last_phases(uint64_t* ring, int size, int n) {
#pragma unroll 1
  for (int i = 0; i < size && i < n; ++i) mbar_poll(ring + i, ((n - 1 - i) / size) & 1);
}

__device__ __forceinline__ int up16(int n) { return (n + 15) & ~15; }

// ---------------------------------------------------------------------------------------- forward
// Work items of 128 queries of a head, key tiles of 96 rows. Two CTAs per SM run items as a stream of tiles: a
// CTA that has loaded its last item takes over one that was not launched yet (cluster launch control), so that
// an item's look-up, first loads and first scores hide behind the item before.
//   warps 0-3   softmax, one thread per query
//   warps 4-7   read an item's output, divide and write it, while the softmax is at the next item
//   warp 8      TMA and items
//   warp 9      scores; TMEM: two buffers of scores (columns 0-95, 96-191), P(t) over the first half of S(t), the
//               output in 192-255, where an item's products accumulate
//   warp 10     products with v
//   warp 11     zero to rows of no sequence
// Registers are moved from the other eight warps to the softmax's: 384 x 80 = 128 (152 + 48 + 40).
//
// The reference that exponents are taken from comes from the maximum of a row's FIRST 32 scores, not a running one: any
// reference gives the same quotient. So a tile costs one pass (no maximum, no rescaling): a packed multiply-add, an
// exponential, a packed sum and half a conversion a score. The tile's sum tells when the reference was too low, or when
// there is none yet (those scores all -inf); the warp then takes the tile's maximum, rescales the output in TMEM and
// does the tile again, whose scores are still there, since P is held in registers until it is accepted. bf16 has room
// for 2^32 above those scores (attn.cuh says what that costs: here values below 2^-80 lose bits, since what falls below
// 2^-126 in the tensor cores' sums is lost). Scores of a standard deviation of 12 over 4096 keys, 190 us if they never
// pass it, take 262 with room for 2^32, 221 with 2^40, 201 with 2^48; those of 2, 190 with any.
// fp16 values end at 65504 and have steps of 2^-24 below 2^-14: P is 2^3 times the weights, so that n keys of little
// weight are off by n 2^-28 of the largest at most (n = 2^17: half a step of the output), and there is room for
// 2^13. 2^8 times would take 260 us instead of 192 at scores of a standard deviation of 3, 2^3 takes 196.
//
// The last tile of a sequence of several ends at the sequence's end and starts inside the tile before: its
// columns `lo` .. are new, the ones below count as -inf, and no row behind the end is read.
//
// Measured: 109 sequences of 271 to 302 rows, 20 heads of 64, bf16: 121 us (323 MB, 2.7 TB/s; 46 GFLOP, 380 TFLOP/s; the
// exponentials alone 39 us at 16 a clock and SM); 4 of 1 to 4096, 16 heads over 4: 193 us (107 GFLOP, 555 TFLOP/s; 8 of
// them the weights' scale);
// one of 37, 20 heads of 24: 6 us.
constexpr int kFwdThreads = 384;
constexpr int KT = 96;
constexpr int kFwdStages = 3;
constexpr uint32_t kKeyTile = KT * 128;

struct FwdItem {
  int first, len, head, n, row0, outer;  // n: key tiles; 0 ends the stream
};

struct FwdSmem {
  uint8_t q[2][kTile], k[kFwdStages][kKeyTile], v[kFwdStages][kKeyTile];
  uint4 stage[4][32 * 2];  // each writing warp: 16 columns of its 32 rows on their way out
  float2 stat[2][BM];      // sum and reference of an item's rows
  FwdItem item[2];
  uint4 answer;
  uint64_t stat_full[2], o_free, item_full[2], item_empty[2], q_full[2], k_full[kFwdStages], k_empty[kFwdStages], v_full[kFwdStages],
      v_empty[kFwdStages], s_full[2], p_full[2], o_done[2], taken, spare_full, spare_empty;
  int2 spare;  // entry and head whose rows of no sequence are next
  uint32_t tmem;
};

// Key tile i of n over `len` rows: its first row, and its columns lo .. hi - 1 that count.
__device__ __forceinline__ int key_tile(int i, int n, int len, int& lo, int& hi) {
  const int from = i == n - 1 && n > 1 ? len - KT : i * KT;
  lo = i * KT - from;
  hi = min(KT, len - from);
  return from;
}

// What P is of the weights in an item of n key tiles, and the largest sum of a tile's weights.
constexpr int kRoom = 32;
template <int DT>
__device__ __forceinline__ float fwd_scale(int n) { return DT == ATLAS_BF16 ? pow2(-kRoom - ceil_log2(n)) : 8.f; }
template <int DT>
constexpr float kLimit = DT == ATLAS_BF16 ? 0x1p32f : 65504.f / 8;

// Weights of a row's tile against `ref` (negated), times `scale` into p, their sum returned.
template <int DT>
__device__ __forceinline__ float fwd_tile(uint32_t buf, float c, float nref, float scale, int lo, int hi, uint32_t (&p)[KT / 2]) {
  const f32x2 c2 = pair(c, c), r2 = pair(nref, nref), s2 = pair(scale, scale);
  uint32_t x[2][32];
  f32x2 sum[2] = {0, 0};
  tmem_ld32(buf, x[0]);
#pragma unroll
  for (int h = 0; h < 3; ++h) {
    tmem_ld_wait();
    if (h < 2) tmem_ld32(buf + h * 32 + 32, x[(h + 1) & 1]);
    if (h * 32 >= hi || h * 32 + 32 <= lo) continue;
    uint32_t(&y)[32] = x[h & 1];
#pragma unroll
    for (int j = 0; j < 32; j += 2) {
      float a, b;
      unpair(fma2(pair(__uint_as_float(y[j]), __uint_as_float(y[j + 1])), c2, r2), a, b);
      a = ex2(a);
      b = ex2(b);
      sum[(j >> 1) & 1] = add2(sum[(j >> 1) & 1], pair(a, b));
      unpair(mul2(pair(a, b), s2), a, b);
      p[h * 16 + j / 2] = pack2<DT>(a, b);
    }
  }
  float a, b;
  unpair(add2(sum[0], sum[1]), a, b);
  return a + b;
}

// Columns outside lo .. hi - 1 of a row's tile become -inf, in TMEM.
__device__ __noinline__ void fwd_mask(uint32_t buf, int lo, int hi) {
#pragma unroll 1
  for (int h = 0; h < KT; h += 16) {
    if (h >= lo && h + 16 <= hi) continue;
    uint32_t x[16];
    tmem_ld16(buf + h, x);
    tmem_ld_wait();
#pragma unroll
    for (int j = 0; j < 16; ++j)
      if (h + j < lo || h + j >= hi) x[j] = 0xFF800000u;
    tmem_st16(buf + h, x);
  }
  tmem_st_wait();
}

// The largest of `n` (a multiple of 16) columns.
__device__ __noinline__ float fwd_max(uint32_t buf, int n) {
  float mx = kNegInf;
#pragma unroll 1
  for (int h = 0; h < n; h += 16) {
    uint32_t x[16];
    tmem_ld16(buf + h, x);
    tmem_ld_wait();
#pragma unroll
    for (int j = 0; j < 16; ++j) mx = fmaxf(mx, __uint_as_float(x[j]));
  }
  return mx;
}

template <int DT>
__global__ void __launch_bounds__(kFwdThreads, 2)
attn_fwd_tc_kernel(const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mk,
                   const __grid_constant__ CUtensorMap mv, const AttnArgs a, int vec) {
  extern __shared__ __align__(1024) uint8_t raw[];
  FwdSmem& s = *reinterpret_cast<FwdSmem*>(raw);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
#pragma unroll 1
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s.item_full[i], 1);
      mbar_init(&s.item_empty[i], 8);
      mbar_init(&s.stat_full[i], 4);
      mbar_init(&s.q_full[i], 1);
      mbar_init(&s.s_full[i], 1);
      mbar_init(&s.p_full[i], 4);
      mbar_init(&s.o_done[i], 1);
    }
#pragma unroll 1
    for (int i = 0; i < kFwdStages; ++i) {
      mbar_init(&s.k_full[i], 1);
      mbar_init(&s.k_empty[i], 1);
      mbar_init(&s.v_full[i], 1);
      mbar_init(&s.v_empty[i], 1);
    }
    mbar_init(&s.taken, 1);
    mbar_init(&s.spare_full, 1);
    mbar_init(&s.spare_empty, 1);
    mbar_init(&s.o_free, 4);
    fence_barrier_init();
  }
  if (warp == 9) tmem_alloc(&s.tmem, 256);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s.tmem;

  if (warp == 8) {
    regs_dec<40>();
    int x = blockIdx.x, head = blockIdx.y, k = 0, t = 0, z = 0, queries = 0;
    uint32_t asked = 0;
    bool more = true, ok = true, answer_due = false;
    while (ok) {
      answer_due = more;
      if (more && elect_one()) {  // the next item is on its way while this one is loaded
        mbar_arrive_expect_tx(&s.taken, 16);
        take_cta_async(&s.answer, &s.taken);
      }
      __syncwarp();
      const SeqBlock b = more ? seq_block(a, x) : SeqBlock{};
      if (more && b.spare) {
        ok = z == 0 || mbar_wait_soon(&s.spare_empty, (z - 1) & 1, 217);
        if (!ok) break;
        if (elect_one()) {
          s.spare = make_int2(x, head);
          mbar_arrive(&s.spare_full);
        }
        __syncwarp();
        ++z;
      }
      if (!more || (b.on && b.first < b.len)) {
        const int r = k & 1, n = more ? (b.len + KT - 1) / KT : 0;
        ok = k < 2 || mbar_wait(&s.item_empty[r], ((k >> 1) & 1) ^ 1, 200);
        if (!ok) break;
        if (elect_one()) {
          s.item[r] = FwdItem{b.first, b.len, head, n, (int)b.row0, (int)b.outer};
          mbar_arrive(&s.item_full[r]);
        }
        __syncwarp();
        if (!more) break;
        const int r0 = (int)b.row0, o = (int)b.outer, kh = head / (a.H / a.Hk);
        if (elect_one()) {
          mbar_arrive_expect_tx(&s.q_full[r], kTile);
          tma_load_4d(s.q[r], &mq, 0, r0 + b.first, head, o, &s.q_full[r]);
        }
        __syncwarp();
        ++queries;
#pragma unroll 1
        for (int i = 0; i < n; ++i, ++t) {
          const int st = t % kFwdStages;
          const uint32_t ph = ((t / kFwdStages) & 1) ^ 1;
          int lo, hi;
          const int row = r0 + key_tile(i, n, b.len, lo, hi);
          ok = t < kFwdStages || (mbar_wait_soon(&s.k_empty[st], ph, 201) && mbar_wait_soon(&s.v_empty[st], ph, 202));
          if (!ok) break;
          if (elect_one()) {
            mbar_arrive_expect_tx(&s.k_full[st], kKeyTile);
            tma_load_4d(s.k[st], &mk, 0, row, kh, o, &s.k_full[st]);
            mbar_arrive_expect_tx(&s.v_full[st], kKeyTile);
            tma_load_4d(s.v[st], &mv, 0, row, kh, o, &s.v_full[st]);
          }
          __syncwarp();
        }
        if (!ok) break;
        ++k;
      }
      ok = mbar_wait_soon(&s.taken, asked & 1, 199);
      if (!ok) break;
      ++asked;
      answer_due = false;
      more = taken_cta(&s.answer, x, head);
      // the answer is read before the next one may overwrite it (generic reads, asynchronous write)
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
    }
    if (z) mbar_wait_soon(&s.spare_empty, (z - 1) & 1, 217);
    __syncwarp();
    if (elect_one()) {  // the end, whatever happened
      s.spare = make_int2(-1, 0);
      mbar_arrive(&s.spare_full);
    }
    __syncwarp();
    // what this warp asked for lands before the CTA leaves; all has, unless a wait gave up
    if (answer_due) mbar_poll(&s.taken, asked & 1);
    last_phases(s.q_full, 2, queries);
    last_phases(s.k_full, kFwdStages, t);
    last_phases(s.v_full, kFwdStages, t);
  } else if (warp == 9) {
    regs_dec<40>();
    const uint32_t base = DT == ATLAS_BF16 ? idesc_bf16_f32(BM, 0) : idesc_f16_f32(BM, 0);
    const uint32_t qd = desc_lo(smem_u32(s.q[0])), kd = desc_lo(smem_u32(s.k[0]));
    bool ok = true;
    int t = 0;
#pragma unroll 1
    for (int k = 0; ok; ++k) {
      const int r = k & 1;
      if (!mbar_wait_soon(&s.item_full[r], (k >> 1) & 1, 211)) break;
      const int n = s.item[r].n, len = s.item[r].len;
      if (!n || !mbar_wait_soon(&s.q_full[r], (k >> 1) & 1, 204)) break;
#pragma unroll 1
      for (int i = 0; i < n; ++i, ++t) {  // S(t) = q k^T into buffer t & 1
        const int st = t % kFwdStages, bf = t & 1;
        ok = mbar_wait_soon(&s.k_full[st], (t / kFwdStages) & 1, 203) &&
             // it overwrites P(t-2): the product that reads it must be done
             (t < 2 || mbar_wait_soon(&s.o_done[bf], ((t >> 1) & 1) ^ 1, 207));
        if (!ok) break;
        tc_fence_after();
        int lo, hi;
        key_tile(i, n, len, lo, hi);
        const uint32_t id = base | (uint32_t)(up16(hi) >> 3) << 17;
        const uint32_t q = qd + r * (kTile >> 4), kk = kd + st * (kKeyTile >> 4), at = tmem + bf * KT;
        if (elect_one()) {
          mma_f16_lo<false>(at, q, kk, id);
          mma_f16_lo<true>(at, q + 2, kk + 2, id);
          mma_f16_lo<true>(at, q + 4, kk + 4, id);
          mma_f16_lo<true>(at, q + 6, kk + 6, id);
          mma_commit(&s.k_empty[st]);
          mma_commit(&s.s_full[bf]);
        }
        __syncwarp();
      }
    }
    last_phases(s.k_empty, kFwdStages, t);  // the products are done, and have said so
    last_phases(s.s_full, 2, t);
  } else if (warp == 10) {
    regs_dec<40>();
    const uint32_t id = (DT == ATLAS_BF16 ? idesc_bf16_f32(BM, 64) : idesc_f16_f32(BM, 64)) | kMnB;
    const uint32_t vd = desc_lo(smem_u32(s.v[0]));
    bool ok = true;
    int t = 0;
#pragma unroll 1
    for (int k = 0; ok; ++k) {
      if (!mbar_wait_soon(&s.item_full[k & 1], (k >> 1) & 1, 213)) break;
      const int n = s.item[k & 1].n, len = s.item[k & 1].len;
      // the last item's output has been read out of where this one's goes
      if (!n || (k && !mbar_wait_soon(&s.o_free, (k - 1) & 1, 214))) break;
#pragma unroll 1
      for (int i = 0; i < n; ++i, ++t) {
        const int st = t % kFwdStages, bf = t & 1;
        int lo, hi;
        key_tile(i, n, len, lo, hi);
        ok = mbar_wait_soon(&s.v_full[st], (t / kFwdStages) & 1, 205);
        if (!ok) break;
        if (hi & 15) zero_tile_rows(s.v[st], hi, up16(hi), lane);  // a sequence of one short tile: rows behind its end
        ok = mbar_wait_soon(&s.p_full[bf], (t >> 1) & 1, 206);
        if (!ok) break;
        tc_fence_after();
        const uint32_t v = vd + st * (kKeyTile >> 4), at = tmem + bf * KT;
        if (elect_one()) {
          uint32_t acc = i > 0;
#pragma unroll
          for (int kk = 0; kk < KT / 16; ++kk)
            if (kk * 16 < hi && kk * 16 + 16 > lo) {
              mma_f16_ts_lo(tmem + 192, at + kk * 8, v + kk * 128, id, acc);
              acc = 1;
            }
          mma_commit(&s.o_done[bf]);
          mma_commit(&s.v_empty[st]);
        }
        __syncwarp();
      }
    }
    last_phases(s.o_done, 2, t);
    last_phases(s.v_empty, kFwdStages, t);
  } else if (warp == 11) {
    regs_dec<40>();
    // Rows of no sequence: 6 us of 125 when the warp that loads the tiles did it in between (109 sequences of 271
    // to 302 rows in a batch of 302, 20 heads). The end is posted whatever happens there, and a wait for the next may be
    // as long as the kernel, so that its limit is a thousand others.
#pragma unroll 1
    for (int z = 0, tries = 0; tries < 1000;) {
      if (!mbar_poll(&s.spare_full, z & 1)) {
        ++tries;
        continue;
      }
      const int2 at = s.spare;
      __syncwarp();
      if (lane == 0) mbar_arrive(&s.spare_empty);
      if (at.x < 0) break;
      const int head = at.y;
      const IdleShare share = idle_share(a, at.x);
#pragma unroll 1
      for (int64_t n = 0; share.from + n < share.end; n += 32) {  // a lane looks up a row, 8 write it
        int64_t o = 0, r = 0;
        const bool on = idle_row(a, share, n, lane, &o, &r);
        if (on) a.lse[(o * a.H + head) * a.rows + r] = 0.f;
#pragma unroll 1
        for (int j = lane >> 3; j < 32; j += 4) {
          const int64_t oj = __shfl_sync(0xFFFFFFFFu, o, j), rj = __shfl_sync(0xFFFFFFFFu, r, j);
          if (__shfl_sync(0xFFFFFFFFu, (int)on, j)) zero_row(a.out, a.so, 2, oj, head, rj, a.D, lane & 7);
        }
      }
      ++z;
      tries = 0;
    }
  } else if (warp < 4) {
    regs_inc<152>();
    const uint32_t lanes = tmem + ((uint32_t)(warp * 32) << 16);
    const float c = a.scale * kLog2e;
    bool ok = true;
#pragma unroll 1
    for (int k = 0, t = 0; ok; ++k) {
      const int r = k & 1;
      ok = mbar_wait_soon(&s.item_full[r], (k >> 1) & 1, 212);
      if (!ok) break;
      const FwdItem it = s.item[r];
      if (!it.n) break;
      const bool live = it.first + warp * 32 < it.len;
      float ref = kNegInf, l = 0.f;  // ref: in base 2, -inf while there is none
      const float scale = fwd_scale<DT>(it.n);
#pragma unroll 1
      for (int i = 0; i < it.n; ++i, ++t) {
        const int bf = t & 1;
        const uint32_t buf = lanes + bf * KT;
        int lo, hi;
        key_tile(i, it.n, it.len, lo, hi);
        ok = mbar_wait_soon(&s.s_full[bf], (t >> 1) & 1, 209);
        if (!ok) break;
        tc_fence_after();
        if (live) {
          // one copy of the tile's code: instruction fetch is what many copies of it run out of first
          if (lo > 0 || hi < KT) fwd_mask(buf, lo, hi);
          if (i == 0) ref = fwd_max(buf, 32) * c;
          uint32_t p[KT / 2];
          float sum;
          for (int again = 0;; ++again) {
            sum = fwd_tile<DT>(buf, c, ref == kNegInf ? 0.f : -ref, scale, lo, hi, p);
            const bool bad = ref == kNegInf || !(sum <= kLimit<DT>);
            if (again || !__any_sync(0xFFFFFFFFu, bad)) break;
            const float mx = fwd_max(buf, KT) * c;
            const float to = bad ? fmaxf(ref, mx) : ref;
            if (i > 0) {
              const float f = ref == to || ref == kNegInf ? 1.f : ex2(ref - to);
              // the products up to here are complete, and P(t) has not been handed over
              ok = mbar_wait_soon(&s.o_done[bf ^ 1], ((t - 1) >> 1) & 1, 208);
              if (!ok) break;
              tc_fence_after();
#pragma unroll 1
              for (int h = 0; h < 64; h += 16) {
                uint32_t o[16];
                tmem_ld16(lanes + 192 + h, o);
                tmem_ld_wait();
#pragma unroll
                for (int d = 0; d < 16; ++d) o[d] = __float_as_uint(__uint_as_float(o[d]) * f);
                tmem_st16(lanes + 192 + h, o);
              }
              l *= f;
            }
            ref = to;
          }
          if (!ok) break;
          l += sum;
#pragma unroll
          for (int h = 0; h < 3; ++h)
            if (h * 32 < hi && h * 32 + 32 > lo) {
              uint32_t w[16];
#pragma unroll
              for (int j = 0; j < 16; ++j) w[j] = p[h * 16 + j];
              tmem_st16(buf + h * 16, w);
            }
          tmem_st_wait();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s.p_full[bf]);
      }
      if (!ok) break;
      s.stat[r][warp * 32 + lane] = make_float2(l, ref);
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&s.stat_full[r]);
        mbar_arrive(&s.item_empty[r]);
      }
    }
  } else {
    regs_dec<48>();
    const int quarter = warp & 3;
    const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16);
#pragma unroll 1
    for (int k = 0, t = 0;; ++k) {
      const int r = k & 1;
      if (!mbar_wait(&s.item_full[r], (k >> 1) & 1, 215)) break;
      const int n = s.item[r].n, len = s.item[r].len, row0 = s.item[r].first + quarter * 32;  // the warp's first row
      if (!n) break;
      t += n;
      // the sums; with them the scores of the last tile are done, so that its product's barrier is at its phase
      if (!mbar_wait(&s.stat_full[r], (k >> 1) & 1, 216) || !mbar_wait(&s.o_done[(t - 1) & 1], ((t - 1) >> 1) & 1, 210)) break;
      tc_fence_after();
      if (row0 < len) {
        const float2 st = s.stat[r][quarter * 32 + lane];
        const float inv = 1.f / (st.x * fwd_scale<DT>(n));
        const int head = s.item[r].head;
        const int64_t outer = s.item[r].outer, to = (int64_t)s.item[r].row0 + row0;
        uint16_t* dst = reinterpret_cast<uint16_t*>(a.out) + outer * a.so.outer + head * a.so.head + to * a.so.row;
        if (row0 + lane < len)
          a.lse[(outer * a.H + head) * a.rows + to + lane] = ((st.y == kNegInf ? 0.f : st.y) + log2f(st.x)) * kLn2;
#pragma unroll 1
        for (int h = 0; h < 4; ++h) {
          uint32_t o[16];
          Packed16 w;
          tmem_ld16(lanes + 192 + h * 16, o);
          tmem_ld_wait();
#pragma unroll
          for (int d = 0; d < 8; ++d) w.w[d] = pack2<DT>(__uint_as_float(o[2 * d]) * inv, __uint_as_float(o[2 * d + 1]) * inv);
          if (vec) {
            // through shared memory (16-byte pieces of row x swapped by x / 4, free of bank conflicts both ways), so
            // that two lanes write 32 contiguous bytes of a row and an instruction covers 16 rows and not 32
            uint4* b = s.stage[quarter];
            b[lane * 2 + ((lane >> 2) & 1)] = make_uint4(w.w[0], w.w[1], w.w[2], w.w[3]);
            b[lane * 2 + (((lane >> 2) & 1) ^ 1)] = make_uint4(w.w[4], w.w[5], w.w[6], w.w[7]);
            __syncwarp();
#pragma unroll
            for (int q = 0; q < 2; ++q) {
              const int x = q * 16 + (lane >> 1), d = (lane & 1) * 8 + h * 16;
              const uint4 y = b[x * 2 + ((lane & 1) ^ ((x >> 2) & 1))];
              if (row0 + x < len && d < a.D) *reinterpret_cast<uint4*>(dst + x * a.so.row + d) = y;
            }
            __syncwarp();
          } else if (row0 + lane < len) {
            store16_single(dst + lane * a.so.row + h * 16, w, a.D - h * 16);
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&s.o_free);
        mbar_arrive(&s.item_empty[r]);
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

// --------------------------------------------------------------------------------------- gradient
// Work items: 128 keys of a key head (dk, dv; the loop runs over the queries of every query head that
// shares it) or 128 queries of a query head (dq; the loop runs over the keys). Scores are computed in
// both, but no sum crosses items. An item's two tiles A0, A1 (k, v or q, dout) stay in shared memory,
// tiles of 64 rows B0, B1 (q, dout or k, v) come in turn:
//   S = A0 B0^T, dP = A1 B1^T, and with the 16-bit P and dS, written over them, as A operands
//   keys: dv += P B1, dk += dS B0;  queries: dq += dS B0, dS as two 16-bit values.
// Queries have no use for P: its place holds what the rounding of dS left over, and a second product adds it. dq is
// the result with the most errors otherwise (dS, delta's output, its own rounding: bf16 2.5e-3 of the norm on the batch
// of 109 sequences below; 1.8e-3 so, 1.7e-3 being its own rounding), and the queries' items then take as long as the
// keys', 15 us more of that batch's 372. The keys' would need a third place.
// One persistent CTA per SM takes items of the list (attn_delta_kernel's) from a counter and runs their tiles as
// one stream, so that an item's start (look-up, first loads) and end (reading the sums) hide behind its neighbours:
//   warps 0-11  three groups of four, each takes every third tile: one thread per row
//   warps 12-15 read an item's sums and write them out, while the groups are at the next item
//   warp 16     TMA: items, A tiles (ring of 3), B tiles with the queries' log-sum-exp and delta (ring)
//   warp 17     S; owns the TMEM
//   warp 18     dP
//   warp 19     sums (products of two small kinds cost their issuing warp 500 clocks a tile each)
// TMEM: three buffers of S and dP (columns 128 x, 128 x + 64), the sums in 384-447 (dv) and 448-511.
//
// Measured (as the forward): 336 us (115 GFLOP that the formulas need, 342 TFLOP/s) and 429 us (267 GFLOP, 622 TFLOP/s).
// A tile of 128 x 64 scores takes 1450 clocks; its products 590, its exponentials 512.
constexpr int kBwdThreads = 640;
constexpr int kGroups = 3;
constexpr int BN = 64;
constexpr uint32_t kHalf = BN * 128;
constexpr int kRing = 2;    // items in flight
constexpr int kStages = 9;  // B tiles in flight

struct BwdItem {
  int seq, first, len, head, keys, n, row0, outer;  // n: loop tiles; 0 ends the stream
  int64_t off;                                      // place of the sequence in the padded vectors
};

struct BwdSmem {
  uint8_t a0[kRing][kTile], a1[kRing][kTile], b0[kStages][kHalf], b1[kStages][kHalf];
  float a_lse[kRing][BM], a_delta[kRing][BM];      // queries: of the item's rows
  float b_lse[kStages][BN], b_delta[kStages][BN];  // keys: of the loop tile's rows
  BwdItem item[kRing];
  uint64_t item_full[kRing], item_empty[kRing], a_full[kRing], b_full[kStages], b_empty[kStages], s_full[3], p_full[3],
      x_done[3], acc_full[kRing], acc_free;
  uint32_t tmem;
};

// fp16's range: 65504 down to steps of 2^-24, full precision down to 2^-14. A probability is held times 2^15 (the
// exponent's reference is 15 lower), full down to 2^-29. dS = P (dP - delta) is held times the power of two that
// brings its bound to 2^15: with |dP| <= |dout_i| |v_j|, and delta a mean of the dP, |dS| <= 2 |dout_i| max_j |v_j|,
// full precision down to 2^-29 of the bound. The maximum over v's rows is the sequence's and key head's; |dout_i| is
// the row's own for dq, and the largest of the key head's queries for dk, whose sums mix them. dv, dk and dq are
// scaled back in fp32. (Norms of fp16 rows are 2^-24 to 2^19: the squares' product is 2^-96 to 2^76.)
__device__ __forceinline__ float dS_scale(float dout2, float v2) {
  const uint32_t u = __float_as_uint(dout2 * v2);
  const int e = (int)(u >> 23) - 127;  // the norms' product is below 2^((e + 2) / 2), rounded down
  return e <= -127 || e >= 128 ? 1.f : __uint_as_float((uint32_t)(14 - ((e + 2) >> 1) + 127) << 23);
}
constexpr float kProbScale = 1 << kProbBits;

// The scale of dS of an item's row (queries), or of all its rows (keys). Rows behind the sequence's end have some
// scale or other: the padded vectors reach 128 values further (AttnArgs), and such a row is not written.
__device__ __forceinline__ float row_scale(const AttnArgs& a, const BwdItem& it, int row) {
  const int64_t kh = (int64_t)it.seq * a.Hk + (it.keys ? it.head : it.head / (a.H / a.Hk));
  const float dout2 = it.keys ? __uint_as_float(__ldg(a.top_dout + kh)) : __ldg(a.norm2 + it.head * a.vec_ld + it.off + row);
  return dS_scale(dout2, __uint_as_float(__ldg(a.top_v + kh)));
}

__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

// What packing (lo, hi) as `packed` has rounded away, packed.
template <int DT>
__device__ __forceinline__ uint32_t rest2(float lo, float hi, uint32_t packed) {
  f32x2 had;
  if (DT == ATLAS_BF16) {
    had = pair(__uint_as_float((packed << 16) ^ 0x80000000u), __uint_as_float((packed & 0xFFFF0000u) ^ 0x80000000u));
  } else {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&packed));
    had = pair(-f.x, -f.y);
  }
  unpair(add2(pair(lo, hi), had), lo, hi);
  return pack2<DT>(lo, hi);
}

// P and dS of 16 columns of a row from their scores x and dP y, as packed pairs (queries: in P's place what the
// packing of dS has rounded away). lse and delta come
// negated, in pairs (two fp32 operations an instruction); `left` columns are before the end.
template <int DT, bool KEYS>
__device__ __forceinline__ void bwd_part(const uint32_t (&x)[16], const uint32_t (&y)[16], f32x2 c2, f32x2 gain2, f32x2 nl, f32x2 nd,
                                         const float* b_lse, const float* b_delta, int left, uint32_t to_p, uint32_t to_d) {
  uint32_t p[8], d[8];
#pragma unroll
  for (int j = 0; j < 16; j += 4) {
    f32x2 l[2] = {nl, nl}, e[2] = {nd, nd};
    if (KEYS) {
      load_pairs(l, b_lse + j);
      load_pairs(e, b_delta + j);
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int o = j + 2 * k;
      float w0, w1, g0, g1;
      unpair(fma2(pair(__uint_as_float(x[o]), __uint_as_float(x[o + 1])), c2, l[k]), w0, w1);
      w0 = ex2(w0);
      w1 = ex2(w1);
      f32x2 g = add2(pair(__uint_as_float(y[o]), __uint_as_float(y[o + 1])), e[k]);
      if (DT == ATLAS_F16) g = mul2(g, gain2);
      unpair(mul2(g, pair(w0, w1)), g0, g1);
      d[j / 2 + k] = pack2<DT>(g0, g1);
      p[j / 2 + k] = KEYS ? pack2<DT>(w0, w1) : rest2<DT>(g0, g1, d[j / 2 + k]);
    }
  }
  if (left < 16) {  // columns behind the end: whatever the scores were, nothing
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t keep = 2 * j + 1 < left ? 0xFFFFFFFFu : 2 * j < left ? 0xFFFFu : 0u;
      p[j] &= keep;
      d[j] &= keep;
    }
  }
  tmem_st8(to_p, p);
  tmem_st8(to_d, d);
}

// One row of a tile: P over the first 32 columns of its scores, dS over the first 32 of dP. The next 16
// columns are under way from TMEM while 16 are computed; what is written lies over columns already read.
template <int DT, bool KEYS>
__device__ __forceinline__ void bwd_tile(uint32_t at, float c, float gain, float nlse, float ndelta, const float* b_lse,
                                         const float* b_delta, int left) {
  const f32x2 c2 = pair(c, c), gain2 = pair(gain, gain), nl = pair(nlse, nlse), nd = pair(ndelta, ndelta);
  uint32_t x[2][16], y[2][16];
  tmem_ld16(at, x[0]);
  tmem_ld16(at + 64, y[0]);
#pragma unroll
  for (int h = 0; h < 4; ++h) {
    if (h * 16 >= left) break;
    tmem_ld_wait();
    if (h < 3) {
      tmem_ld16(at + h * 16 + 16, x[(h + 1) & 1]);
      tmem_ld16(at + 64 + h * 16 + 16, y[(h + 1) & 1]);
    }
    bwd_part<DT, KEYS>(x[h & 1], y[h & 1], c2, gain2, nl, nd, b_lse + h * 16, b_delta + h * 16, left - h * 16, at + h * 8,
                       at + 64 + h * 8);
  }
  tmem_ld_wait();
  tmem_st_wait();
}

template <int DT>
__global__ void __launch_bounds__(kBwdThreads, 1)
attn_bwd_tc_kernel(const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mk,
                   const __grid_constant__ CUtensorMap mv, const __grid_constant__ CUtensorMap mdo,
                   const __grid_constant__ AttnArgs a, int vec) {
  extern __shared__ __align__(1024) uint8_t raw[];
  BwdSmem& s = *reinterpret_cast<BwdSmem*>(raw);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, group = a.H / a.Hk;
  if (threadIdx.x == 0) {
#pragma unroll 1
    for (int i = 0; i < kRing; ++i) {
      mbar_init(&s.item_full[i], 1);
      mbar_init(&s.item_empty[i], 4 * kGroups + 7);
      mbar_init(&s.a_full[i], 1);
      mbar_init(&s.acc_full[i], 1);
    }
#pragma unroll 1
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&s.b_full[i], 1);
      mbar_init(&s.b_empty[i], 1);
    }
    for (int i = 0; i < 3; ++i) {
      mbar_init(&s.s_full[i], 2);
      mbar_init(&s.p_full[i], 4);
      mbar_init(&s.x_done[i], 1);
    }
    mbar_init(&s.acc_free, 4);
    fence_barrier_init();
  }
  if (warp == 17) tmem_alloc(&s.tmem, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s.tmem;

  if (warp == 16) {
    if (elect_one()) {
      const int blocks = (int)min((int64_t)*a.listed, attn_blocks(a.outer, a.rows, a.B)), total = blocks * (a.Hk + a.H);
      int next = (int)atomicAdd(a.counter, 1u), k = 0, t = 0, rows = 0;
      while (true) {
        BwdItem it{};
        if (next < total) {  // keys first: theirs are the longest items
          const int y = next / blocks;
          const int4 b = a.list[next - y * blocks];
          next = (int)atomicAdd(a.counter, 1u);
          it.keys = y < a.Hk;
          it.head = it.keys ? y : y - a.Hk;
          it.seq = b.x; it.first = b.y; it.len = b.z;
          it.row0 = a.packed ? b.w : 0;
          it.outer = a.packed ? 0 : b.x;
          it.off = seq_off(b.x, b.w);
          it.n = (b.z + BN - 1) / BN * (it.keys ? group : 1);
        }
        const int r = k % kRing;
        if (k >= kRing && !mbar_wait_soon(&s.item_empty[r], ((k / kRing) & 1) ^ 1, 211)) break;
        s.item[r] = it;
        mbar_arrive(&s.item_full[r]);
        if (!it.n) break;
        const bool keys = it.keys;
        const int kh = it.head / group;
        const float *lse2 = a.lse2 + it.off, *delta2 = a.delta2 + it.off;
        mbar_arrive_expect_tx(&s.a_full[r], 2 * kTile + (keys ? 0 : 2 * BM * 4));
        for (int half = 0; half < 2; ++half) {  // boxes of 64 rows
          tma_load_4d(s.a0[r] + half * kHalf, keys ? &mk : &mq, 0, it.row0 + it.first + half * BN, it.head, it.outer, &s.a_full[r]);
          tma_load_4d(s.a1[r] + half * kHalf, keys ? &mv : &mdo, 0, it.row0 + it.first + half * BN, it.head, it.outer, &s.a_full[r]);
        }
        if (!keys) {
          bulk_load(s.a_lse[r], lse2 + it.head * a.vec_ld + it.first, BM * 4, &s.a_full[r]);
          bulk_load(s.a_delta[r], delta2 + it.head * a.vec_ld + it.first, BM * 4, &s.a_full[r]);
        }
        ++rows;
        int row = 0, h = keys ? it.head * group : kh;
        bool ok = true;
#pragma unroll 1
        for (int i = 0; i < it.n; ++i, ++t) {
          const int st = t % kStages;
          ok = t < kStages || mbar_wait_soon(&s.b_empty[st], ((t / kStages) & 1) ^ 1, 212);
          if (!ok) break;
          mbar_arrive_expect_tx(&s.b_full[st], 2 * kHalf + (keys ? 2 * BN * 4 : 0));
          tma_load_4d(s.b0[st], keys ? &mq : &mk, 0, it.row0 + row, h, it.outer, &s.b_full[st]);
          tma_load_4d(s.b1[st], keys ? &mdo : &mv, 0, it.row0 + row, h, it.outer, &s.b_full[st]);
          if (keys) {
            bulk_load(s.b_lse[st], lse2 + h * a.vec_ld + row, BN * 4, &s.b_full[st]);
            bulk_load(s.b_delta[st], delta2 + h * a.vec_ld + row, BN * 4, &s.b_full[st]);
          }
          row += BN;
          if (row >= it.len) {
            row = 0;
            ++h;
          }
        }
        if (!ok) break;
        ++k;
      }
      // the copies land before the CTA leaves; all have, unless a wait gave up
      last_phases(s.a_full, kRing, rows);
      last_phases(s.b_full, kStages, t);
    }
  } else if (warp == 17 || warp == 18) {
    // Warp 17: S, warp 18: dP. While the tensor core reads its operands, everything else that touches shared
    // memory takes about 300 clocks, a wait that is over as well: one warp with both could not keep up.
    const bool dp = warp == 18;
    const uint32_t base = DT == ATLAS_BF16 ? idesc_bf16_f32(BM, 0) : idesc_f16_f32(BM, 0);
    bool ok = true;
    int t = 0;
#pragma unroll 1
    for (int k = 0; ok; ++k) {
      const int r = k % kRing;
      if (!mbar_wait_soon(&s.item_full[r], (k / kRing) & 1, 213)) break;
      const int n = s.item[r].n, len = s.item[r].len, keys = s.item[r].keys;
      if (!n || !mbar_wait_soon(&s.a_full[r], (k / kRing) & 1, 214)) break;
      const uint32_t ar = desc_lo(smem_u32(dp ? s.a1[r] : s.a0[r]));
#pragma unroll 1
      for (int i = 0, row = 0; i < n; ++i, ++t) {
        const int x = t % 3, st = t % kStages, cols = min(BN, len - row), c16 = up16(cols);
        uint8_t* tile = dp ? s.b1[st] : s.b0[st];
        ok = mbar_wait_soon(&s.b_full[st], (t / kStages) & 1, 215);
        if (!ok) break;
        // rows behind the end: summed over in dk or dq (queries of S, keys) and in dv (dout, for keys)
        if ((cols & 15) && (keys || !dp)) zero_tile_rows(tile, cols, c16, lane);
        ok = t < 3 || mbar_wait_soon(&s.x_done[x], ((t / 3) & 1) ^ 1, 216);
        if (!ok) break;
        tc_fence_after();
        const uint32_t br = desc_lo(smem_u32(tile)), at = tmem + x * 128 + (dp ? 64 : 0);
        const uint32_t id = base | (uint32_t)(c16 >> 3) << 17;
        if (elect_one()) {
          mma_f16_lo<false>(at, ar, br, id);
          mma_f16_lo<true>(at, ar + 2, br + 2, id);
          mma_f16_lo<true>(at, ar + 4, br + 4, id);
          mma_f16_lo<true>(at, ar + 6, br + 6, id);
          if (i == n - 1) mma_commit(&s.item_empty[r]);
          mma_commit(&s.s_full[x]);
        }
        __syncwarp();
        row += BN;
        if (row >= len) row = 0;
      }
    }
    last_phases(s.s_full, 3, t);  // the products are done, and have said so (with the other warp's of the same tiles)
  } else if (warp == 19) {
    const uint32_t base = DT == ATLAS_BF16 ? idesc_bf16_f32(BM, 64) : idesc_f16_f32(BM, 64), id = base | kMnB;
    bool ok = true;
    int t = 0;
#pragma unroll 1
    for (int k = 0; ok; ++k) {
      const int r = k % kRing;
      if (!mbar_wait_soon(&s.item_full[r], (k / kRing) & 1, 224)) break;
      const int n = s.item[r].n, len = s.item[r].len, keys = s.item[r].keys;
      if (!n || (k && !mbar_wait_soon(&s.acc_free, (k - 1) & 1, 217))) break;
#pragma unroll 1
      for (int i = 0, row = 0; i < n; ++i, ++t) {
        const int x = t % 3, st = t % kStages, cols = min(BN, len - row);
        ok = mbar_wait_soon(&s.p_full[x], (t / 3) & 1, 218);
        if (!ok) break;
        tc_fence_after();
        const uint32_t br0 = desc_lo(smem_u32(s.b0[st])), br1 = desc_lo(smem_u32(s.b1[st])), at = tmem + x * 128;
        if (elect_one()) {
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
            if (kk * 16 < cols) {
              if (keys) mma_f16_ts_lo(tmem + 384, at + kk * 8, br1 + kk * 128, id, i > 0 || kk > 0);
              mma_f16_ts_lo(tmem + 448, at + 64 + kk * 8, br0 + kk * 128, id, i > 0 || kk > 0);
              if (!keys) mma_f16_ts_lo(tmem + 448, at + kk * 8, br0 + kk * 128, id, 1);
            }
          if (i == n - 1) {
            mma_commit(&s.acc_full[r]);
            mma_commit(&s.item_empty[r]);
          }
          mma_commit(&s.x_done[x]);
          mma_commit(&s.b_empty[st]);
        }
        __syncwarp();
        row += BN;
        if (row >= len) row = 0;
      }
    }
    last_phases(s.x_done, 3, t);
    last_phases(s.b_empty, kStages, t);
  } else if (warp >= 4 * kGroups) {
    const int quarter = warp & 3;
    const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16);
#pragma unroll 1
    for (int k = 0;; ++k) {
      const int r = k % kRing;
      if (!mbar_wait_soon(&s.item_full[r], (k / kRing) & 1, 225)) break;
      const BwdItem& it = s.item[r];
      if (!it.n || !mbar_wait_soon(&s.acc_full[r], (k / kRing) & 1, 223)) break;
      tc_fence_after();
      const int row = it.first + quarter * 32 + lane;
      if (it.first + quarter * 32 < it.len) {
        const bool keys = it.keys;
        const float mul = DT == ATLAS_F16 ? a.scale / row_scale(a, it, row) : a.scale;
        const float mul_dv = DT == ATLAS_F16 ? 1.f / kProbScale : 1.f;
#pragma unroll 1
        for (int h = keys ? 0 : 2; h < 4; ++h) {  // dv (keys), then dk or dq, 32 columns at a time
          uint32_t v[32];
          tmem_ld32(lanes + 384 + h * 32, v);
          tmem_ld_wait();
          const float f = h < 2 ? mul_dv : mul;
          const Strides& so = h < 2 ? a.sdv : keys ? a.sdk : a.sdq;
          uint16_t* dst = reinterpret_cast<uint16_t*>(h < 2 ? a.dv : keys ? a.dk : a.dq) + it.outer * so.outer +
                          it.head * so.head + ((int64_t)it.row0 + row) * so.row;
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            Packed16 w;
            const int col = (h & 1) * 32 + e * 16;
#pragma unroll
            for (int d = 0; d < 8; ++d)
              w.w[d] = pack2<DT>(__uint_as_float(v[e * 16 + 2 * d]) * f, __uint_as_float(v[e * 16 + 2 * d + 1]) * f);
            if (row < it.len && col < a.D) {
              if (vec) {
                *reinterpret_cast<uint4*>(dst + col) = make_uint4(w.w[0], w.w[1], w.w[2], w.w[3]);
                if (col + 8 < a.D) *reinterpret_cast<uint4*>(dst + col + 8) = make_uint4(w.w[4], w.w[5], w.w[6], w.w[7]);
              } else {
                store16_single(dst + col, w, a.D - col);
              }
            }
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&s.acc_free);
        mbar_arrive(&s.item_empty[r]);
      }
    }
  } else {
    const int g = warp >> 2, quarter = warp & 3;
    const int own = quarter * 32 + lane;
    const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16);
    const float c = a.scale * kLog2e;
    bool ok = true;
#pragma unroll 1
    for (int k = 0, t = 0; ok; ++k) {
      const int r = k % kRing;
      ok = mbar_wait_soon(&s.item_full[r], (k / kRing) & 1, 219);
      if (!ok) break;
      const BwdItem it = s.item[r];
      if (!it.n) break;
      const bool live = it.first + quarter * 32 < it.len, keys = it.keys;
      float lse = 0.f, delta = 0.f, gain = 1.f;
      if (DT == ATLAS_F16) gain = row_scale(a, it, it.first + own) / kProbScale;
      if (!keys) {
        ok = mbar_wait_soon(&s.a_full[r], (k / kRing) & 1, 220);
        if (!ok) break;
        lse = s.a_lse[r][own];
        delta = s.a_delta[r][own];
      }
      int left = it.len;  // columns from here to the end of the head
#pragma unroll 1
      for (int i = 0; i < it.n; ++i, ++t, left -= BN) {
        if (left <= 0) left = it.len;
        if (t % kGroups != g) continue;
        const int x = t % 3, st = t % kStages;
        ok = mbar_wait_soon(&s.s_full[x], (t / 3) & 1, 221) && (!keys || mbar_wait_soon(&s.b_full[st], (t / kStages) & 1, 222));
        if (!ok) break;
        tc_fence_after();
        if (live) {
          const uint32_t at = lanes + x * 128;
          if (keys) bwd_tile<DT, true>(at, c, gain, 0.f, 0.f, s.b_lse[st], s.b_delta[st], left);
          else bwd_tile<DT, false>(at, c, gain, lse, delta, nullptr, nullptr, left);
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s.p_full[x]);
      }
      if (!ok) break;
      __syncwarp();
      if (lane == 0) mbar_arrive(&s.item_empty[r]);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 17) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
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
  if (int rc = make_map(&mk, a.k, DT, a.sk, a.outer, a.Hk, a.rows, a.D, KT)) return rc;
  if (int rc = make_map(&mv, a.v, DT, a.sv, a.outer, a.Hk, a.rows, a.D, KT)) return rc;
  const int bytes = sizeof(FwdSmem);
  static bool done[64] = {};
  if (int rc = attn_smem_once(attn_fwd_tc_kernel<DT>, bytes, done)) return rc;
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
  const int bytes = sizeof(BwdSmem);
  static bool done[64] = {};
  if (int rc = attn_smem_once(attn_bwd_tc_kernel<DT>, bytes, done)) return rc;
  const int vec = a.D % 8 == 0 && map_ok(a.dq, a.sdq, a.outer, a.H, a.rows) && map_ok(a.dk, a.sdk, a.outer, a.Hk, a.rows) &&
                  map_ok(a.dv, a.sdv, a.outer, a.Hk, a.rows);
  if (cudaMemsetAsync(DT == ATLAS_F16 ? a.top_dout : a.counter, 0, (size_t)(DT == ATLAS_F16 ? 2 * a.B * a.Hk + 2 : 2) * 4, st) != cudaSuccess)
    return fail(ATLAS_ERR_CUDA, "attention_grad: clearing the workspace failed");
  if (int rc = attn_delta(a, DT, st)) return rc;
  const int64_t items = a.cap * (a.Hk + a.H);
  attn_bwd_tc_kernel<DT><<<(unsigned)(items < num_sms() ? items : num_sms()), kBwdThreads, bytes, st>>>(mq, mk, mv, mdo, a, vec);
  return check_launch("attention_grad");
}

}  // namespace

// Whether the tensor-core kernels take these tensors: 16-bit, every stride a multiple of 16 bytes (a
// positive one: an expanded axis has none that TMA accepts), a positive scale (the row maximum is
// taken before the scale).
bool attn_tc_takes(const AttnArgs& a, int dtype, bool grad) {
  if (dtype == ATLAS_F32 || !(a.scale > 0.f)) return false;
  if (grad && (a.cap * (a.H + a.Hk) >= (1LL << 30) || !map_ok(a.dout, a.sdo, a.outer, a.H, a.rows))) return false;
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
