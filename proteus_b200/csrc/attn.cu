// Host entry points of attention over the valid rows of a batch (atlas_attention) and its gradient
// (atlas_attention_grad): argument checks and the choice of kernel.
#include "attn.cuh"

namespace atlas {

int attn_simt(const AttnArgs& a, int dtype, bool grad, cudaStream_t st);
bool attn_tc_takes(const AttnArgs& a, int dtype, bool grad);
int attn_tc(const AttnArgs& a, int dtype, bool grad, cudaStream_t st);

namespace {

thread_local int grad_kernels = 0;  // of this thread's last atlas_attention_grad

Strides at(const int64_t* s, int i) { return Strides{s[3 * i], s[3 * i + 1], s[3 * i + 2]}; }

int check(const AttnArgs& a, int dtype, const char* what) {
  ATLAS_REQUIRE(dtype == ATLAS_F32 || dtype == ATLAS_BF16 || dtype == ATLAS_F16, "%s: unknown dtype %d", what, dtype);
  ATLAS_REQUIRE(a.outer >= 1 && a.rows >= 1 && a.rows < (1LL << 31) - 256 && a.B >= 1 && a.B < (1LL << 30), "%s: bad shape", what);
  ATLAS_REQUIRE(a.packed ? a.outer == 1 : a.outer == a.B, "%s: outer must be %s", what, a.packed ? "1" : "the batch");
  ATLAS_REQUIRE(a.H >= 1 && a.H <= 65535 && a.Hk >= 1 && a.H % a.Hk == 0, "%s: heads must be a multiple of the key heads", what);
  ATLAS_REQUIRE(a.D >= 1 && a.D <= kAttnMaxDim, "%s: head dimension must be in [1, %d]", what, kAttnMaxDim);
  ATLAS_REQUIRE(a.cap >= attn_blocks(a.outer, a.rows, a.B) && a.cap <= (1LL << 29),
                "%s: the block table has too few or too many entries", what);
  ATLAS_REQUIRE(a.q && a.k && a.v && a.lse && a.cu && a.blocks && a.counts, "%s: null pointer", what);
  ATLAS_REQUIRE((uintptr_t)a.blocks % 8 == 0, "%s: the block table must be 8-byte aligned", what);
  return ATLAS_OK;
}

}  // namespace
}  // namespace atlas

using namespace atlas;

extern "C" int atlas_attention(const void* q, const void* k, const void* v, int dtype, const int64_t* strides_host,
                               int64_t outer, int64_t rows, int64_t H, int64_t Hk, int64_t D, const int32_t* cu,
                               const int32_t* blocks, const int64_t* counts, int64_t B, int64_t cap, int packed,
                               double scale, void* out, float* lse, void* stream) {
  ATLAS_REQUIRE(strides_host, "attention: null pointer");
  AttnArgs a{};
  a.q = q; a.k = k; a.v = v; a.out = out; a.lse = lse;
  a.sq = at(strides_host, 0); a.sk = at(strides_host, 1); a.sv = at(strides_host, 2); a.so = at(strides_host, 3);
  a.cu = cu; a.blocks = blocks; a.counts = counts;
  a.outer = outer; a.rows = rows; a.B = B; a.cap = cap;
  a.H = H < 1 || H > 65535 ? 0 : (int)H; a.Hk = Hk < 1 || Hk > 65535 ? 0 : (int)Hk; a.D = D < 1 || D > kAttnMaxDim ? 0 : (int)D;
  a.packed = packed; a.scale = (float)scale;
  if (int rc = check(a, dtype, "attention")) return rc;
  ATLAS_REQUIRE(out, "attention: null pointer");
  return (attn_tc_takes(a, dtype, false) ? attn_tc : attn_simt)(a, dtype, false, (cudaStream_t)stream);
}

extern "C" int atlas_attention_grad_kernels(void) { return grad_kernels; }

extern "C" int64_t atlas_attention_grad_ws_bytes(int64_t outer, int64_t rows, int64_t H, int64_t Hk, int64_t B) {
  return 16 * attn_blocks(outer, rows, B) + 4 * (3 * H * attn_vec_ld(outer, rows, B) + 2 * B * Hk + 2);
}

extern "C" int atlas_attention_grad(const void* dout, const void* q, const void* k, const void* v, const void* out,
                                    const float* lse, int dtype, const int64_t* strides_host, int64_t outer, int64_t rows,
                                    int64_t H, int64_t Hk, int64_t D, const int32_t* cu, const int32_t* blocks,
                                    const int64_t* counts, int64_t B, int64_t cap, int packed, double scale, void* dq,
                                    void* dk, void* dv, void* ws, int64_t ws_bytes, void* stream) {
  ATLAS_REQUIRE(strides_host, "attention_grad: null pointer");
  AttnArgs a{};
  a.dout = dout; a.q = q; a.k = k; a.v = v; a.o = out; a.lse = const_cast<float*>(lse);
  a.dq = dq; a.dk = dk; a.dv = dv;
  a.sdo = at(strides_host, 0); a.sq = at(strides_host, 1); a.sk = at(strides_host, 2); a.sv = at(strides_host, 3);
  a.so = at(strides_host, 4); a.sdq = at(strides_host, 5); a.sdk = at(strides_host, 6); a.sdv = at(strides_host, 7);
  a.cu = cu; a.blocks = blocks; a.counts = counts;
  a.outer = outer; a.rows = rows; a.B = B; a.cap = cap;
  a.H = H < 1 || H > 65535 ? 0 : (int)H; a.Hk = Hk < 1 || Hk > 65535 ? 0 : (int)Hk; a.D = D < 1 || D > kAttnMaxDim ? 0 : (int)D;
  a.packed = packed; a.scale = (float)scale;
  if (int rc = check(a, dtype, "attention_grad")) return rc;
  ATLAS_REQUIRE(dout && out && dq && dk && dv && ws, "attention_grad: null pointer");
  ATLAS_REQUIRE(ws_bytes >= atlas_attention_grad_ws_bytes(outer, rows, H, Hk, B) && (uintptr_t)ws % 16 == 0,
                "attention_grad: workspace too small, or not 16-byte aligned");
  const bool tc = attn_tc_takes(a, dtype, true);
  grad_kernels = tc ? 2 : 3;  // delta, then one kernel, or on CUDA cores one for the keys and one for the queries
  if (!tc) {
    a.delta = (float*)ws;
    return attn_simt(a, dtype, true, (cudaStream_t)stream);
  }
  a.vec_ld = attn_vec_ld(outer, rows, B);
  a.list = (int4*)ws;
  a.lse2 = (float*)(a.list + attn_blocks(outer, rows, B));
  a.delta2 = a.lse2 + H * a.vec_ld;
  a.norm2 = a.delta2 + H * a.vec_ld;
  a.top_dout = (uint32_t*)(a.norm2 + H * a.vec_ld);
  a.top_v = a.top_dout + B * Hk;
  a.counter = a.top_v + B * Hk;
  a.listed = a.counter + 1;
  return attn_tc(a, dtype, true, (cudaStream_t)stream);
}
