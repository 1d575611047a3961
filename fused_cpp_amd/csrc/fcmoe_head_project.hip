// fcmoe_head_project.hip -- per-head products out[t, h, :] = W[h] x[t, h, :]
// around the absorbed form of latent attention: queries into the latent space
// (K = 128 -> N = 512 for the DeepSeek heads) and latent outputs back to head
// values (512 -> 128).
//
// The weights are packed once into MFMA operand order (fcmoe_pack_experts, one
// "expert" a head): a 16-channel x 32-value tile is 1 KB, lane l's 16 bytes at
// 16 l, so a wave reads one with one coalesced load straight into registers.
// x rows are read in place, 16 bytes a lane: rows of a head lie H * K apart,
// and the 64 bytes a row gives one load are half a cache line whose other half
// the next load takes. Nothing goes through LDS: each wave owns MT x 16 tokens
// and NT x 16 channels of one head for the whole of K, and the only reuse
// between waves (weights between token blocks, x between channel blocks) is
// left to the L1 and L2.
//
// out^T = W x^T: rows are channels, columns tokens, so that a lane ends with 4
// neighbouring channels of one token and stores 8 bytes.
//
// Bound: at few tokens by the weights (2 H N K bytes from HBM), at many by x
// and out (the products reach the matrix units' rate only past what the bytes
// allow: K N / (K + N) is 100 flops a byte).
#include "fcmoe_internal.h"
#include "fcmoe_latent.h"

namespace fcmoe {

namespace {

struct HeadProject {
  const uint16_t* x;
  int64_t xt, xh;
  const uint8_t* w;
  int64_t w_head;  // bytes of a packed head
  uint16_t* out;
  int64_t ot, oh;
  int64_t tokens, heads;
  int N, K, n_tiles, k_chunks, n_blocks;
  int64_t t_blocks, items;
};

constexpr int kProjWaves = 4;

template <int MT, int NT>
__global__ __launch_bounds__(kProjWaves * kWave) void head_project_kernel(const HeadProject p) {
  const int lane = (int)threadIdx.x % kWave;
  const int64_t item = (int64_t)blockIdx.x * kProjWaves + threadIdx.x / kWave;
  if (item >= p.items) return;
  // channel blocks fastest (they share x), then heads' token blocks
  const int nb = (int)(item % p.n_blocks);
  const int64_t rest = item / p.n_blocks;
  const int64_t tb = rest % p.t_blocks, h = rest / p.t_blocks;
  const int64_t t0 = tb * (16 * MT);
  const int col = lane % 16, kq = lane / 16;
  const uint16_t* xr[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    const int64_t t = t0 + 16 * m + col;
    // rows past the last token re-read it; their columns are not stored
    xr[m] = p.x + (t < p.tokens ? t : p.tokens - 1) * p.xt + h * p.xh + 8 * kq;
  }
  const uint8_t* wr[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int tile = nb * NT + n;
    wr[n] = p.w + h * p.w_head + (int64_t)(tile < p.n_tiles ? tile : p.n_tiles - 1) * p.k_chunks * 1024 + 16 * lane;
  }
  v4f acc[MT][NT];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int n = 0; n < NT; ++n) acc[m][n] = v4f{0, 0, 0, 0};
  // K is a multiple of 8: a lane's 8 values lie inside K or past it as a whole;
  // past it the packed weights are zero and x is taken as zero.
  const int full = p.K / 32;
  constexpr int AHEAD = MT * NT == 1 ? 16 : MT * NT == 4 ? 8 : 4;  // chunks whose loads are in flight together
#pragma unroll AHEAD
  for (int c = 0; c < full; ++c) {
    v8bf xf[MT], wf[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) wf[n] = *(const v8bf*)(wr[n] + (int64_t)c * 1024);
#pragma unroll
    for (int m = 0; m < MT; ++m) xf[m] = *(const v8bf*)(xr[m] + 32 * c);
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int n = 0; n < NT; ++n) acc[m][n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wf[n], xf[m], acc[m][n], 0, 0, 0);
  }
  if (full < p.k_chunks) {
    const bool in = 32 * full + 8 * kq < p.K;
    v8bf zero;
#pragma unroll
    for (int i = 0; i < 8; ++i) zero[i] = (__bf16)0.0f;
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const v8bf xf = in ? *(const v8bf*)(xr[m] + 32 * full) : zero;
#pragma unroll
      for (int n = 0; n < NT; ++n)
        acc[m][n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(*(const v8bf*)(wr[n] + (int64_t)full * 1024), xf, acc[m][n], 0, 0, 0);
    }
  }
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    const int64_t t = t0 + 16 * m + col;
    if (t >= p.tokens) continue;
    uint16_t* o = p.out + t * p.ot + h * p.oh;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int ch = (nb * NT + n) * 16 + 4 * kq;
      // N is a multiple of 8: a lane's 4 channels are all inside it or all past it
      if (ch < p.N) *(uint2*)(o + ch) = make_uint2(pack_bf16(acc[m][n][0], acc[m][n][1]), pack_bf16(acc[m][n][2], acc[m][n][3]));
    }
  }
}

template <int MT, int NT>
void head_project_launch(HeadProject p, hipStream_t stream) {
  p.n_blocks = (p.n_tiles + NT - 1) / NT;
  p.t_blocks = ceil_div(p.tokens, 16 * MT);
  p.items = p.n_blocks * p.t_blocks * p.heads;
  hipLaunchKernelGGL((head_project_kernel<MT, NT>), dim3((unsigned)ceil_div(p.items, kProjWaves)),
                     dim3(kProjWaves * kWave), 0, stream, p);
}

}  // namespace

}  // namespace fcmoe

using namespace fcmoe;

extern "C" int fcmoe_head_projection(const fcmoe_head_projection_args* a, hipStream_t stream) {
  if (!a) return fail(FCMOE_EINVAL, "head_projection: NULL args");
  if (a->tokens < 0 || a->tokens > INT32_MAX || a->heads <= 0 || a->heads > 65536 || a->n <= 0 || a->k <= 0 ||
      a->n % 8 || a->k % 8 || a->n > 65536 || a->k > 65536)
    return fail(FCMOE_EINVAL, "head_projection: n and k must be positive multiples of 8");
  if (a->tokens == 0) return FCMOE_OK;
  if (!a->x || !a->w_packed || !a->out) return fail(FCMOE_EINVAL, "head_projection: NULL pointer");
  if (a->x_token_stride % 8 || a->x_head_stride % 8 || (uintptr_t)a->x % 16 || (uintptr_t)a->w_packed % 16)
    return fail(FCMOE_EINVAL, "head_projection: x rows must start at multiples of 16 bytes");
  if (a->out_token_stride % 4 || a->out_head_stride % 4 || (uintptr_t)a->out % 8)
    return fail(FCMOE_EINVAL, "head_projection: out rows must start at multiples of 8 bytes");
  HeadProject p{};
  p.x = a->x, p.xt = a->x_token_stride, p.xh = a->x_head_stride;
  p.w = (const uint8_t*)a->w_packed, p.w_head = fcmoe_packed_expert_bytes(2, a->n, a->k, 1);
  p.out = a->out, p.ot = a->out_token_stride, p.oh = a->out_head_stride;
  p.tokens = a->tokens, p.heads = a->heads;
  p.N = (int)a->n, p.K = (int)a->k;
  p.n_tiles = (int)ceil_div(a->n, 16), p.k_chunks = (int)ceil_div(a->k, 32);
  if (ceil_div(a->tokens, 16) * a->heads * p.n_tiles > INT32_MAX)
    return fail(FCMOE_EINVAL, "head_projection: too many tokens");
  // The largest tile of tokens x channels that still gives every SIMD a wave (4 a
  // CU, 256 CUs): a smaller one reads x and the weights more often, a larger one
  // leaves too few loads in flight. Up to 16 tokens there is one tile of them, up
  // to 32 one of two, and wider ones would hold rows that are not there. 128 heads,
  // weights from memory, us for 16 x 16, 32 x 32, 32 x 64, 64 x 64, 64 x 128 (*:
  // taken): 128 -> 512 at 32 tokens 10.0, 7.2*, 7.9, 8.8, 11.1, at 64 15.7, 12.2,
  // 10.9, 10.9*, 14.2, at 300 57, 37, 31, 29, 31*, at 2047 377, 257, 208, 184, 162*;
  // 512 -> 128 at 32 11.3*, 12.6, 13.9, 18, 25, at 128 26, 15.4, 14.2*, 20, 25, at
  // 300 49, 32, 27, 27*, 25, at 512 82, 49, 40, 33, 30*. Of 787 shapes (64 to 512 values,
  // 1 to 128 heads, 1 to 4096 tokens) it takes 1.017 of the best tile's time on
  // average, 1.28 at worst; with 512 waves instead 1.057, with 2048 1.031.
  constexpr int64_t kSimds = 1024;
  const auto fills = [&](int64_t mt, int64_t nt) { return ceil_div(a->tokens, 16 * mt) * a->heads * ceil_div(p.n_tiles, nt) >= kSimds; };
  if (a->tokens > 32 && fills(4, 8))
    head_project_launch<4, 8>(p, stream);
  else if (a->tokens > 32 && fills(4, 4))
    head_project_launch<4, 4>(p, stream);
  else if (a->tokens > 32 && fills(2, 4))
    head_project_launch<2, 4>(p, stream);
  else if (a->tokens > 16 && fills(2, 2))
    head_project_launch<2, 2>(p, stream);
  else
    head_project_launch<1, 1>(p, stream);
  return check_launch("head_projection");
}
