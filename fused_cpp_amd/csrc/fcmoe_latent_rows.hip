// fcmoe_latent_rows.hip -- the row operators around latent attention: per-head
// RMS norm with the position rotation, and the append of latent rows to a
// paged cache.
//
// Both are one pass over rows of bf16: a row (one token's head, or one token's
// latent row) lies in the registers of LPR lanes, 8 values (16 bytes) a lane
// and chunk, so that the sum of squares, the row maximum of an 8-bit cache and
// the rotation's partner values need no second read of it.
//
//   norm:      y_d = x_d * rsqrt(sum_d x_d^2 / D + eps) * w_d
//   rotation:  (a, b) -> (a cos - b sin, b cos + a sin), the pair's angle from
//              the table row of the token's position; the inverse turns by
//              -angle. Pairs are neighbours (interleaved) or P/2 apart.
//
// Sums, norms and rotations are binary32; the result is rounded once, to bf16
// (nearest even) or e4m3 (nearest even, values past 448 to 448).
#include "fcmoe_device.h"
#include "fcmoe_internal.h"
#include "fcmoe_latent.h"

namespace fcmoe {

namespace {

constexpr int kRowThreads = 256;

__device__ __forceinline__ int64_t index_at(const void* p, int is_i64, int64_t i) {
  return is_i64 ? ((const int64_t*)p)[i] : (int64_t)((const int32_t*)p)[i];
}

__device__ __forceinline__ void unpack8(const uint4& u, float* v) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __uint_as_float(w[i] << 16);
    v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}

__device__ __forceinline__ uint4 pack8(const float* v) {
  return make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7]));
}

// Rotates the 8 values v of rotary chunk rc (values 8 rc .. 8 rc + 7 of the
// rotated part); `pv` are the partner chunk's values when pairs lie P/2 apart.
// row: the position's table row, cos [P/2] then sin [P/2]; nullptr: the
// position lies outside the table, and the values become NaN rather than
// turned by some other position's angle.
__device__ __forceinline__ void rotate8(float* v, const float* pv, int rc, int P, const float* row, bool interleaved,
                                        float sign) {
  const float nan = __uint_as_float(0x7fc00000u);
  if (interleaved) {
    float c[4] = {nan, nan, nan, nan}, s[4] = {nan, nan, nan, nan};
    if (row) {
      const float4 cc = *(const float4*)(row + 4 * rc), ss = *(const float4*)(row + P / 2 + 4 * rc);
      c[0] = cc.x, c[1] = cc.y, c[2] = cc.z, c[3] = cc.w;
      s[0] = ss.x, s[1] = ss.y, s[2] = ss.z, s[3] = ss.w;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float a = v[2 * i], b = v[2 * i + 1], sn = sign * s[i];
      v[2 * i] = a * c[i] - b * sn;
      v[2 * i + 1] = b * c[i] + a * sn;
    }
  } else {
    const bool hi = rc >= P / 16;
    const int at = 8 * (hi ? rc - P / 16 : rc);
    const float turn = hi ? sign : -sign;  // b cos + a sin, a cos - b sin
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float c = row ? row[at + i] : nan, s = row ? row[P / 2 + at + i] : nan;
      v[i] = v[i] * c + pv[i] * (turn * s);
    }
  }
}

struct NormRope {
  const uint16_t* x;
  uint16_t* out;
  int64_t xt, xh, ot, oh;  // token and head strides, in elements
  int64_t rows;            // tokens * heads
  int heads, D, P;
  const void* positions;
  int pos_i64;
  const float* table;
  int64_t table_rows;
  const uint16_t* weight;
  int normalize, inverse, interleaved;
  float eps;
};

// LPR lanes hold one row, CPL chunks of 8 values each. A workgroup takes
// 256 / LPR rows at a time and RPT such groups, all of whose loads are issued
// before the first is used (a row is a short dependent chain: load, reduce,
// store).
template <int LPR, int CPL, int RPT>
__global__ __launch_bounds__(kRowThreads) void norm_rope_kernel(const NormRope p) {
  constexpr int RPG = kRowThreads / LPR;  // rows of a group
  const int sub = (int)threadIdx.x % LPR;
  const int64_t row0 = (int64_t)blockIdx.x * (RPG * RPT) + threadIdx.x / LPR;
  const int chunks = p.D / 8, first_rot = (p.D - p.P) / 8, half = p.P / 16;
  uint4 raw[RPT][CPL], partner[RPT][CPL];
  int64_t token[RPT], pos[RPT];
  const uint16_t* src[RPT];
#pragma unroll
  for (int r = 0; r < RPT; ++r) {
    const int64_t row = row0 + r * RPG;
    token[r] = row < p.rows ? row / p.heads : 0;
    const int64_t head = row < p.rows ? row - token[r] * p.heads : 0;
    src[r] = p.x + token[r] * p.xt + head * p.xh;
    pos[r] = index_at(p.positions, p.pos_i64, token[r]);
#pragma unroll
    for (int k = 0; k < CPL; ++k) {
      const int c = sub + k * LPR;
      raw[r][k] = c < chunks ? *(const uint4*)(src[r] + 8 * c) : make_uint4(0, 0, 0, 0);
      partner[r][k] = make_uint4(0, 0, 0, 0);
      if (!p.interleaved && c >= first_rot && c < chunks) {
        const int rc = c - first_rot;
        partner[r][k] = *(const uint4*)(src[r] + 8 * (first_rot + (rc < half ? rc + half : rc - half)));
      }
    }
  }
#pragma unroll
  for (int r = 0; r < RPT; ++r) {
    const int64_t row = row0 + r * RPG;
    float inv = 1.0f;
    float v[CPL][8];
#pragma unroll
    for (int k = 0; k < CPL; ++k) unpack8(raw[r][k], v[k]);
    if (p.normalize) {
      float s = 0.0f;
#pragma unroll
      for (int k = 0; k < CPL; ++k)
#pragma unroll
        for (int i = 0; i < 8; ++i) s = __builtin_fmaf(v[k][i], v[k][i], s);
#pragma unroll
      for (int o = LPR / 2; o > 0; o >>= 1) s += __shfl_xor(s, o);
      inv = 1.0f / sqrtf(s / (float)p.D + p.eps);
    }
    if (row >= p.rows) continue;
    const float* trow = (uint64_t)pos[r] < (uint64_t)p.table_rows ? p.table + pos[r] * p.P : nullptr;
    uint16_t* dst = p.out + token[r] * p.ot + (row - token[r] * p.heads) * p.oh;
#pragma unroll
    for (int k = 0; k < CPL; ++k) {
      const int c = sub + k * LPR;
      if (c >= chunks) continue;
      const bool rot = c >= first_rot;
      const int rc = c - first_rot;
      float pv[8];
      unpack8(partner[r][k], pv);
      if (p.normalize) {
        float w[8] = {1, 1, 1, 1, 1, 1, 1, 1}, pw[8] = {1, 1, 1, 1, 1, 1, 1, 1};
        if (p.weight) {
          unpack8(*(const uint4*)(p.weight + 8 * c), w);
          if (rot && !p.interleaved)
            unpack8(*(const uint4*)(p.weight + 8 * (first_rot + (rc < half ? rc + half : rc - half))), pw);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          v[k][i] = v[k][i] * inv * w[i];
          pv[i] = pv[i] * inv * pw[i];
        }
      }
      if (rot) rotate8(v[k], pv, rc, p.P, trow, p.interleaved != 0, p.inverse ? -1.0f : 1.0f);
      *(uint4*)(dst + 8 * c) = pack8(v[k]);
    }
  }
}

// Rows of any width and alignment: one wave a row, one value a lane at a time.
// Both values of a pair belong to one lane, so a call in place reads a value
// before the lane that owns it writes it. Bound by loads of 2 bytes a lane, of
// each value twice: 4096 rows of 1536 values take 26 us, where a copy of them
// takes 5.
__global__ __launch_bounds__(kRowThreads) void norm_rope_any_kernel(const NormRope p) {
  const int lane = (int)threadIdx.x % kWave;
  const int64_t row = (int64_t)blockIdx.x * (kRowThreads / kWave) + threadIdx.x / kWave;
  if (row >= p.rows) return;
  const int64_t token = row / p.heads, head = row - token * p.heads;
  const uint16_t* src = p.x + token * p.xt + head * p.xh;
  uint16_t* dst = p.out + token * p.ot + head * p.oh;
  float inv = 1.0f;
  if (p.normalize) {
    float s = 0.0f;
    for (int d = lane; d < p.D; d += kWave) {
      const float v = bf16_to_f32(src[d]);
      s = __builtin_fmaf(v, v, s);
    }
    s = wave_sum(s);
    inv = 1.0f / sqrtf(s / (float)p.D + p.eps);
  }
  auto at = [&](int d) {
    const float v = bf16_to_f32(src[d]);
    return p.normalize ? v * inv * (p.weight ? bf16_to_f32(p.weight[d]) : 1.0f) : v;
  };
  const int keep = p.D - p.P;
  for (int d = lane; d < keep; d += kWave) dst[d] = round_bf16(at(d));
  const int64_t pos = index_at(p.positions, p.pos_i64, token);
  const float* trow = (uint64_t)pos < (uint64_t)p.table_rows ? p.table + pos * p.P : nullptr;
  for (int i = lane; i < p.P / 2; i += kWave) {
    const int da = keep + (p.interleaved ? 2 * i : i), db = p.interleaved ? da + 1 : da + p.P / 2;
    const float a = at(da), b = at(db);
    const float c = trow ? trow[i] : __uint_as_float(0x7fc00000u);
    const float s = trow ? (p.inverse ? -trow[p.P / 2 + i] : trow[p.P / 2 + i]) : __uint_as_float(0x7fc00000u);
    dst[da] = round_bf16(a * c - b * s);
    dst[db] = round_bf16(b * c + a * s);
  }
}

template <int LPR, int CPL>
void norm_rope_launch(const NormRope& p, hipStream_t stream) {
  constexpr int RPG = kRowThreads / LPR;
  // Two row groups in flight once the workgroups go round many times; below
  // that one group each spreads the rows further. One and two, us: rows of 512
  // 8192 groups 18.0, 18.9, 16384 33.5, 34.9, 32768 62.8, 61.0, 65536 122.8,
  // 117.8; of 192 16384 31.4, 32.2, 32768 61.2, 59.1; of 1024 32768 95.4, 95.3.
  if (p.rows >= (int64_t)RPG * 32768) {
    hipLaunchKernelGGL((norm_rope_kernel<LPR, CPL, 2>), dim3((unsigned)ceil_div(p.rows, RPG * 2)), dim3(kRowThreads),
                       0, stream, p);
  } else {
    hipLaunchKernelGGL((norm_rope_kernel<LPR, CPL, 1>), dim3((unsigned)ceil_div(p.rows, RPG)), dim3(kRowThreads), 0,
                       stream, p);
  }
}

struct Append {
  const uint16_t* kv;  // [tokens, W] rows of stride ldkv
  int64_t ldkv, tokens;
  const void* positions;
  const void* slots;
  int pos_i64, slot_i64;
  const float* table;
  int64_t table_rows;
  int rot;  // rotated values at the row's end
  const uint16_t* weight;
  float eps;
  int interleaved;
  uint16_t* rows_out;  // [tokens, W] or nullptr
  fcmoe_latent_cache c;
};

// One wave a token: chunk c of the row (values 8 c .. 8 c + 7) lies in lane
// c % 64, register c / 64. The rotated chunks never straddle the two registers
// (R is a multiple of 512 where the rotated part follows it at chunk 64, and
// smaller rows fill one register), so a partner chunk is one lane exchange.
template <int R, int P, bool E4M3>
__global__ __launch_bounds__(kRowThreads) void append_kernel(const Append p) {
  constexpr int W = R + P, CH = W / 8, CPL = (CH + kWave - 1) / kWave;
  const int lane = (int)threadIdx.x % kWave;
  const int64_t t = (int64_t)blockIdx.x * (kRowThreads / kWave) + threadIdx.x / kWave;
  if (t >= p.tokens) return;
  const int64_t slot = index_at(p.slots, p.slot_i64, t);
  const bool store = (uint64_t)slot < (uint64_t)(p.c.pages * p.c.page_size);
  if (!store && !p.rows_out) return;
  const int64_t pos = index_at(p.positions, p.pos_i64, t);
  const float* trow = (uint64_t)pos < (uint64_t)p.table_rows ? p.table + pos * p.rot : nullptr;
  const uint16_t* src = p.kv + t * p.ldkv;
  float v[CPL][8];
  float s = 0.0f;
#pragma unroll
  for (int k = 0; k < CPL; ++k) {
    const int c = lane + k * kWave;
    unpack8(c < CH ? *(const uint4*)(src + 8 * c) : make_uint4(0, 0, 0, 0), v[k]);
    if (c < R / 8) {
#pragma unroll
      for (int i = 0; i < 8; ++i) s = __builtin_fmaf(v[k][i], v[k][i], s);
    }
  }
  s = wave_sum(s);
  const float inv = 1.0f / sqrtf(s / (float)R + p.eps);
  const int first_rot = (W - p.rot) / 8, half = p.rot / 16;
  float top = 0.0f;
#pragma unroll
  for (int k = 0; k < CPL; ++k) {
    const int c = lane + k * kWave;
    if (c < R / 8) {
      float w[8] = {1, 1, 1, 1, 1, 1, 1, 1};
      if (p.weight) unpack8(*(const uint4*)(p.weight + 8 * c), w);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[k][i] = v[k][i] * inv * w[i];
    }
    const bool rot = c >= first_rot && c < CH;
    const int rc = c - first_rot;
    float pv[8];
    if (!p.interleaved) {
      const int from = (rc < half ? c + half : c - half) % kWave;
#pragma unroll
      for (int i = 0; i < 8; ++i) pv[i] = __shfl(v[k][i], rot ? from : lane);
    }
    if (rot) rotate8(v[k], pv, rc, p.rot, trow, p.interleaved != 0, 1.0f);
    if (c < CH) {
      if (p.rows_out) *(uint4*)(p.rows_out + t * W + 8 * c) = pack8(v[k]);
#pragma unroll
      for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(v[k][i]));
    }
  }
  if (!store) return;
  const int64_t page = slot / p.c.page_size, in = slot - page * p.c.page_size;
  if constexpr (E4M3) {
    top = wave_max(top);
    // max / 448 is 0 for a zero row and for one of values too small for a scale of their own, which become zeros
    const float largest = top / kE4M3Max, scale = largest > 0.0f ? largest : 1.0f;
    if (lane == 0) p.c.scale[page * p.c.scale_page_stride + in] = scale;
#pragma unroll
    for (int k = 0; k < CPL; ++k) {
      const int c = lane + k * kWave;
      if (c >= CH) continue;
      float q[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float d = v[k][i] / scale;
        q[i] = d > kE4M3Max ? kE4M3Max : d < -kE4M3Max ? -kE4M3Max : d;  // a NaN stays one
      }
      const uint2 u = make_uint2(pack_e4m3(q[0], q[1], q[2], q[3]), pack_e4m3(q[4], q[5], q[6], q[7]));
      if (c < R / 8)
        *(uint2*)((uint8_t*)p.c.latent + page * p.c.latent_page_stride + in * p.c.latent_row_stride + 8 * c) = u;
      else
        *(uint2*)((uint8_t*)p.c.rope + page * p.c.rope_page_stride + in * p.c.rope_row_stride + 8 * c - R) = u;
    }
  } else {
#pragma unroll
    for (int k = 0; k < CPL; ++k) {
      const int c = lane + k * kWave;
      if (c >= CH) continue;
      const uint4 u = pack8(v[k]);
      if (c < R / 8)
        *(uint4*)((uint16_t*)p.c.latent + page * p.c.latent_page_stride + in * p.c.latent_row_stride + 8 * c) = u;
      else
        *(uint4*)((uint16_t*)p.c.rope + page * p.c.rope_page_stride + in * p.c.rope_row_stride + 8 * c - R) = u;
    }
  }
}

template <int R, int P>
void append_launch(const Append& a, hipStream_t stream) {
  const dim3 g((unsigned)ceil_div(a.tokens, kRowThreads / kWave)), b(kRowThreads);
  if (a.c.e4m3)
    hipLaunchKernelGGL((append_kernel<R, P, true>), g, b, 0, stream, a);
  else
    hipLaunchKernelGGL((append_kernel<R, P, false>), g, b, 0, stream, a);
}

}  // namespace

// A cache the kernels can read: dims they are compiled for, rows of whole
// 16-byte pieces (both the attention's loads and the append's stores are).
int check_latent_cache(const fcmoe_latent_cache& c, const char* what) {
  const std::string w(what);
  if ((c.latent_dim != 512 && c.latent_dim != 256) || (c.rope_dim != 64 && c.rope_dim != 0))
    return fail(FCMOE_EINVAL, w + ": latent_dim must be 256 or 512 and rope_dim 0 or 64");
  if (c.pages < 0 || c.page_size <= 0 || c.page_size > (1 << 20) || c.pages > INT32_MAX)
    return fail(FCMOE_EINVAL, w + ": bad page count or page size");
  if (c.pages > 0 && (!c.latent || (c.rope_dim && !c.rope) || (c.e4m3 && !c.scale)))
    return fail(FCMOE_EINVAL, w + ": NULL cache pointer");
  const int64_t unit = c.e4m3 ? 16 : 8;  // elements of 16 bytes
  if (c.latent_page_stride % unit || c.latent_row_stride % unit || (uintptr_t)c.latent % 16 || c.latent_row_stride < 0 ||
      c.latent_page_stride < 0)
    return fail(FCMOE_EINVAL, w + ": cache rows must start at multiples of 16 bytes");
  if (c.rope_dim && (c.rope_page_stride % unit || c.rope_row_stride % unit || (uintptr_t)c.rope % 16 ||
                     c.rope_row_stride < 0 || c.rope_page_stride < 0))
    return fail(FCMOE_EINVAL, w + ": cache rows must start at multiples of 16 bytes");
  return FCMOE_OK;
}

}  // namespace fcmoe

using namespace fcmoe;

extern "C" int fcmoe_head_norm_rope(const fcmoe_head_norm_rope_args* a, hipStream_t stream) {
  if (!a) return fail(FCMOE_EINVAL, "head_norm_rope: NULL args");
  if (a->tokens < 0 || a->heads <= 0 || a->dim <= 0 || a->dim > 65536 || a->heads > 65536)
    return fail(FCMOE_EINVAL, "head_norm_rope: bad shape");
  if (a->rope_dim < 0 || a->rope_dim % 2 || a->rope_dim > a->dim)
    return fail(FCMOE_EINVAL, "head_norm_rope: rope_dim must be even and at most dim");
  if (a->weight && !a->normalize) return fail(FCMOE_EINVAL, "head_norm_rope: a weight needs normalize");
  if (a->tokens == 0) return FCMOE_OK;
  if (!a->x || !a->out || !a->positions || (a->rope_dim && !a->cos_sin) || a->table_rows < 0)
    return fail(FCMOE_EINVAL, "head_norm_rope: NULL pointer");
  NormRope p{};
  p.x = a->x, p.out = a->out;
  p.xt = a->x_token_stride, p.xh = a->x_head_stride, p.ot = a->out_token_stride, p.oh = a->out_head_stride;
  if (a->tokens > INT32_MAX || a->tokens * a->heads / 4 > INT32_MAX) return fail(FCMOE_EINVAL, "head_norm_rope: too many rows");
  p.rows = a->tokens * a->heads;
  p.heads = (int)a->heads, p.D = (int)a->dim, p.P = (int)a->rope_dim;
  p.positions = a->positions, p.pos_i64 = a->positions_i64;
  p.table = a->cos_sin, p.table_rows = a->table_rows;
  p.weight = a->weight, p.normalize = a->normalize, p.inverse = a->inverse, p.interleaved = a->interleaved;
  p.eps = a->eps;
  // Rows of whole 16-byte pieces, pairs that stay within pieces (interleaved)
  // or pair whole pieces (half apart).
  const bool wide = p.D % 8 == 0 && p.D <= 1024 && p.P % (p.interleaved ? 8 : 16) == 0 && p.xt % 8 == 0 &&
                    p.xh % 8 == 0 && p.ot % 8 == 0 && p.oh % 8 == 0 && (uintptr_t)p.x % 16 == 0 &&
                    (uintptr_t)p.out % 16 == 0 && (uintptr_t)p.weight % 16 == 0 && (uintptr_t)p.table % 16 == 0 &&
                    (p.interleaved == 0 || p.P / 2 % 4 == 0);
  if (!wide) {
    hipLaunchKernelGGL(norm_rope_any_kernel, dim3((unsigned)ceil_div(p.rows, kRowThreads / kWave)), dim3(kRowThreads),
                       0, stream, p);
    return check_launch("head_norm_rope");
  }
  const int chunks = p.D / 8;
  if (chunks <= 8)
    norm_rope_launch<8, 1>(p, stream);
  else if (chunks <= 16)
    norm_rope_launch<16, 1>(p, stream);
  else if (chunks <= 32)
    norm_rope_launch<32, 1>(p, stream);
  else if (chunks <= 64)
    norm_rope_launch<64, 1>(p, stream);
  else
    norm_rope_launch<64, 2>(p, stream);
  return check_launch("head_norm_rope");
}

extern "C" int fcmoe_latent_cache_append(const fcmoe_latent_append_args* a, hipStream_t stream) {
  if (!a) return fail(FCMOE_EINVAL, "latent_cache_append: NULL args");
  if (const int rc = check_latent_cache(a->cache, "latent_cache_append")) return rc;
  const int64_t W = a->cache.latent_dim + a->cache.rope_dim;
  if (a->tokens < 0 || a->tokens > INT32_MAX || a->kv_row_stride % 8 || a->kv_row_stride < 0)
    return fail(FCMOE_EINVAL, "latent_cache_append: bad token count or row stride");
  if (a->cache.rope_dim ? a->rot_dim != a->cache.rope_dim
                        : (a->rot_dim < 0 || a->rot_dim % 16 || a->rot_dim > a->cache.latent_dim))
    return fail(FCMOE_EINVAL, "latent_cache_append: the table must rotate rope_dim values, or a multiple of 16 of the "
                              "latent's when rope_dim is 0");
  if (a->tokens == 0) return FCMOE_OK;
  if (!a->kv || !a->positions || !a->slots || (a->rot_dim && !a->cos_sin) || a->table_rows < 0 ||
      (uintptr_t)a->kv % 16 || (uintptr_t)a->rows_out % 16 || (uintptr_t)a->weight % 16 || (uintptr_t)a->cos_sin % 16)
    return fail(FCMOE_EINVAL, "latent_cache_append: NULL or unaligned pointer");
  Append p{};
  p.kv = a->kv, p.ldkv = a->kv_row_stride, p.tokens = a->tokens;
  p.positions = a->positions, p.slots = a->slots, p.pos_i64 = a->positions_i64, p.slot_i64 = a->slots_i64;
  p.table = a->cos_sin, p.table_rows = a->table_rows, p.rot = (int)a->rot_dim;
  p.weight = a->weight, p.eps = a->eps, p.interleaved = a->interleaved, p.rows_out = a->rows_out;
  p.c = a->cache;
  if (W == 576)
    append_launch<512, 64>(p, stream);
  else if (W == 512)
    append_launch<512, 0>(p, stream);
  else if (W == 320)
    append_launch<256, 64>(p, stream);
  else
    append_launch<256, 0>(p, stream);
  return check_launch("latent_cache_append");
}
