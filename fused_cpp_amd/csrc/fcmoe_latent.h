// fcmoe_latent.h -- device helpers shared by the latent-attention kernels.
//
// Matrix layouts used throughout (64-lane wavefront, l the lane):
//   16x16x32 bf16: A lane l holds row l % 16, k 8 (l / 16) .. + 7; B the same
//     with the column; C lane l holds column l % 16, rows 4 (l / 16) + i.
//   32x32x16 bf16: A lane l holds row l % 32, k 8 (l / 32) .. + 7; B the same
//     with the column; C lane l holds column l % 32, row 8 (i / 4) +
//     4 (l / 32) + i % 4 in register i.
// Attention computes S^T = K Q^T (rows are keys, columns query rows) and
// O^T = V^T P^T: a query row then is one column, i.e. one lane, through both
// products, so its softmax statistics are per-lane scalars and P^T's registers
// are already where the second product's B operand wants them, for a key order
// of the k dimension that V^T's reads follow.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "fcmoe_device.h"

namespace fcmoe {

typedef float v2f __attribute__((ext_vector_type(2)));
typedef float v16f __attribute__((ext_vector_type(16)));
typedef __bf16 v2bf __attribute__((ext_vector_type(2)));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef int v2i __attribute__((ext_vector_type(2)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));

typedef __attribute__((address_space(3))) uint8_t lds_u8;

constexpr int kBufWord3 = 0x00020000;  // raw buffer resource word 3 for gfx9: 32-bit data format, no swizzle
constexpr float kE4M3Max = 448.0f;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// Two binary32 values to bf16 in one word (v_cvt_pk_bf16_f32: nearest even, NaN kept).
__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
  v2f f;
  f[0] = a;
  f[1] = b;
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(f, v2bf));
}
__device__ __forceinline__ uint16_t round_bf16(float a) { return (uint16_t)(pack_bf16(a, a) & 0xffffu); }

// Four binary32 values to e4m3 (nearest even; |v| <= 448 or NaN).
__device__ __forceinline__ uint32_t pack_e4m3(float a, float b, float c, float d) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
}

// Eight e4m3 bytes to eight bf16 values (exact).
__device__ __forceinline__ v8bf widen_e4m3(v2i u) {
  v8bf r;
  const v2bf a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(u[0], 1.0f, false);
  const v2bf b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(u[0], 1.0f, true);
  const v2bf c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(u[1], 1.0f, false);
  const v2bf d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(u[1], 1.0f, true);
  r[0] = a[0], r[1] = a[1], r[2] = b[0], r[3] = b[1], r[4] = c[0], r[5] = c[1], r[6] = d[0], r[7] = d[1];
  return r;
}

// Transposing LDS reads. Within each group of 16 lanes, ds_read_b64_tr_b16
// takes a block of 4 rows x 16 values (row j at the addresses of lanes 4 j ..
// 4 j + 3, 8 bytes each) and gives lane i column i; ds_read_b64_tr_b8 takes
// 8 rows x 16 bytes (row j at lanes 2 j, 2 j + 1) and gives lane i column i.
__device__ __forceinline__ v4s read_tr16(const lds_u8* __restrict__ p) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) v4s*)p);
}
__device__ __forceinline__ v2i read_tr8(const lds_u8* __restrict__ p) {
  return __builtin_amdgcn_ds_read_tr8_b64_v2i32((__attribute__((address_space(3))) v2i*)p);
}
__device__ __forceinline__ v8bf join_tr16(v4s lo, v4s hi) {
  typedef short v8s __attribute__((ext_vector_type(8)));
  return __builtin_bit_cast(v8bf, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
}

// 16 bytes a lane from memory straight to LDS: lane l's land at dst + 16 l
// (dst the same in all lanes). Counts in vmcnt. The second form reads a buffer
// at a byte offset, zeros past its end (which a part
// that is the same for all lanes does not count against).
__device__ __forceinline__ void load_lds16(const void* src, lds_u8* dst) {
  __builtin_amdgcn_global_load_lds((__attribute__((address_space(1))) void*)src,
                                   (__attribute__((address_space(3))) void*)dst, 16, 0, 0);
}
__device__ __forceinline__ void load_lds16(const __amdgpu_buffer_rsrc_t src, lds_u8* dst, uint32_t offset,
                                           uint32_t uniform_offset = 0) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(src, (__attribute__((address_space(3))) void*)dst, 16, offset, uniform_offset, 0, 0);
}
__device__ __forceinline__ void load_lds4(const __amdgpu_buffer_rsrc_t src, lds_u8* dst, uint32_t offset) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(src, (__attribute__((address_space(3))) void*)dst, 4, offset, 0, 0, 0);
}

template <int N>
__device__ __forceinline__ void wait_vm() {
  static_assert(N >= 0 && N < 64, "vmcnt range");
  __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | (7 << 4) | (15 << 8));
}
// This wave's loads (to registers and to LDS) and LDS accesses have ended, then the workgroup barrier.
__device__ __forceinline__ void loads_barrier() {
  __builtin_amdgcn_s_waitcnt(0x0070);  // vmcnt(0) lgkmcnt(0)
  __builtin_amdgcn_s_barrier();
}
// LDS accesses only.
__device__ __forceinline__ void lds_only_barrier() {
  __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
  __builtin_amdgcn_s_barrier();
}

// The value of lane l ^ 32.
__device__ __forceinline__ float other_half(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  // lanes 0..31 of r[1] hold the upper half's values, lanes 32..63 of r[0] the lower half's
  return __uint_as_float((threadIdx.x & 32) ? r[0] : r[1]);
}

// A value the compiler cannot see through: what depends on it is formed after this point.
__device__ __forceinline__ int64_t opaque_uniform(int64_t v) {
  asm volatile("" : "+s"(v));
  return v;
}
__device__ __forceinline__ int opaque_uniform(int v) {
  asm volatile("" : "+s"(v));
  return v;
}
// The lane's number, formed anew: what depends on it is neither kept in a register nor hoisted past this point. (The
// instructions are the compiler's, which puts the waits around them that a product in flight asks for.)
__device__ __forceinline__ int lane_now() {
  const uint32_t all = (uint32_t)opaque_uniform(-1);
  return (int)__builtin_amdgcn_mbcnt_hi(all, __builtin_amdgcn_mbcnt_lo(all, 0));
}
// A value that is the same in all lanes, in scalar registers.
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ int64_t uniform(int64_t v) {
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)v);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_readfirstlane((int)((uint64_t)v >> 32));
  return (int64_t)(((uint64_t)hi << 32) | lo);
}
__device__ __forceinline__ float uniform(float v) {
  return __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(v)));
}

// The wave's number in its workgroup, known to be the same in all its lanes.
__device__ __forceinline__ int wave_index() { return __builtin_amdgcn_readfirstlane((int)threadIdx.x / kWave); }
// Lane l's value, in scalar registers (l the same for the whole wave).
__device__ __forceinline__ uint64_t lane_value(uint64_t v, int l) {
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, l);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), l);
  return ((uint64_t)hi << 32) | lo;
}

// Lengths that the device reads are bounded here, so that no value of them
// leads a kernel outside the tensors and workspaces the host has checked.
struct SeqSpan {
  int64_t q0;  // first query token
  int n;       // query tokens; below 0 where the next start lies below this one, until follow()
  int64_t k0;  // first key (expanded form)
  int len;     // keys
};

__device__ __forceinline__ int64_t clamp64(int64_t v, int64_t lo, int64_t hi) {
  return v < lo ? lo : v > hi ? hi : v;
}

// Inclusive sum over the wave's lanes: DPP moves within rows of 16, then the
// rows' ends to the rows behind them (an LDS-crossbar scan costs six dependent
// round trips).
template <int CTRL, int ROWS>
__device__ __forceinline__ int64_t add_dpp(int64_t v) {
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)v, CTRL, ROWS, 0xf, true);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)((uint64_t)v >> 32), CTRL, ROWS, 0xf, true);
  return v + (int64_t)(((uint64_t)hi << 32) | lo);
}
__device__ __forceinline__ int64_t wave_scan(int64_t v) {
  v = add_dpp<0x111, 0xf>(v);  // row_shr:1
  v = add_dpp<0x112, 0xf>(v);  // row_shr:2
  v = add_dpp<0x114, 0xf>(v);  // row_shr:4
  v = add_dpp<0x118, 0xf>(v);  // row_shr:8
  v = add_dpp<0x142, 0xa>(v);  // row_bcast:15 into rows 1 and 3
  v = add_dpp<0x143, 0xc>(v);  // row_bcast:31 into rows 2 and 3
  return v;
}

// Inclusive maximum over the wave's lanes of values that are not negative.
template <int CTRL, int ROWS>
__device__ __forceinline__ int max_dpp(int v) {
  return max(v, __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xf, true));
}
__device__ __forceinline__ int wave_scan_max(int v) {
  v = max_dpp<0x111, 0xf>(v);
  v = max_dpp<0x112, 0xf>(v);
  v = max_dpp<0x114, 0xf>(v);
  v = max_dpp<0x118, 0xf>(v);
  v = max_dpp<0x142, 0xa>(v);
  v = max_dpp<0x143, 0xc>(v);
  return v;
}

// Query spans of 64 neighbouring sequences, one a lane, made to follow one
// another: a start below an earlier one counts as that one. So no token belongs
// to two sequences, and a batch has no more rows than tokens whatever the
// starts are, which is what row groups, row blocks and workspaces are counted
// by. `high` is the largest start before these sequences; returns the one
// behind them. Starts in order cost a compare a lane.
__device__ __forceinline__ int follow(SeqSpan& s, int high) {
  if (__any(s.n < 0 || s.q0 < high)) {
    const int end = (int)s.q0 + s.n, first = max(high, wave_scan_max((int)s.q0));
    s.q0 = first;
    s.n = max(end - first, 0);
  }
  return __builtin_amdgcn_readlane((int)s.q0 + s.n, kWave - 1);
}

// Finds the sequence that item `item` (0 <= item) falls into, where a sequence
// with span s holds count(s) items: its index and span and the items before it;
// -1 past the last. The whole wave takes part and gets the same answer.
template <typename S, typename F>
__device__ __forceinline__ int find_sequence(int batch, int64_t item, S span, F count, SeqSpan* found, int64_t* before) {
  int64_t base = 0;
  int high = 0;
  for (int b0 = 0; b0 < batch; b0 += kWave) {
    const int b = b0 + lane_now();
    SeqSpan s{high, 0, 0, 0};
    if (b < batch) s = span(b);
    high = follow(s, high);
    const int64_t mine = b < batch ? count(s) : 0;
    const int64_t upto = base + wave_scan(mine);
    const uint64_t hit = __ballot(upto > item);
    if (hit) {
      const int first = __ffsll((unsigned long long)hit) - 1;
      found->q0 = (int64_t)lane_value((uint64_t)s.q0, first);
      found->k0 = (int64_t)lane_value((uint64_t)s.k0, first);
      found->n = __builtin_amdgcn_readlane(s.n, first);
      found->len = __builtin_amdgcn_readlane(s.len, first);
      *before = (int64_t)lane_value((uint64_t)(upto - mine), first);
      return b0 + first;
    }
    base = (int64_t)lane_value((uint64_t)upto, kWave - 1);
  }
  *before = base;
  return -1;
}
// Items of the whole batch.
template <typename S, typename F>
__device__ __forceinline__ int64_t count_items(int batch, S span, F count) {
  int64_t sum = 0;
  int high = 0;
  for (int b0 = 0; b0 < batch; b0 += kWave) {
    const int b = b0 + lane_now();
    SeqSpan s{high, 0, 0, 0};
    if (b < batch) s = span(b);
    high = follow(s, high);
    sum += b < batch ? count(s) : 0;
  }
  return (int64_t)lane_value((uint64_t)wave_scan(sum), kWave - 1);
}

// Tokens that no sequence holds (before the first start, behind the largest)
// become zero, their lse -inf: the workgroups of an attention launch share
// them out, `wg` of `wgs`. For outputs that the call allocates; a caller's own
// output keeps those rows.
__device__ __forceinline__ void zero_uncovered(const int32_t* starts, int batch, int64_t tokens, int heads, int dim,
                                               uint16_t* out, int64_t ot, int64_t oh, float* lse, int64_t wg,
                                               int64_t wgs) {
  const int64_t first = clamp64(starts[0], 0, tokens);
  int64_t end = clamp64(starts[batch], 0, tokens);
  if (first == 0 && end == tokens) return;
  int top = (int)end;
  for (int b = lane_now(); b < batch; b += kWave) top = max(top, (int)clamp64(starts[b], 0, tokens));
  end = __builtin_amdgcn_readlane(wave_scan_max(top), kWave - 1);
  for (int64_t t = wg; t < tokens; t += wgs) {
    if (t >= first && t < end) continue;
    for (int k = (int)threadIdx.x; k < heads * (dim / 4); k += (int)blockDim.x) {
      const int h = k / (dim / 4), d = k % (dim / 4) * 4;
      *(uint2*)(out + t * ot + h * oh + d) = make_uint2(0, 0);
    }
    if (lse)
      for (int h = (int)threadIdx.x; h < heads; h += (int)blockDim.x) lse[t * heads + h] = -INFINITY;
  }
}

}  // namespace fcmoe
