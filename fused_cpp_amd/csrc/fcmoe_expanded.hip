// fcmoe_expanded.hip -- latent attention in its expanded form: causal
// attention over per-head keys and values, for prompts.
//
//   s_ij = scale * (q_i[:N] . k_j + q_i[N:] . r_j),  out_i = sum_j softmax_j(s_ij) v_j
//
// kv [S, H, N + V] is the up-projection's output (keys then values of a head),
// r [S, P] the rotated key part that all heads share: both are read where they
// lie, nothing is concatenated. Sequences are packed: sequence b has query
// tokens query_starts[b] .. [b + 1] and keys kv_starts[b] .. [b + 1]; query i
// of n sees keys 0 .. L - n + i (causal) or all L.
//
// One pass over the keys with the running maximum and sum of the softmax.
// Products are S^T = K Q^T and O^T = V^T P^T (see fcmoe_latent.h): Q stays in
// registers, P never leaves them, and V^T comes from transposing LDS reads. A
// workgroup of four waves owns a block of query rows of one head and walks the
// keys in tiles of 64, brought straight from memory to LDS ahead of their use.
// Two kernels:
//
// narrow: 128 rows, 32 a wave, two workgroups a CU, whose waves fill each
//   other's waits. What one has before its first tile and behind its last (some
//   8000 and 2000 clocks) is hidden by the other as far as that has tiles left; a
//   tile of one takes some 5000 clocks, in which each SIMD has 2560 of products
//   for the two.
// wide: 256 rows, 64 a wave, one workgroup a CU: every fragment read from LDS
//   feeds two products, and the exponentials of one tile stand between the
//   products of the next, written out in that order. 16384 tokens, 16 heads: 1120
//   us against 1400, 1.23 PFLOP/s of what causality leaves (large matrix products
//   reach 1.23 to 1.5); the matrix units are busy 0.65 of the launch's clocks, masked
//   tiles and the ends of row blocks included.
#include <type_traits>

#include "fcmoe_internal.h"
#include "fcmoe_latent.h"

namespace fcmoe {

namespace {

constexpr int kExpWaves = 4;
constexpr int kNarrowRows = 32 * kExpWaves, kWideRows = 64 * kExpWaves;  // query rows of a workgroup
constexpr int kKRing = 3, kVRing = 4;     // slots of K tiles and of V tiles
constexpr int kExpKeys = 64;              // keys of a tile

struct Expanded {
  const uint16_t* q;
  int64_t qt, qh;
  const uint16_t* kv;
  int64_t kt, kh;
  const uint16_t* r;
  int64_t rt;
  const int32_t* q_starts;
  const int32_t* kv_starts;
  int64_t tokens, keys;
  int batch, heads, causal, splits;
  int rows;        // of a row block: kNarrowRows or kWideRows
  int64_t blocks;  // upper bound of the batch's row blocks
  float scale;
  uint16_t* out;
  int64_t ot, oh;
  float* lse;        // [tokens, heads] or nullptr
  float* part_o;     // splits > 1: [splits][blocks * heads][4 waves][V / 8][64 lanes][4]
  float* part_lse;   // [splits][blocks * heads][128], base 2
  int zero_tail;
};

__device__ __forceinline__ SeqSpan expanded_span(const Expanded& p, int b) {
  SeqSpan s;
  s.q0 = clamp64(p.q_starts[b], 0, p.tokens);
  s.n = (int)(clamp64(p.q_starts[b + 1], 0, p.tokens) - s.q0);
  s.k0 = clamp64(p.kv_starts[b], 0, p.keys);
  s.len = (int)(clamp64(p.kv_starts[b + 1], s.k0, p.keys) - s.k0);
  return s;
}

// Keys that query row i of a sequence sees.
__device__ __forceinline__ int expanded_limit(const Expanded& p, const SeqSpan& s, int i) {
  if (!p.causal) return s.len;
  const int v = s.len - s.n + i + 1;
  return v < 0 ? 0 : v > s.len ? s.len : v;
}

// LDS swizzle: 16-byte unit u of key row k is stored at u ^ swz(k) (within the
// row part's units). K reads take one unit of 32 neighbouring keys, V^T reads
// units of 4 neighbouring keys in pairs: with key bits (b0 b1) moved up by one
// and b2 below them both fall on distinct banks.
__device__ __forceinline__ int swz(int key) { return ((key & 3) << 1) | ((key >> 2) & 1) | (key & 8); }

template <int N, int P, int V>
__global__ __launch_bounds__(kExpWaves * kWave, 2) void expanded_narrow_kernel(const Expanded p) {
  constexpr int DK = N + P;
  constexpr int RB = 2 * (N + V);                  // bytes of a kv row
  constexpr int KV_BYTES = kExpKeys * RB;          // kv rows, then the shared key rows
  constexpr int TILE_BYTES = KV_BYTES + kExpKeys * 2 * P;
  constexpr int KV_LOADS = KV_BYTES / 1024 / kExpWaves, R_LOADS = kExpKeys * 2 * P / 1024 / kExpWaves;
  constexpr int UNITS = RB / 16;                   // 16-byte units of a kv row
  constexpr int KMASK = N / 8 - 1, VMASK = V / 8 - 1;
  constexpr int TO = V / 32;
  static_assert((N == 64 || N == 128) && V == N && (P == 0 || P == 64), "compiled head sizes");
  __shared__ __align__(1024) uint8_t smem[2 * TILE_BYTES];
  lds_u8* lds = (lds_u8*)smem;

  if (p.zero_tail)
    zero_uncovered(p.q_starts, p.batch, p.tokens, p.heads, V, p.out, p.ot, p.oh, p.lse, blockIdx.x, gridDim.x);
  const int lane = (int)threadIdx.x % kWave, wave = (int)threadIdx.x / kWave;
  // heads fastest: concurrent workgroups of one head share an XCD's L2 when
  // the heads are a multiple of 8; row blocks from the last (the longest rows
  // of a causal sequence) to the first
  const uint32_t items = (uint32_t)(p.blocks * p.heads);  // 32-bit divisions: a 64-bit one takes a hundred instructions
  const uint32_t split = blockIdx.x / items, item = blockIdx.x - split * items;
  const int head = (int)(item % (uint32_t)p.heads);
  const int64_t block = p.blocks - 1 - item / (uint32_t)p.heads;
  int64_t before;
  SeqSpan seq;
  const int b = find_sequence(
      p.batch, block, [&](int s) { return expanded_span(p, s); },
      [](const SeqSpan& s) { return ((int64_t)s.n + kNarrowRows - 1) / kNarrowRows; }, &seq, &before);
  if (b < 0) return;
  const int i0 = (int)(block - before) * kNarrowRows;
  const int wave_i0 = i0 + 32 * wave;
  const bool live = wave_i0 < seq.n;
  const int wave_i1 = min(wave_i0 + 31, seq.n - 1);
  const int lim_min = live ? expanded_limit(p, seq, wave_i0) : 0;
  const int lim_max = live ? expanded_limit(p, seq, wave_i1) : 0;
  const int my_i = min(wave_i0 + lane % 32, seq.n - 1);
  const int my_lim = expanded_limit(p, seq, my_i);

  const int tiles = (expanded_limit(p, seq, min(i0 + kNarrowRows, seq.n) - 1) + kExpKeys - 1) / kExpKeys;
  // tiles <= 2^25 and splits <= 64
  const int t_begin = (int)((uint32_t)tiles * split / (uint32_t)p.splits);
  const int t_end = (int)((uint32_t)tiles * (split + 1) / (uint32_t)p.splits);

  // ---- stage loads: wave w brings keys 16 w .. 16 w + 15 of a tile
  const char* kv_base = (const char*)(p.kv + seq.k0 * p.kt + head * p.kh);
  const char* r_base = P ? (const char*)(p.r + seq.k0 * p.rt) : nullptr;
  const uint32_t kv_step = (uint32_t)p.kt * 2, r_step = P ? (uint32_t)p.rt * 2 : 0;
  auto stage = [&](int tile, int buf) {
    lds_u8* dst = lds + buf * TILE_BYTES;
    const int first = tile * kExpKeys;
    const int last = seq.len - 1 - first;  // keys past the sequence re-read its last one; their scores are masked
    const char* kb = kv_base + (int64_t)first * kv_step;
#pragma unroll
    for (int u = 0; u < KV_LOADS; ++u) {
      const int piece = wave * KV_LOADS + u;
      const int key = piece * (64 / UNITS) + lane / UNITS;
      const int slot = lane % UNITS;
      const int unit = slot ^ (swz(key) & KMASK);  // KMASK == VMASK: keys and values keep to their halves of the row
      load_lds16(kb + (uint32_t)((uint32_t)min(key, last) * kv_step + unit * 16), dst + piece * 1024);
    }
    if constexpr (P > 0) {
      const char* rb = r_base + (int64_t)first * r_step;
#pragma unroll
      for (int u = 0; u < R_LOADS; ++u) {
        const int piece = wave * R_LOADS + u;
        const int key = piece * 8 + lane / 8;
        const int unit = (lane % 8) ^ (swz(key) & 7);
        load_lds16(rb + (uint32_t)((uint32_t)min(key, last) * r_step + unit * 16), dst + KV_BYTES + piece * 1024);
      }
    }
  };

  if (t_begin < t_end) stage(t_begin, 0);

  // ---- Q: B operand, column lane % 32, values 16 ks + 8 (lane / 32) ..
  v8bf qf[DK / 16];
  {
    const uint16_t* qrow = p.q + (seq.q0 + my_i) * p.qt + head * p.qh + 8 * (lane / 32);
#pragma unroll
    for (int ks = 0; ks < DK / 16; ++ks) qf[ks] = *(const v8bf*)(qrow + 16 * ks);
  }

  // ---- fragment addresses within a buffer
  const int half = lane / 32;
  const int krow = lane % 32;
  const int kx = swz(krow);
  int va[VMASK >= 15 ? 4 : 2];
  {
    const int g = lane / 16, i = lane % 16, j = i / 4, e = 2 * (g & 1) + (i % 4) / 2;
    const int key = 4 * half + j;
#pragma unroll
    for (int t = 0; t < (VMASK >= 15 ? 4 : 2); ++t)
      va[t] = key * RB + 2 * N + (((4 * t + e) ^ swz(key)) & VMASK) * 16 + (i & 1) * 8;
  }

  const float c2 = p.scale * kLog2e;
  float m = -INFINITY, l = 0.0f;
  v16f o[TO];
#pragma unroll
  for (int t = 0; t < TO; ++t)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[t][i] = 0.0f;

  for (int tile = t_begin; tile < t_end; ++tile) {
    const int buf = (tile - t_begin) & 1;
    loads_barrier();  // the tile has landed; everyone is done with the other buffer
    if (tile + 1 < t_end) stage(tile + 1, buf ^ 1);
    if (tile * kExpKeys >= lim_max) continue;
    const lds_u8* kb = lds + buf * TILE_BYTES;

    v16f s[2];
#pragma unroll
    for (int hf = 0; hf < 2; ++hf)
#pragma unroll
      for (int i = 0; i < 16; ++i) s[hf][i] = 0.0f;
#pragma unroll
    for (int ks = 0; ks < DK / 16; ++ks) {
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        const int unit = ks < N / 16 ? (2 * ks + half) ^ (kx & KMASK) : (2 * (ks - N / 16) + half) ^ (kx & 7);
        const int at = ks < N / 16 ? (krow + 32 * hf) * RB + unit * 16 : KV_BYTES + (krow + 32 * hf) * 2 * P + unit * 16;
        const v8bf kf = *(const __attribute__((address_space(3))) v8bf*)(kb + at);
        s[hf] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf, qf[ks], s[hf], 0, 0, 0);
      }
    }

    if ((tile + 1) * kExpKeys > lim_min) {
      const int lim = my_lim - tile * kExpKeys - 4 * half;
#pragma unroll
      for (int hf = 0; hf < 2; ++hf)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (32 * hf + 8 * (i / 4) + i % 4 >= lim) s[hf][i] = -INFINITY;
    }
    float top = s[0][0];
#pragma unroll
    for (int i = 1; i < 16; ++i) top = fmaxf(top, s[0][i]);
#pragma unroll
    for (int i = 0; i < 16; ++i) top = fmaxf(top, s[1][i]);
    top = fmaxf(top, other_half(top));
    // The reference point m only has to be near the maximum (exp2 of up to
    // 2^8 is far inside binary32 and bf16): O is rescaled when some row's
    // maximum has grown past it by more than that, seldom after the first tile.
    if (__any((top - m) * c2 > 8.0f)) {
      const float mn = fmaxf(m, top);
      const float a = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((m - mn) * c2);
      m = mn;
      l *= a;
#pragma unroll
      for (int t = 0; t < TO; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[t][i] *= a;
    }
    const float mc = m == -INFINITY ? 0.0f : m * c2;
    // The weights go into P V as bf16, off by at most 2^-8 of themselves: a product's operands are of one type, and a second
    // part of each would double the products. Their sum is of what they were before (of the rounded ones it would leave the
    // output's error as it is, and lse worse).
    v8bf pf[4];
#pragma unroll
    for (int st = 0; st < 4; ++st) {
      float e[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        e[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[st / 2][8 * (st % 2) + i], c2, -mc));
        l += e[i];
      }
      v4u w;
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = pack_bf16(e[2 * i], e[2 * i + 1]);
      pf[st] = __builtin_bit_cast(v8bf, w);
    }
#pragma unroll
    for (int st = 0; st < 4; ++st)
#pragma unroll
      for (int t = 0; t < TO; ++t) {
        const v4s lo = read_tr16(kb + va[t] + 16 * st * RB);
        const v4s hi = read_tr16(kb + va[VMASK >= 15 ? t ^ 2 : t] + (16 * st + 8) * RB);
        o[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(join_tr16(lo, hi), pf[st], o[t], 0, 0, 0);
      }
  }

  l += other_half(l);
  if (!live) return;
  const bool mine = wave_i0 + lane % 32 < seq.n;
  // a row that sees no key has l == 0: its output is 0 and its lse -inf
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  if (p.splits > 1) {
    const int64_t at = ((int64_t)split * items + item) * kExpWaves + wave;
    if (lane < 32) p.part_lse[at * 32 + lane] = l == 0.0f ? -INFINITY : __builtin_fmaf(m, c2, log2f(l));
    float4* po = (float4*)p.part_o + at * (TO * 4) * 64 + lane;
#pragma unroll
    for (int t = 0; t < TO; ++t)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        po[(4 * t + g) * 64] = make_float4(o[t][4 * g] * inv, o[t][4 * g + 1] * inv, o[t][4 * g + 2] * inv, o[t][4 * g + 3] * inv);
    return;
  }
  if (!mine) return;
  const int64_t token = seq.q0 + wave_i0 + lane % 32;
  if (p.lse && lane < 32) p.lse[token * p.heads + head] = l == 0.0f ? -INFINITY : __builtin_fmaf(m, p.scale, logf(l));
  uint16_t* orow = p.out + token * p.ot + head * p.oh + 4 * half;
#pragma unroll
  for (int t = 0; t < TO; ++t)
#pragma unroll
    for (int g = 0; g < 4; ++g)
      *(uint2*)(orow + 32 * t + 8 * g) = make_uint2(pack_bf16(o[t][4 * g] * inv, o[t][4 * g + 1] * inv),
                                                    pack_bf16(o[t][4 * g + 2] * inv, o[t][4 * g + 3] * inv));
}

// acc (+)= K fragment x Q fragment, Q in accumulation registers; O^T (in
// accumulation registers) += V^T fragment x P fragment. The compiler does not
// know these for MFMAs, so the waits it would put in stand around them:
// operands_ready where an ordinary instruction may just have written an operand
// (two states), mfma_done and acc_done before anything else touches an
// accumulator.
template <bool FIRST>
__device__ __forceinline__ void mfma_qk(v16f& acc, const v8bf& k, const v8bf& q) {
  if constexpr (FIRST)
    asm volatile("v_mfma_f32_32x32x16_bf16 %0, %1, %2, 0" : "=&v"(acc) : "v"(k), "a"(q));
  else
    asm volatile("v_mfma_f32_32x32x16_bf16 %0, %1, %2, %0" : "+v"(acc) : "v"(k), "a"(q));
}
__device__ __forceinline__ void mfma_pv(v16f& acc, const v8bf& v, const v4u& p) {
  asm volatile("v_mfma_f32_32x32x16_bf16 %0, %1, %2, %0" : "+a"(acc) : "v"(v), "v"(p));
}
__device__ __forceinline__ void operands_ready() { asm volatile("s_nop 1"); }

// All products into O have left the matrix pipe.
template <int TO>
__device__ __forceinline__ void acc_done(v16f (&o)[2][TO]) {
  asm volatile("s_nop 15\n\ts_nop 7" : "+a"(o[0][0]), "+a"(o[0][1]), "+a"(o[1][0]), "+a"(o[1][1]));
  if constexpr (TO == 4) asm volatile("" : "+a"(o[0][2]), "+a"(o[0][3]), "+a"(o[1][2]), "+a"(o[1][3]));
}

// The same for S, for products that ended 24 or 8 states before.
template <int STATES>
__device__ __forceinline__ void mfma_done(v16f (&s)[2][2]) {
  static_assert(STATES == 24 || STATES == 8, "");
  if constexpr (STATES == 24)
    asm volatile("s_nop 15\n\ts_nop 7" : "+v"(s[0][0]), "+v"(s[0][1]), "+v"(s[1][0]), "+v"(s[1][1]));
  else
    asm volatile("s_nop 7" : "+v"(s[0][0]), "+v"(s[0][1]), "+v"(s[1][0]), "+v"(s[1][1]));
}
// One value to the compiler, which would pass its 16 parts around loops and
// branches one by one, those of an accumulator in ordinary registers.
__device__ __forceinline__ void whole(v16f& v) { asm volatile("" : "+v"(v)); }
__device__ __forceinline__ void whole_acc(v16f& v) { asm volatile("" : "+a"(v)); }

// All but this wave's last N loads have landed, then the workgroup barrier.
template <int N>
__device__ __forceinline__ void meet() {
  wait_vm<N>();
  __builtin_amdgcn_s_barrier();
}
template <typename T>
__device__ __forceinline__ void here_one(T& v) {
  asm volatile("" : "+v"(v));
}
// These values are formed here: the compiler would move them behind the next
// branch, out of the products' shadow.
template <typename... T>
__device__ __forceinline__ void here(T&... v) {
  (here_one(v), ...);
}

__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_of(const char* base, uint32_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc((void*)base, (short)0, (int)bytes, kBufWord3);
}

// f(integral_constant<int, 0>), f(integral_constant<int, 1>) ..
template <int N, int I = 0, typename F>
__device__ __forceinline__ void unroll(F f) {
  if constexpr (I < N) {
    f(std::integral_constant<int, I>{});
    unroll<N, I + 1>(f);
  }
}

// Step j of J takes items begin(j) .. begin(j + 1) of n.
constexpr int share_of(int j, int steps, int n) { return (n * j) / steps; }

template <int N, int P, int V>
__global__ __launch_bounds__(kExpWaves * kWave, 1) void expanded_wide_kernel(const Expanded p) {
  constexpr int DK = N + P, KS = DK / 16, TO = V / 32, NV = 4 * TO;
  constexpr int KSLOT = kExpKeys * 2 * (N + P), VSLOT = kExpKeys * 2 * V, VOFF = kKRing * KSLOT;
  constexpr int KL = N / 32, RL = P / 32, VL = V / 32;  // a wave's loads (1 KB each) of a tile: its 16 keys
  constexpr int LOADS = KL + RL + VL;
  constexpr int kAhead = 3, vAhead = 5;  // fragments are read this many uses ahead
  static_assert((N == 64 || N == 128) && V == N && (P == 0 || P == 64), "compiled head sizes");
  __shared__ __align__(1024) uint8_t smem[kKRing * KSLOT + kVRing * VSLOT];
  lds_u8* lds = (lds_u8*)smem;

  if (p.zero_tail)
    zero_uncovered(p.q_starts, p.batch, p.tokens, p.heads, V, p.out, p.ot, p.oh, p.lse, blockIdx.x, gridDim.x);
  const int lane = (int)threadIdx.x % kWave, wave = wave_index();
  const uint32_t items = (uint32_t)(p.blocks * p.heads);  // 32-bit divisions: a 64-bit one takes a hundred instructions
  const uint32_t split = blockIdx.x / items, item = blockIdx.x - split * items;
  const int head = (int)(item % (uint32_t)p.heads);
  const int64_t block = p.blocks - 1 - item / (uint32_t)p.heads;
  int64_t before;
  SeqSpan seq;
  const int b = find_sequence(
      p.batch, block, [&](int s) { return expanded_span(p, s); },
      [](const SeqSpan& s) { return ((int64_t)s.n + kWideRows - 1) / kWideRows; }, &seq, &before);
  if (b < 0) return;
  const int i0 = (int)(block - before) * kWideRows;
  const int wave_i0 = i0 + 64 * wave;
  const bool live = wave_i0 < seq.n;
  const int lim_min = live ? expanded_limit(p, seq, wave_i0) : 0;
  const int lim_max = live ? expanded_limit(p, seq, min(wave_i0 + 63, seq.n - 1)) : 0;
  const int tiles = (expanded_limit(p, seq, min(i0 + kWideRows, seq.n) - 1) + kExpKeys - 1) / kExpKeys;
  // tiles <= 2^25 and splits <= 64
  const int t_begin = (int)((uint32_t)tiles * split / (uint32_t)p.splits);
  const int t_end = (int)((uint32_t)tiles * (split + 1) / (uint32_t)p.splits);
  const int w_end = min(t_end, (lim_max + kExpKeys - 1) / kExpKeys);  // this wave's tiles end here
  const int half = lane / 32;

  // ---- stage loads: wave w brings keys 16 w .. 16 w + 15 of a tile
  const uint32_t kv_step = (uint32_t)p.kt * 2, r_step = P ? (uint32_t)p.rt * 2 : 0;
  const char* kv_base = (const char*)(p.kv + seq.k0 * p.kt + head * p.kh);
  const char* r_base = P ? (const char*)(p.r + seq.k0 * p.rt) : nullptr;
  constexpr int KPL = 512 / N;  // keys of a load
  uint32_t kv_lane[KL], r_lane[P ? RL : 1];
#pragma unroll
  for (int u = 0; u < KL; ++u) {
    const int key = u * KPL + lane / (N / 8);
    kv_lane[u] = (16 * wave + key) * kv_step + (((lane % (N / 8)) ^ (swz(key) & (N / 8 - 1))) * 16);
  }
#pragma unroll
  for (int u = 0; u < RL; ++u)
    r_lane[u] = (16 * wave + 8 * u + lane / 8) * r_step + (((lane % 8) ^ (swz(lane / 8) & 7)) * 16);
  // Keys past the sequence read as zeros (the buffer ends with its last row),
  // and so does a tile past the end: every step issues the same loads.
  struct Loads {
    __amdgpu_buffer_rsrc_t k, r, v;
    lds_u8 *kd, *vd;
  };
  int k_tile = t_begin, v_tile = t_begin, k_to = 0, v_to = 0;  // the tiles to load next and their slots
  auto keys_of = [&](int tile) { return tile < t_end ? min(seq.len - 1 - tile * kExpKeys, kExpKeys) : -1; };
  auto next_k = [&](Loads& n) {
    const int keys = keys_of(k_tile);  // but one
    const int64_t first = (int64_t)k_tile * kExpKeys;
    n.k = rows_of(kv_base + first * kv_step, keys < 0 ? 0 : (uint32_t)keys * kv_step + 2 * N);
    if constexpr (P > 0) n.r = rows_of(r_base + first * r_step, keys < 0 ? 0 : (uint32_t)keys * r_step + 2 * P);
    n.kd = lds + k_to * KSLOT;
    ++k_tile;
    k_to = k_to == kKRing - 1 ? 0 : k_to + 1;
  };
  auto next_v = [&](Loads& n) {
    const int keys = keys_of(v_tile);
    n.v = rows_of(kv_base + (int64_t)v_tile * kExpKeys * kv_step + 2 * N, keys < 0 ? 0 : (uint32_t)keys * kv_step + 2 * V);
    n.vd = lds + VOFF + v_to * VSLOT;
    ++v_tile;
    v_to = v_to == kVRing - 1 ? 0 : v_to + 1;
  };
  auto load_k = [&](const Loads& n, int i) {
    if (i < KL)
      load_lds16(n.k, n.kd + (wave * KL + i) * 1024, kv_lane[i]);
    else
      load_lds16(n.r, n.kd + kExpKeys * 2 * N + (wave * RL + i - KL) * 1024, r_lane[i - KL]);
  };
  auto load_v = [&](const Loads& n, int i) { load_lds16(n.v, n.vd + (wave * VL + i) * 1024, kv_lane[i]); };
  Loads ld;
#pragma unroll
  for (int step = 0; step < 3; ++step) {
    if (step > 0) {
      next_v(ld);
#pragma unroll
      for (int i = 0; i < VL; ++i) load_v(ld, i);
    }
    next_k(ld);
#pragma unroll
    for (int i = 0; i < KL + RL; ++i) load_k(ld, i);
  }

  // ---- Q: B operand, column lane % 32, values 16 ks + 8 (lane / 32) ..
  v8bf q[2][KS];
  int lim[2];
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int i = min(wave_i0 + 32 * r + lane % 32, seq.n - 1);
    lim[r] = expanded_limit(p, seq, i) - 4 * half;
    const uint16_t* qrow = p.q + (seq.q0 + i) * p.qt + head * p.qh + 8 * half;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) q[r][ks] = *(const v8bf*)(qrow + 16 * ks);
  }

  // ---- fragment addresses within a slot
  const int krow = lane % 32;
  const int ka = krow * 2 * N + (((half ^ swz(krow)) & (N / 8 - 1)) * 16);
  const int ra = kExpKeys * 2 * N + krow * 2 * P + (((half ^ swz(krow)) & 7) * 16);
  int va;
  {
    const int g = lane / 16, i = lane % 16, j = i / 4, e = 2 * (g & 1) + (i % 4) / 2;
    const int key = 4 * half + j;
    va = key * 2 * V + ((e ^ swz(key)) & (V / 8 - 1)) * 16 + (i & 1) * 8;
  }

  const float c2 = p.scale * kLog2e;
  constexpr int NM = 4 * KS, MEET = NV;  // products of S; of P V before the waves meet
  // m: a row's reference point in units of log2, -inf while it has seen no key; mz the same with 0 for that
  float m[2], mz[2], l[2] = {0.0f, 0.0f};
  float x[2][2][16];
  v16f s[2][2];

  // S = K Q^T of the tile at kb, whose first fragments are read; between(j) follows product j.
  v8bf kf[kAhead + 1][2];
  auto k_read = [&](const lds_u8* kb, int ks) {
#pragma unroll
    for (int hf = 0; hf < 2; ++hf)
      kf[ks % (kAhead + 1)][hf] =
          ks < N / 16 ? *(const __attribute__((address_space(3))) v8bf*)(kb + (ka ^ (32 * ks)) + 32 * hf * 2 * N)
                      : *(const __attribute__((address_space(3))) v8bf*)(kb + (ra ^ (32 * (ks - N / 16))) + 32 * hf * 2 * P);
  };
  auto scores = [&](const lds_u8* kb, auto between) {
    unroll<NM>([&](auto j_) {
      constexpr int j = decltype(j_)::value, ks = j / 4, hf = j / 2 % 2, r = j % 2;
      if constexpr (j % 4 == 0 && ks + kAhead < KS) k_read(kb, ks + kAhead);
      __builtin_amdgcn_sched_barrier(0);
      mfma_qk<ks == 0>(s[r][hf], kf[ks % (kAhead + 1)][hf], q[r][ks]);
      __builtin_amdgcn_sched_barrier(0);
      between(j_);
    });
  };
  auto mask = [&](int tile) {
    mfma_done<24>(s);
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (32 * hf + 8 * (i / 4) + i % 4 >= lim[r] - tile * kExpKeys) s[r][hf][i] = -INFINITY;
        whole(s[r][hf]);
      }
  };
  // From S to the exponents x, in 16 operations of four.
  auto exponents = [&](int g) {
    float* to = &x[g / 8][g % 8 / 4][4 * (g % 4)];
#pragma unroll
    for (int i = 0; i < 4; ++i) to[i] = __builtin_fmaf(s[g / 8][g % 8 / 4][4 * (g % 4) + i], c2, -mz[g / 8]);
    here(to[0], to[1], to[2], to[3]);
  };

  // Before the first tile: its S and exponents.
  wait_vm<2 * LOADS>();
  lds_only_barrier();
  {
#pragma unroll
    for (int ks = 0; ks < kAhead; ++ks) k_read(lds, ks);
    operands_ready();
    scores(lds, [](auto) {});
    if ((t_begin + 1) * kExpKeys > lim_min) mask(t_begin);
    mfma_done<24>(s);
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      float top = s[r][0][0];
#pragma unroll
      for (int i = 1; i < 32; ++i) top = fmaxf(top, s[r][i / 16][i % 16]);
      m[r] = fmaxf(top, other_half(top)) * c2;
      mz[r] = m[r] == -INFINITY ? 0.0f : m[r];
    }
    unroll<16>([&](auto k_) { exponents(decltype(k_)::value); });
  }
  bool unset = __any(m[0] == -INFINITY || m[1] == -INFINITY);
  wait_vm<LOADS>();
  lds_only_barrier();
  next_v(ld);
  next_k(ld);
#pragma unroll
  for (int i = 0; i < VL; ++i) load_v(ld, i);
#pragma unroll
  for (int ks = 0; ks < kAhead; ++ks) k_read(lds + KSLOT, ks);

  v16f o[2][TO];
#pragma unroll
  for (int r = 0; r < 2; ++r)
#pragma unroll
    for (int t = 0; t < TO; ++t) {
#pragma unroll
      for (int i = 0; i < 16; ++i) o[r][t][i] = 0.0f;
      whole_acc(o[r][t]);
    }

  // Step t forms S of tile t + 1 while tile t's exponentials are taken, then
  // adds P V of tile t while the exponents of tile t + 1 are formed. A wave's
  // last step has no tile t + 1: what it forms of it is not used.
  // The reference point only has to be near the maximum, so maxima are not taken
  // tile by tile: m stays the first tile's until the weights of a tile show that
  // some row has grown far past it (their sum is beyond 2^14, far inside
  // binary32 and bf16) and the tile's are taken anew.
  // The waves meet in the midst of P V: there all but the loads since their last
  // meeting have landed, K of t + 2 and V of t + 1 with them, and the slots of K of
  // t + 1 and V of t - 1 are free. V of t, which is still read, keeps its slot
  // until the next meeting. K's loads go between the products of S, V's behind the meeting.
  int k_at = 1, v_at = 0;  // slots of K of t + 1, of V of t
  for (int t = t_begin; t < t_end; ++t) {
    const lds_u8* kb = lds + k_at * KSLOT;
    const lds_u8* vb = lds + VOFF + v_at * VSLOT;
    k_at = k_at == kKRing - 1 ? 0 : k_at + 1;
    v_at = v_at == kVRing - 1 ? 0 : v_at + 1;
    if (t >= w_end) {
#pragma unroll
      for (int i = 0; i < KL + RL; ++i) load_k(ld, i);
      meet<LOADS>();
      next_v(ld);
      next_k(ld);
#pragma unroll
      for (int i = 0; i < VL; ++i) load_v(ld, i);
      continue;
    }
    v4s vlo[vAhead + 1], vhi[vAhead + 1];
    v4u pw[2][4];
    float e[2][4], sum[2][2] = {{0.0f, 0.0f}, {0.0f, 0.0f}};
    auto v_read = [&](int n) {
      const int st = n / TO, tt = n % TO;
      vlo[n % (vAhead + 1)] = read_tr16(vb + (va ^ (tt << 6)) + 16 * st * 2 * V);
      vhi[n % (vAhead + 1)] = read_tr16(vb + (va ^ ((TO == 4 ? tt ^ 2 : tt) << 6)) + (16 * st + 8) * 2 * V);
    };
    // The weights rounded to bf16 for P V and summed before that, as in the other form.
    auto finish = [&](int g) {  // group g: row tile g / 8, key half (g % 8) / 4, registers 4 (g % 4) ..
      const float* w = e[g & 1];
      sum[g / 8][0] += w[0] + w[1];
      sum[g / 8][1] += w[2] + w[3];
      uint32_t p0 = pack_bf16(w[0], w[1]), p1 = pack_bf16(w[2], w[3]);
      here(p0, p1, sum[g / 8][0], sum[g / 8][1]);
      pw[g / 8][g % 8 / 2][2 * (g & 1)] = p0;
      pw[g / 8][g % 8 / 2][2 * (g & 1) + 1] = p1;
    };
    auto weigh = [&](int op) {  // 48 operations: two exponentials each, every third what follows of the group before
      const int g = op / 3;
      if (op % 3 == 2) {
        if (g > 0) finish(g - 1);
      } else {
#pragma unroll
        for (int i = 2 * (op % 3); i < 2 * (op % 3) + 2; ++i)
          e[g & 1][i] = __builtin_amdgcn_exp2f(x[g / 8][g % 8 / 4][4 * (g % 4) + i]);
      }
    };
    scores(kb, [&](auto j_) {
      constexpr int j = decltype(j_)::value;
      unroll<share_of(j + 1, NM, KL + RL) - share_of(j, NM, KL + RL)>(
          [&](auto k_) { load_k(ld, share_of(j, NM, KL + RL) + decltype(k_)::value); });
      if constexpr (j % 2 == 0 && j >= NM - 2 * vAhead) v_read((j - NM) / 2 + vAhead);
      unroll<share_of(j + 1, NM, 48) - share_of(j, NM, 48)>([&](auto k_) { weigh(share_of(j, NM, 48) + decltype(k_)::value); });
    });
    finish(15);
    __builtin_amdgcn_sched_barrier(0);

    if (unset || __any(sum[0][0] + sum[0][1] > 16384.0f || sum[1][0] + sum[1][1] > 16384.0f)) {
      acc_done<TO>(o);
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        float top = x[r][0][0];
#pragma unroll
        for (int i = 1; i < 32; ++i) top = fmaxf(top, x[r][i / 16][i % 16]);
        top = fmaxf(top, other_half(top));
        const float mn = fmaxf(m[r], mz[r] + top), a = m[r] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m[r] - mn);
        const float mnz = mn == -INFINITY ? 0.0f : mn, by = mnz - mz[r];
        m[r] = mn, mz[r] = mnz;
        l[r] *= a;
#pragma unroll
        for (int i = 0; i < 32; ++i) x[r][i / 16][i % 16] -= by;
        sum[r][0] = sum[r][1] = 0.0f;
#pragma unroll
        for (int tt = 0; tt < TO; ++tt) {
#pragma unroll
          for (int i = 0; i < 16; ++i) o[r][tt][i] *= a;
          whole_acc(o[r][tt]);  // back before the next: few ordinary registers pass between
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      unroll<48>([&](auto k_) { weigh(decltype(k_)::value); });
      finish(15);
      unset = __any(m[0] == -INFINITY || m[1] == -INFINITY);
      operands_ready();
    }
    l[0] += sum[0][0] + sum[0][1];
    l[1] += sum[1][0] + sum[1][1];
    if (t + 1 < w_end && (t + 2) * kExpKeys > lim_min) mask(t + 1);
    unroll<2 * NV>([&](auto j_) {
      constexpr int j = decltype(j_)::value, n = j / 2, r = j % 2;
      if constexpr (r == 0 && n + vAhead < NV) v_read(n + vAhead);
      __builtin_amdgcn_sched_barrier(0);
      mfma_pv(o[r][n % TO], join_tr16(vlo[n % (vAhead + 1)], vhi[n % (vAhead + 1)]), pw[r][n / TO]);
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (j == MEET) {
        meet<LOADS>();
        next_v(ld);
        next_k(ld);
      }
      if constexpr (j > MEET && j <= MEET + VL) load_v(ld, j - MEET - 1);
      if constexpr (j >= 2 * NV - kAhead) k_read(lds + k_at * KSLOT, j - 2 * NV + kAhead);
      if constexpr (j == 3) {
        mfma_done<8>(s);  // four products on: S's last ones have left the pipe
      } else if constexpr (j > 3) {
        unroll<share_of(j - 3, 2 * NV - 4, 16) - share_of(j - 4, 2 * NV - 4, 16)>(
            [&](auto k_) { exponents(share_of(j - 4, 2 * NV - 4, 16) + decltype(k_)::value); });
      }
    });
    __builtin_amdgcn_sched_barrier(0);
  }

  acc_done<TO>(o);
  if (!live) return;
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    l[r] += other_half(l[r]);
    const int i = wave_i0 + 32 * r + lane % 32;
    // a row that sees no key has l == 0: its output is 0 and its lse -inf
    const float inv = l[r] == 0.0f ? 0.0f : 1.0f / l[r];
    if (p.splits > 1) {
      const int64_t at = (((int64_t)split * items + item) * kExpWaves + wave) * 2 + r;
      if (lane < 32) p.part_lse[at * 32 + lane] = l[r] == 0.0f ? -INFINITY : m[r] + log2f(l[r]);
      float4* po = (float4*)p.part_o + at * (TO * 4) * 64 + lane;
#pragma unroll
      for (int t = 0; t < TO; ++t)
#pragma unroll
        for (int g = 0; g < 4; ++g)
          po[(4 * t + g) * 64] = make_float4(o[r][t][4 * g] * inv, o[r][t][4 * g + 1] * inv, o[r][t][4 * g + 2] * inv,
                                             o[r][t][4 * g + 3] * inv);
      continue;
    }
    if (i >= seq.n) continue;
    const int64_t token = seq.q0 + i;
    if (p.lse && lane < 32) p.lse[token * p.heads + head] = l[r] == 0.0f ? -INFINITY : (m[r] + log2f(l[r])) * kLn2;
    uint16_t* orow = p.out + token * p.ot + head * p.oh + 4 * half;
#pragma unroll
    for (int t = 0; t < TO; ++t)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *(uint2*)(orow + 32 * t + 8 * g) = make_uint2(pack_bf16(o[r][t][4 * g] * inv, o[r][t][4 * g + 1] * inv),
                                                      pack_bf16(o[r][t][4 * g + 2] * inv, o[r][t][4 * g + 3] * inv));
  }
}

// Joins the splits of a row block: out = sum_s 2^(lse_s - max) O_s / sum_s 2^(lse_s - max).
// A workgroup takes 32 of the values (blockIdx.y): a CU takes some 10 bytes a clock
// from beyond its L2, so the partials are read by many (two chunks of 65 tokens
// behind 20000, 32 heads: 20 us a launch by one each, 11 so).
template <int V>
__global__ __launch_bounds__(kExpWaves * kWave) void expanded_combine_kernel(const Expanded p) {
  const int lane = (int)threadIdx.x % kWave, strips = p.rows / 32;
  const int64_t item = (int64_t)blockIdx.x * kExpWaves / strips;  // strips are a multiple of the waves
  const int strip = (int)((int64_t)blockIdx.x * kExpWaves % strips) + (int)threadIdx.x / kWave;
  const int head = (int)(item % p.heads);
  const int64_t block = p.blocks - 1 - item / p.heads;
  int64_t before;
  SeqSpan seq;
  const int b = find_sequence(
      p.batch, block, [&](int s) { return expanded_span(p, s); },
      [&](const SeqSpan& s) { return ((int64_t)s.n + p.rows - 1) / p.rows; }, &seq, &before);
  if (b < 0) return;
  const int i = (int)(block - before) * p.rows + 32 * strip + lane % 32;
  if (i >= seq.n) return;
  const int64_t step = p.blocks * p.heads * strips;
  const int64_t at = item * strips + strip;
  float top = -INFINITY;
  for (int s = 0; s < p.splits; ++s) top = fmaxf(top, p.part_lse[(at + s * step) * 32 + lane % 32]);
  float total = 0.0f;
  const int k0 = 4 * (int)blockIdx.y;
  float4 acc[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) acc[k] = make_float4(0, 0, 0, 0);
#pragma unroll 4
  for (int s = 0; s < p.splits; ++s) {
    const float ls = p.part_lse[(at + s * step) * 32 + lane % 32];
    if (ls == -INFINITY) continue;  // no key of this split: nothing was stored that may be read
    const float w = __builtin_amdgcn_exp2f(ls - top);
    total += w;
    const float4* po = (const float4*)p.part_o + (at + s * step) * (V / 8) * 64 + lane;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float4 v = po[(k0 + k) * 64];
      acc[k].x = __builtin_fmaf(w, v.x, acc[k].x);
      acc[k].y = __builtin_fmaf(w, v.y, acc[k].y);
      acc[k].z = __builtin_fmaf(w, v.z, acc[k].z);
      acc[k].w = __builtin_fmaf(w, v.w, acc[k].w);
    }
  }
  const float inv = total == 0.0f ? 0.0f : 1.0f / total;
  const int64_t token = seq.q0 + i;
  if (p.lse && blockIdx.y == 0 && lane < 32) p.lse[token * p.heads + head] = total == 0.0f ? -INFINITY : (top + log2f(total)) * kLn2;
  uint16_t* orow = p.out + token * p.ot + head * p.oh + 4 * (lane / 32);
#pragma unroll
  for (int k = 0; k < 4; ++k)
    *(uint2*)(orow + 8 * (k0 + k)) = make_uint2(pack_bf16(acc[k].x * inv, acc[k].y * inv), pack_bf16(acc[k].z * inv, acc[k].w * inv));
}

// Rows of a row block. 256 make two products of each K and V fragment read from
// LDS but leave a workgroup alone on its CU, with what comes before its first
// tile and behind its last in the open: it pays from some 16 tiles a row on
// average. The averages are over the batch: lengths are on the device, so one
// long prompt among many short ones takes the form that the short ones ask for.
// Measured wide against narrow, 128 + 64 / 128: 128 heads of 1500
// tokens 132 us, 129, of 2048 210, 225; 16 heads of 4 x 4096 188, 200; 160 tokens
// behind 8000, 128 heads, 191, 244; but 32 x 128 tokens, 128 heads, 167, 82.
int expanded_rows(const fcmoe_expanded_args* a) {
  const int64_t n = a->tokens / a->batch, keys = a->keys / a->batch;
  return n > 128 && keys - n / 2 >= 1024 ? kWideRows : kNarrowRows;
}

int64_t expanded_blocks(const fcmoe_expanded_args* a) {
  return a->tokens / expanded_rows(a) + (a->batch < a->tokens ? a->batch : a->tokens);
}

// Splits of the key axis: enough workgroups for one (256 rows) or two (128 rows)
// a CU where the row blocks alone are fewer, each with at least 4 tiles of an
// average sequence's keys. One token, 4 heads, us with 1, 4, 8, 16, 32 and 64 of
// them (*: taken): behind 1000 keys 28.5, 15.1*, 14.1, 16.1, 21.1, 29.2, behind
// 4000 97, 33, 23.1, 20.4*, 24.9, 39, behind 32000 735, 196, 106, 65, 51, 60*;
// 2 x 128 tokens, 32 heads behind 16000 387, 169*, 131, 153, 183, 253.
int expanded_splits(const fcmoe_expanded_args* a) {
  const int64_t items = expanded_blocks(a) * a->heads;
  if (items <= 0) return 1;
  const int64_t want = ceil_div(expanded_rows(a) == kWideRows ? 256 : 512, items);
  const int64_t most = ceil_div(ceil_div(a->keys, a->batch > 0 ? a->batch : 1), 4 * kExpKeys);
  int64_t s = want < most ? want : most;
  return (int)(s < 1 ? 1 : s > 64 ? 64 : s);
}

size_t expanded_part_lse_bytes(const fcmoe_expanded_args* a, int splits) {
  return (size_t)round_up((int64_t)splits * expanded_blocks(a) * a->heads * expanded_rows(a) * 4, 256);
}

template <int N, int P, int V>
void expanded_launch(const Expanded& p, hipStream_t stream) {
  const dim3 grid((unsigned)(p.blocks * p.heads * p.splits)), block(kExpWaves * kWave);
  if (p.rows == kWideRows)
    hipLaunchKernelGGL((expanded_wide_kernel<N, P, V>), grid, block, 0, stream, p);
  else
    hipLaunchKernelGGL((expanded_narrow_kernel<N, P, V>), grid, block, 0, stream, p);
  if (p.splits > 1)
    hipLaunchKernelGGL((expanded_combine_kernel<V>), dim3((unsigned)(p.blocks * p.heads * (p.rows / 32 / kExpWaves)), V / 32), block, 0,
                       stream, p);
}

}  // namespace

}  // namespace fcmoe

using namespace fcmoe;

extern "C" size_t fcmoe_expanded_attention_workspace_bytes(const fcmoe_expanded_args* a) {
  if (!a || a->tokens <= 0 || a->batch <= 0 || a->heads <= 0 || a->v_dim <= 0 || a->keys < 0) return 0;
  const int splits = expanded_splits(a);
  if (splits <= 1) return 0;
  return expanded_part_lse_bytes(a, splits) +
         (size_t)splits * (size_t)expanded_blocks(a) * (size_t)a->heads * (size_t)expanded_rows(a) * (size_t)a->v_dim * 4;
}

extern "C" int fcmoe_expanded_attention(const fcmoe_expanded_args* a, hipStream_t stream) {
  if (!a) return fail(FCMOE_EINVAL, "expanded_attention: NULL args");
  if (!((a->nope_dim == 128 && a->v_dim == 128) || (a->nope_dim == 64 && a->v_dim == 64)) ||
      (a->rope_dim != 0 && a->rope_dim != 64))
    return fail(FCMOE_EINVAL, "expanded_attention: key/value dims must be 128/128 or 64/64, rope_dim 0 or 64");
  if (a->tokens < 0 || a->tokens > INT32_MAX || a->keys < 0 || a->keys > INT32_MAX || a->batch <= 0 ||
      a->batch > (1 << 20) || a->heads <= 0 || a->heads > 65536)
    return fail(FCMOE_EINVAL, "expanded_attention: bad shape");
  if (!(a->scale > 0.0f) || !(a->scale < INFINITY))
    return fail(FCMOE_EINVAL, "expanded_attention: scale must be positive and finite");
  if (a->tokens == 0) return FCMOE_OK;
  if (!a->q || !a->query_starts || !a->kv_starts || !a->out || (a->keys > 0 && (!a->kv || (a->rope_dim && !a->k_rope))))
    return fail(FCMOE_EINVAL, "expanded_attention: NULL pointer");
  if (a->q_token_stride % 8 || a->q_head_stride % 8 || (uintptr_t)a->q % 16 || a->kv_token_stride % 8 ||
      a->kv_head_stride % 8 || (uintptr_t)a->kv % 16 || a->k_rope_token_stride % 8 || (uintptr_t)a->k_rope % 16)
    return fail(FCMOE_EINVAL, "expanded_attention: rows must start at multiples of 16 bytes");
  if (a->out_token_stride % 4 || a->out_head_stride % 4 || (uintptr_t)a->out % 8)
    return fail(FCMOE_EINVAL, "expanded_attention: out rows must start at multiples of 8 bytes");
  // a tile's 64 rows are addressed by 32-bit offsets from its first
  if (a->kv_token_stride < 0 || a->kv_token_stride >= (1 << 24) || a->k_rope_token_stride < 0 ||
      a->k_rope_token_stride >= (1 << 24))
    return fail(FCMOE_EINVAL, "expanded_attention: token strides must be below 2^24 values");
  Expanded p{};
  p.q = a->q, p.qt = a->q_token_stride, p.qh = a->q_head_stride;
  p.kv = a->kv, p.kt = a->kv_token_stride, p.kh = a->kv_head_stride;
  p.r = a->k_rope, p.rt = a->k_rope_token_stride;
  p.q_starts = a->query_starts, p.kv_starts = a->kv_starts;
  p.tokens = a->tokens, p.keys = a->keys;
  p.batch = (int)a->batch, p.heads = (int)a->heads, p.causal = a->causal;
  p.scale = a->scale;
  p.out = a->out, p.ot = a->out_token_stride, p.oh = a->out_head_stride, p.lse = a->lse;
  p.zero_tail = a->zero_uncovered;
  p.rows = expanded_rows(a);
  p.blocks = expanded_blocks(a);
  p.splits = expanded_splits(a);
  if (p.blocks * p.heads * p.splits > INT32_MAX) return fail(FCMOE_EINVAL, "expanded_attention: too many row blocks");
  if (p.splits > 1) {
    if (!a->workspace || a->workspace_bytes < fcmoe_expanded_attention_workspace_bytes(a))
      return fail(FCMOE_ESPACE, "expanded_attention: workspace too small");
    if ((uintptr_t)a->workspace % 16) return fail(FCMOE_EINVAL, "expanded_attention: unaligned workspace");
    p.part_lse = (float*)a->workspace;
    p.part_o = (float*)((char*)a->workspace + expanded_part_lse_bytes(a, p.splits));
  }
  if (a->nope_dim == 128 && a->rope_dim == 64)
    expanded_launch<128, 64, 128>(p, stream);
  else if (a->nope_dim == 128)
    expanded_launch<128, 0, 128>(p, stream);
  else if (a->rope_dim == 64)
    expanded_launch<64, 64, 64>(p, stream);
  else
    expanded_launch<64, 0, 64>(p, stream);
  return check_launch("expanded_attention");
}
