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
// One pass over the keys with the running maximum and sum of the softmax. A
// workgroup owns 128 query rows of one head, 32 a wave, and walks the keys in
// tiles of 64 through two LDS buffers filled straight from memory
// (global_load_lds) while the other buffer is computed. Products are S^T = K
// Q^T and O^T = V^T P^T (see fcmoe_latent.h): Q stays in registers, P never
// leaves them, and V^T comes from transposing LDS reads.
#include "fcmoe_internal.h"
#include "fcmoe_latent.h"

namespace fcmoe {

namespace {

constexpr int kExpWaves = 4;
constexpr int kExpRows = 32 * kExpWaves;  // query rows of a workgroup
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
  s.n = (int)(clamp64(p.q_starts[b + 1], s.q0, p.tokens) - s.q0);
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
__global__ __launch_bounds__(kExpWaves * kWave, 2) void expanded_kernel(const Expanded p) {
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
  const int64_t item = (int64_t)blockIdx.x % (p.blocks * p.heads);
  const int split = (int)((int64_t)blockIdx.x / (p.blocks * p.heads));
  const int head = (int)(item % p.heads);
  const int64_t block = p.blocks - 1 - item / p.heads;
  int64_t before;
  SeqSpan seq;
  const int b = find_sequence(
      p.batch, block, [&](int s) { return expanded_span(p, s); },
      [](const SeqSpan& s) { return ((int64_t)s.n + kExpRows - 1) / kExpRows; }, &seq, &before);
  if (b < 0) return;
  const int i0 = (int)(block - before) * kExpRows;
  const int wave_i0 = i0 + 32 * wave;
  const bool live = wave_i0 < seq.n;
  const int wave_i1 = min(wave_i0 + 31, seq.n - 1);
  const int lim_min = live ? expanded_limit(p, seq, wave_i0) : 0;
  const int lim_max = live ? expanded_limit(p, seq, wave_i1) : 0;
  const int my_i = min(wave_i0 + lane % 32, seq.n - 1);
  const int my_lim = expanded_limit(p, seq, my_i);

  const int tiles = (expanded_limit(p, seq, min(i0 + kExpRows, seq.n) - 1) + kExpKeys - 1) / kExpKeys;
  const int t_begin = (int)((int64_t)tiles * split / p.splits), t_end = (int)((int64_t)tiles * (split + 1) / p.splits);

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
    const int64_t at = ((int64_t)split * p.blocks * p.heads + item) * kExpWaves + wave;
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

// Joins the splits of a row block: out = sum_s 2^(lse_s - max) O_s / sum_s 2^(lse_s - max).
template <int V>
__global__ __launch_bounds__(kExpWaves * kWave) void expanded_combine_kernel(const Expanded p) {
  const int lane = (int)threadIdx.x % kWave, wave = (int)threadIdx.x / kWave;
  const int64_t item = (int64_t)blockIdx.x;
  const int head = (int)(item % p.heads);
  const int64_t block = p.blocks - 1 - item / p.heads;
  int64_t before;
  SeqSpan seq;
  const int b = find_sequence(
      p.batch, block, [&](int s) { return expanded_span(p, s); },
      [](const SeqSpan& s) { return ((int64_t)s.n + kExpRows - 1) / kExpRows; }, &seq, &before);
  if (b < 0) return;
  const int i = (int)(block - before) * kExpRows + 32 * wave + lane % 32;
  if (i >= seq.n) return;
  const int64_t step = p.blocks * p.heads * kExpWaves;
  const int64_t at = item * kExpWaves + wave;
  float top = -INFINITY;
  for (int s = 0; s < p.splits; ++s) top = fmaxf(top, p.part_lse[(at + s * step) * 32 + lane % 32]);
  float total = 0.0f;
  float4 acc[V / 8];
#pragma unroll
  for (int k = 0; k < V / 8; ++k) acc[k] = make_float4(0, 0, 0, 0);
  for (int s = 0; s < p.splits; ++s) {
    const float ls = p.part_lse[(at + s * step) * 32 + lane % 32];
    if (ls == -INFINITY) continue;  // no key of this split: nothing was stored that may be read
    const float w = __builtin_amdgcn_exp2f(ls - top);
    total += w;
    const float4* po = (const float4*)p.part_o + (at + s * step) * (V / 8) * 64 + lane;
#pragma unroll
    for (int k = 0; k < V / 8; ++k) {
      const float4 v = po[k * 64];
      acc[k].x = __builtin_fmaf(w, v.x, acc[k].x);
      acc[k].y = __builtin_fmaf(w, v.y, acc[k].y);
      acc[k].z = __builtin_fmaf(w, v.z, acc[k].z);
      acc[k].w = __builtin_fmaf(w, v.w, acc[k].w);
    }
  }
  const float inv = total == 0.0f ? 0.0f : 1.0f / total;
  const int64_t token = seq.q0 + i;
  if (p.lse && lane < 32) p.lse[token * p.heads + head] = total == 0.0f ? -INFINITY : (top + log2f(total)) * kLn2;
  uint16_t* orow = p.out + token * p.ot + head * p.oh + 4 * (lane / 32);
#pragma unroll
  for (int k = 0; k < V / 8; ++k)
    *(uint2*)(orow + 8 * k) = make_uint2(pack_bf16(acc[k].x * inv, acc[k].y * inv), pack_bf16(acc[k].z * inv, acc[k].w * inv));
}

int64_t expanded_blocks(const fcmoe_expanded_args* a) {
  return a->tokens / kExpRows + (a->batch < a->tokens ? a->batch : a->tokens);
}

// Splits of the key axis: enough workgroups for two a CU where the row blocks
// alone are fewer, each with at least 4 tiles of an average sequence's keys.
int expanded_splits(const fcmoe_expanded_args* a) {
  const int64_t items = expanded_blocks(a) * a->heads;
  if (items <= 0) return 1;
  const int64_t want = ceil_div(512, items);
  const int64_t most = ceil_div(ceil_div(a->keys, a->batch > 0 ? a->batch : 1), 4 * kExpKeys);
  int64_t s = want < most ? want : most;
  return (int)(s < 1 ? 1 : s > 64 ? 64 : s);
}

size_t expanded_part_lse_bytes(const fcmoe_expanded_args* a, int splits) {
  return (size_t)round_up((int64_t)splits * expanded_blocks(a) * a->heads * kExpRows * 4, 256);
}

template <int N, int P, int V>
void expanded_launch(const Expanded& p, hipStream_t stream) {
  hipLaunchKernelGGL((expanded_kernel<N, P, V>), dim3((unsigned)(p.blocks * p.heads * p.splits)),
                     dim3(kExpWaves * kWave), 0, stream, p);
  if (p.splits > 1)
    hipLaunchKernelGGL((expanded_combine_kernel<V>), dim3((unsigned)(p.blocks * p.heads)), dim3(kExpWaves * kWave), 0,
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
         (size_t)splits * (size_t)expanded_blocks(a) * (size_t)a->heads * kExpRows * (size_t)a->v_dim * 4;
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
