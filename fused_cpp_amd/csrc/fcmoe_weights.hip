// fcmoe_weights.hip -- what each cached token receives of the softmax weights
// of a call's query rows:
//
//   a_j = prev_j + sum over rows r that see j of exp(scale * q_r . k_j - lse_r)
//
// A row r is a (query token, head) pair with q_r = (ql_r, qr_r) and the log of its
// softmax's sum, which the attention call returns; k_j is the cached row. One
// pass over the cache, no running maximum. With few rows the cache's bytes
// bound it (2 (R + P) a row), with many the matrix units (2 (R + P) flops a
// pair).
//
// S^T = K Q^T by 16x16x32 products, keys in rows: a wave holds the fragments
// of its own 16 KT keys in registers, straight from memory (no other wave
// needs them, and a wave's waits are filled by the others), and walks the query
// rows, which lie in LDS in chunks of CH. A key's sum over rows is then a sum
// over a wave's lanes and chunks: no atomics, and an order that depends on
// nothing but the sizes.
//
// The blocks of 128 KT keys of all sequences are divided evenly among the
// workgroups. Where a sequence has many rows they are split too (`splits`), each
// split's sums left in the workspace for a second launch to add in order.
//
// 64 sequences of up to 8192, 16 heads 69 us, 4.5 TB/s; 32 tokens of 128 heads
// over 2 x 16384 170 us, 0.9 PFLOP/s (188 with each query fragment read where it
// is used and lse between the chunks).
#include "fcmoe_internal.h"
#include "fcmoe_latent.h"

namespace fcmoe {

namespace {

constexpr int kWtWaves = 8;

struct Weights {
  const uint16_t* ql;
  int64_t qlt, qlh;
  const uint16_t* qr;
  int64_t qrt, qrh;
  fcmoe_latent_cache c;
  const int32_t* table;
  int64_t width, table_stride;
  const int32_t* lens;
  const int32_t* q_starts;
  const float* lse;  // [tokens, heads]
  int64_t tokens;
  int batch, heads;
  float scale;
  const float* prev;
  int64_t prev_stride;
  float* out;
  int64_t out_stride;
  int64_t positions;  // of a sequence in out
  float* part;        // splits > 1: [splits][batch][positions]
  int splits, block;  // keys of a block
};

__device__ __forceinline__ SeqSpan weights_span(const Weights& p, int b) {
  SeqSpan s;
  if (p.q_starts) {
    s.q0 = clamp64(p.q_starts[b], 0, p.tokens);
    s.n = (int)(clamp64(p.q_starts[b + 1], 0, p.tokens) - s.q0);
  } else {
    s.q0 = b;
    s.n = b < p.tokens ? 1 : 0;
  }
  const int64_t reach = p.c.pages > 0 ? p.width * p.c.page_size : 0;
  s.k0 = 0;
  s.len = (int)clamp64(p.lens[b], 0, reach < INT32_MAX - 512 ? reach : INT32_MAX - 512);
  return s;
}
// Keys of a sequence that have a place in `out`.
__device__ __forceinline__ int weights_keys(const Weights& p, int len) { return (int)(len < p.positions ? len : p.positions); }

// LDS swizzles of the query rows, as the attention's bf16 key rows.
__device__ __forceinline__ int swz_row(int r) { return ((r & 3) << 1) | ((r >> 2) & 1) | (r & 8); }

template <int R, int P, bool F8, int KT, int CH>
__global__ __launch_bounds__(kWtWaves* kWave, KT == 1 ? 4 : 2) void weights_kernel(const Weights p) {
  constexpr int ELEM = F8 ? 1 : 2;
  constexpr int KS = (R + P) / 32, RS = R / 32, THREADS = kWtWaves * kWave;
  constexpr int LU = R / 8, RPW = CH / kWtWaves;  // 16-byte units of a query row's latent part; rows that a wave brings
  constexpr int MT = CH / 16, CHUNK = CH * 2 * (R + P);
  constexpr int BLOCK = kWtWaves * 16 * KT;
  __shared__ __align__(1024) uint8_t smem[2 * CHUNK];
  __shared__ float2 info[2][CH];  // a row's log2 of its sum, and the keys it sees as an integer (0: it has no weights)
  lds_u8* lds = (lds_u8*)smem;
  const int lane = (int)threadIdx.x % kWave, wave = wave_index();
  const int lq = lane / 16, lr = lane % 16;
  const float c2 = uniform(p.scale * kLog2e);

  auto blocks_of = [&](const SeqSpan& s) { return (weights_keys(p, s.len) + BLOCK - 1) / BLOCK; };
  auto count = [&](const SeqSpan& s) { return (int64_t)blocks_of(s) * p.splits; };
  auto span = [&](int b) { return weights_span(p, b); };

  // places that no block holds keep what they had
  if (!p.part && !(p.prev == p.out && p.prev_stride == p.out_stride)) {
    const int64_t pieces = (p.positions + 4095) / 4096;
    for (int64_t k = blockIdx.x; k < pieces * p.batch; k += gridDim.x) {
      const int b = (int)(k / pieces);
      const int64_t first = weights_keys(p, weights_span(p, b).len), j0 = k % pieces * 4096;
      const int64_t j1 = j0 + 4096 < p.positions ? j0 + 4096 : p.positions;
      for (int64_t j = (j0 > first ? j0 : first) + threadIdx.x; j < j1; j += THREADS)
        p.out[b * p.out_stride + j] = p.prev ? p.prev[b * p.prev_stride + j] : 0.0f;
    }
  }

  const int64_t units = count_items(p.batch, span, count);
  int64_t u = units * blockIdx.x / gridDim.x;
  const int64_t u_end = units * (blockIdx.x + 1) / gridDim.x;
  while (u < u_end) {
    SeqSpan seq;
    int64_t before;
    const int b = uniform(find_sequence(p.batch, u, span, count, &seq, &before));
    const int nb = blocks_of(seq), rel = (int)(u - before);
    const int split = uniform(rel / nb), kb0 = uniform(rel - split * nb);
    const int run = uniform((int)(nb - kb0 < u_end - u ? nb - kb0 : u_end - u));
    u += run;
    const int rows = seq.n * p.heads, chunks = (rows + CH - 1) / CH;
    const int c0 = (int)((int64_t)chunks * split / p.splits), c1 = (int)((int64_t)chunks * (split + 1) / p.splits);
    const int32_t* table = p.table + (int64_t)b * p.table_stride;

    // ---- a chunk of query rows to LDS: wave w brings rows RPW w .., the latent
    // parts straight from memory, the key parts (rows too short for a load
    // each) through a register
    v4i held{};
    float held_lse = 0.0f;
    auto take = [&](int chunk, int buf) {
      const int ln = lane_now();
      auto row_of = [&](int at, int& i, int& h) {
        const int row = min(chunk * CH + at, rows - 1);
        i = row / p.heads;
        h = row - i * p.heads;
      };
      int i, h;
      row_of(RPW * wave + ln % RPW, i, h);
      const uint64_t ql = (uint64_t)(p.ql + (seq.q0 + i) * p.qlt + h * p.qlh);
#pragma unroll
      for (int k = 0; k < RPW; ++k) {
        const __amdgpu_buffer_rsrc_t row = __builtin_amdgcn_make_buffer_rsrc((void*)lane_value(ql, k), (short)0, 2 * R, kBufWord3);
        const int at = RPW * wave + k;
        if (R == 512 || ln < LU) load_lds16(row, lds + buf * CHUNK + at * 2 * R, (uint32_t)(ln ^ swz_row(at)) * 16);
      }
      if constexpr (P > 0) {
        if (ln < 8 * RPW) {
          row_of(RPW * wave + ln / 8, i, h);
          held = *(const v4i*)(p.qr + (seq.q0 + i) * p.qrt + h * p.qrh + ln % 8 * 8);
        }
      }
      const int tid = kWave * wave + ln;
      if (tid < CH) {
        row_of(tid, i, h);
        held_lse = p.lse[(seq.q0 + i) * p.heads + h];
      }
    };
    auto place = [&](int chunk, int buf) {
      const int ln = lane_now();
      if constexpr (P > 0) {
        const int row = RPW * wave + ln / 8;
        if (ln < 8 * RPW)
          *(__attribute__((address_space(3))) v4i*)(lds + buf * CHUNK + CH * 2 * R + row * 2 * P + ((ln % 8) ^ (swz_row(row) & 7)) * 16) = held;
      }
      const int tid = kWave * wave + ln;
      if (tid < CH) {
        // a place without a row, or a row without a sum, sees no keys: its scores may then be anything, NaN as well
        const int row = chunk * CH + tid, i = min(row, rows - 1) / p.heads;
        const bool counts = row < rows && held_lse != -INFINITY;
        info[buf][tid] = make_float2(counts ? held_lse * kLog2e : 0.0f, __int_as_float(counts ? max(seq.len - seq.n + i + 1, 0) : 0));
      }
    };

    v8bf kf[KT][KS];
    float sc[KT][4], sum[KT][4];
    // ---- this wave's keys of block kb
    auto keys = [&](int kb) {
#pragma unroll
      for (int t = 0; t < KT; ++t) {
        const int key = min(kb * BLOCK + (wave * KT + t) * 16 + lr, seq.len - 1);
        const int page = key / (int)p.c.page_size, in = key - page * (int)p.c.page_size;
        int32_t id = table[page];
        const bool bad = (uint64_t)(int64_t)id >= (uint64_t)p.c.pages;
        if (bad) id = 0;
        const char* lat = (const char*)p.c.latent + (id * p.c.latent_page_stride + in * p.c.latent_row_stride) * ELEM + 16 * lq;
        const char* rope = P ? (const char*)p.c.rope + (id * p.c.rope_page_stride + in * p.c.rope_row_stride) * ELEM + 16 * lq : nullptr;
        float scale = 1.0f;
        if constexpr (F8) {
          // 16 bytes serve two steps: values 64 m + 16 (lane / 16) + 8 (step % 2) ..
          scale = p.c.scale[id * p.c.scale_page_stride + in];
          v4i raw[KS / 2];
#pragma unroll
          for (int m = 0; m < KS / 2; ++m) raw[m] = *(const v4i*)(m < RS / 2 ? lat + 64 * m : rope + 64 * (m - RS / 2));
#pragma unroll
          for (int m = 0; m < KS / 2; ++m) {
            kf[t][2 * m] = widen_e4m3(v2i{raw[m][0], raw[m][1]});
            kf[t][2 * m + 1] = widen_e4m3(v2i{raw[m][2], raw[m][3]});
          }
        } else {
#pragma unroll
          for (int ks = 0; ks < KS; ++ks) kf[t][ks] = *(const v8bf*)(ks < RS ? lat + 64 * ks : rope + 64 * (ks - RS));
        }
        if (bad) kf[t][0][0] = __builtin_bit_cast(__bf16, (uint16_t)0x7fc0);  // its weights become NaN
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          sc[t][i] = F8 ? __shfl(scale, 4 * lq + i) : 1.0f;
          sum[t][i] = 0.0f;
        }
      }
    };
    auto compute = [&](int kb, int buf) {
      // a fragment's address: unit 4 k + lane / 16 of the row (8-bit keys: 8 (k / 2) + 2 (lane / 16) + k % 2), formed from
      // the lane here and by an XOR a step, or addresses for every step would be kept
      const int ln = lane_now(), cq = ln / 16, cr = ln % 16;
      const lds_u8* base = lds + buf * CHUNK;
      const int la = cr * 2 * R + (((F8 ? 2 * cq : cq) ^ swz_row(cr)) * 16);
      const int ra = CH * 2 * R + cr * 2 * P + (((F8 ? 2 * cq : cq) ^ (swz_row(cr) & 7)) * 16);
      auto q_at = [&](int ks) {
        if (ks >= RS) return ra ^ (F8 ? (ks - RS) << 4 : (ks - RS) << 6);
        return F8 ? (la ^ ((ks & 1) << 4 | (ks >> 1 & 1) << 7)) + (ks >> 2) * 256 : (la ^ ((ks & 3) << 6)) + (ks >> 2) * 256;
      };
      v4f s[MT][KT];
#pragma unroll
      for (int r = 0; r < MT; ++r)
#pragma unroll
        for (int t = 0; t < KT; ++t) s[r][t] = v4f{0, 0, 0, 0};
      // Query fragments are read AHEAD uses ahead, in a pinned order: left to itself the compiler reads each where it is used,
      // and every one waits out the LDS latency.
      constexpr int READS = KS * MT, AHEAD = KT == 1 ? 1 : 4, RING = AHEAD + 1;
      v8bf q[RING];
      auto read = [&](int n) {
        const int ks = n / MT, r = n % MT;
        q[n % RING] = *(const __attribute__((address_space(3))) v8bf*)(base + q_at(ks) + 16 * r * (ks < RS ? 2 * R : 2 * P));
      };
#pragma unroll
      for (int n = 0; n < AHEAD; ++n) read(n);
#pragma unroll
      for (int n = 0; n < READS; ++n) {
        if (n + AHEAD < READS) read(n + AHEAD);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int t = 0; t < KT; ++t)
          s[n % MT][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf[t][n / MT], q[n % RING], s[n % MT][t], 0, 0, 0);
        __builtin_amdgcn_sched_barrier(0);
      }
#pragma unroll
      for (int r = 0; r < MT; ++r) {
        const float2 in = info[buf][16 * r + cr];
#pragma unroll
        for (int t = 0; t < KT; ++t) {
          const int left = __float_as_int(in.y) - (kb * BLOCK + (wave * KT + t) * 16 + 4 * cq);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(F8 ? s[r][t][i] * sc[t][i] : s[r][t][i], c2, -in.x));
            sum[t][i] += i < left ? e : 0.0f;
          }
        }
      }
    };
    // Lane 4 t + i of each 16 has key i of its four in tile t.
    auto store = [&](int kb) {
      float mine = 0.0f;
#pragma unroll
      for (int t = 0; t < KT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float v = sum[t][i];
#pragma unroll
          for (int o = 1; o < 16; o <<= 1) v += __shfl_xor(v, o);
          mine = lr == 4 * t + i ? v : mine;
        }
      const int key = kb * BLOCK + (wave * KT + lr / 4) * 16 + 4 * lq + lr % 4;
      if (lr >= 4 * KT || key >= weights_keys(p, seq.len)) return;
      if (p.part)
        p.part[((int64_t)split * p.batch + b) * p.positions + key] = mine;
      else
        p.out[b * p.out_stride + key] = (p.prev ? p.prev[b * p.prev_stride + key] : 0.0f) + mine;
    };

    if (c1 - c0 <= 2) {  // the rows stay in LDS for all of these blocks
      lds_only_barrier();
      for (int c = c0; c < c1; ++c) {
        take(c, c - c0);
        place(c, c - c0);
      }
      loads_barrier();
      for (int kb = kb0; kb < kb0 + run; ++kb) {
        keys(kb);
        for (int c = c0; c < c1; ++c) compute(kb, c - c0);
        store(kb);
      }
    } else {
      for (int kb = kb0; kb < kb0 + run; ++kb) {
        lds_only_barrier();
        take(c0, 0);
        place(c0, 0);
        keys(kb);
        for (int c = c0; c < c1; ++c) {
          const int buf = (c - c0) & 1;
          loads_barrier();  // chunk c has landed; everyone is done with the other buffer
          if (c + 1 < c1) take(c + 1, buf ^ 1);
          compute(kb, buf);
          if (c + 1 < c1) place(c + 1, buf ^ 1);
        }
        store(kb);
      }
    }
  }
}

// The splits' sums, in their order.
__global__ __launch_bounds__(256) void weights_join_kernel(const Weights p) {
  const int64_t j = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int b = (int)blockIdx.y;
  if (j >= p.positions) return;
  float v = p.prev ? p.prev[b * p.prev_stride + j] : 0.0f;
  if (j < weights_span(p, b).len) {
    float s = 0.0f;
    for (int k = 0; k < p.splits; ++k) s += p.part[((int64_t)k * p.batch + b) * p.positions + j];
    v += s;
  }
  p.out[b * p.out_stride + j] = v;
}

struct WeightsPlan {
  bool few;  // rows of a sequence: keys in blocks of 128, two workgroups a CU
  int splits;
  int64_t wgs;
  size_t bytes;
};

// Times in us, 16-bit and 8-bit rows. Rows of a sequence: blocks of 128 keys, two workgroups a CU, against 256, one: 64
// sequences of up to 8192, 24 rows 61 and 40, 75 and 51; 32 rows 61 and 40, 74 and 52; 48 rows 65 and 47, 75 and 52; 64 rows
// 65 and 46, 75 and 53; one of 131072, 64 rows 36 and 27, 36 and 29: a line at 64 would do better than this one at 32.
// Splits, a quarter of the chunks of 64 rows and 8 at most, against none: 64 tokens of 16 heads over one of 16384 33 and 29,
// 71 and 67; 256 tokens of 16 heads, 8 of 2048, 105 and 96, 272 and 271; 32 tokens of 128 heads over 2 of 16384 182 and 162,
// 262 and 237, over one of 300 46 and 43, 240 and 239. They do not look at the blocks there are: 16 tokens of 128 heads over
// 32 of 4096 take 473 and 386 for 316 and 303, 4 tokens of 128 heads over one of 131072 116 and 99 for 100 and 88. A
// sequence's own rows do not count either, the mean does: 512 tokens of 16 heads among 63 sequences of one, 8192 long, are
// one split's few blocks of a few workgroups and take 3800, 30 times what the bytes do.
WeightsPlan weights_plan(const fcmoe_attention_weights_args* a) {
  WeightsPlan pl{};
  const int64_t rows = ceil_div(a->tokens, a->batch) * a->heads;
  pl.few = rows <= 32;
  const int64_t chunks = ceil_div(rows, 64);
  pl.splits = pl.few || chunks <= 4 ? 1 : (int)(chunks / 4 < 8 ? chunks / 4 : 8);
  int dev = 0, cus = 256;
  if (hipGetDevice(&dev) != hipSuccess || hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess)
    (void)hipGetLastError();
  const int64_t reach = a->table_width * a->cache.page_size;
  const int64_t most = a->batch * pl.splits * ceil_div(reach < a->positions ? reach : a->positions, pl.few ? 128 : 256);
  const int64_t slots = (int64_t)cus * (pl.few ? 2 : 1);
  pl.wgs = most < slots ? (most > 0 ? most : 1) : slots;
  pl.bytes = pl.splits > 1 ? (size_t)pl.splits * (size_t)a->batch * (size_t)a->positions * 4 : 0;
  return pl;
}

template <int R, int P, bool F8>
void weights_launch(const Weights& p, const WeightsPlan& pl, hipStream_t stream) {
  const dim3 g((unsigned)pl.wgs), b(kWtWaves * kWave);
  if (pl.few)
    hipLaunchKernelGGL((weights_kernel<R, P, F8, 1, 32>), g, b, 0, stream, p);
  else
    hipLaunchKernelGGL((weights_kernel<R, P, F8, 2, 64>), g, b, 0, stream, p);
  if (p.splits > 1)
    hipLaunchKernelGGL(weights_join_kernel, dim3((unsigned)ceil_div(p.positions, 256), (unsigned)p.batch), dim3(256), 0, stream, p);
}

int check_weights(const fcmoe_attention_weights_args* a) {
  if (!a) return fail(FCMOE_EINVAL, "attention_weights: NULL args");
  if (const int rc = check_latent_cache(a->cache, "attention_weights")) return rc;
  if (a->tokens < 0 || a->tokens > INT32_MAX || a->batch <= 0 || a->batch > 65535 || a->heads <= 0 || a->heads > 65536 ||
      a->tokens * a->heads > INT32_MAX / 2 || a->table_width < 0 || a->table_width > INT32_MAX || a->page_table_stride < 0 ||
      a->positions < 0 || a->positions > INT32_MAX - 512)
    return fail(FCMOE_EINVAL, "attention_weights: bad shape");
  if (!a->query_starts && a->tokens != a->batch)
    return fail(FCMOE_EINVAL, "attention_weights: without query_starts there is one token a sequence");
  return FCMOE_OK;
}

}  // namespace

}  // namespace fcmoe

using namespace fcmoe;

extern "C" size_t fcmoe_attention_weights_workspace_bytes(const fcmoe_attention_weights_args* a) {
  return check_weights(a) == FCMOE_OK ? weights_plan(a).bytes : 0;
}

extern "C" int fcmoe_attention_weights(const fcmoe_attention_weights_args* a, hipStream_t stream) {
  if (const int rc = check_weights(a)) return rc;
  if (!(a->scale > 0.0f) || !(a->scale < INFINITY))
    return fail(FCMOE_EINVAL, "attention_weights: scale must be positive and finite");
  if (a->positions == 0) return FCMOE_OK;
  if (!a->out || !a->kv_lens || (a->table_width > 0 && !a->page_table) ||
      (a->tokens > 0 && (!a->q_latent || (a->cache.rope_dim && !a->q_rope) || !a->lse)))
    return fail(FCMOE_EINVAL, "attention_weights: NULL pointer");
  if (a->q_latent_token_stride % 8 || a->q_latent_head_stride % 8 || (uintptr_t)a->q_latent % 16 ||
      a->q_rope_token_stride % 8 || a->q_rope_head_stride % 8 || (uintptr_t)a->q_rope % 16)
    return fail(FCMOE_EINVAL, "attention_weights: query rows must start at multiples of 16 bytes");
  const WeightsPlan pl = weights_plan(a);
  if (pl.bytes && (!a->workspace || a->workspace_bytes < pl.bytes)) return fail(FCMOE_ESPACE, "attention_weights: workspace too small");
  if ((uintptr_t)a->workspace % 16) return fail(FCMOE_EINVAL, "attention_weights: unaligned workspace");
  Weights p{};
  p.ql = a->q_latent, p.qlt = a->q_latent_token_stride, p.qlh = a->q_latent_head_stride;
  p.qr = a->q_rope, p.qrt = a->q_rope_token_stride, p.qrh = a->q_rope_head_stride;
  p.c = a->cache;
  p.table = a->page_table, p.width = a->table_width, p.table_stride = a->page_table_stride;
  p.lens = a->kv_lens, p.q_starts = a->query_starts, p.lse = a->lse;
  p.tokens = a->tokens, p.batch = (int)a->batch, p.heads = (int)a->heads, p.scale = a->scale;
  p.prev = a->previous, p.prev_stride = a->previous_stride;
  p.out = a->out, p.out_stride = a->out_stride, p.positions = a->positions;
  p.splits = pl.splits;
  p.part = pl.splits > 1 ? (float*)a->workspace : nullptr;
  const bool f8 = a->cache.e4m3 != 0;
  if (a->cache.latent_dim == 512) {
    if (a->cache.rope_dim == 64)
      f8 ? weights_launch<512, 64, true>(p, pl, stream) : weights_launch<512, 64, false>(p, pl, stream);
    else
      f8 ? weights_launch<512, 0, true>(p, pl, stream) : weights_launch<512, 0, false>(p, pl, stream);
  } else {
    if (a->cache.rope_dim == 64)
      f8 ? weights_launch<256, 64, true>(p, pl, stream) : weights_launch<256, 64, false>(p, pl, stream);
    else
      f8 ? weights_launch<256, 0, true>(p, pl, stream) : weights_launch<256, 0, false>(p, pl, stream);
  }
  return check_launch("attention_weights");
}
