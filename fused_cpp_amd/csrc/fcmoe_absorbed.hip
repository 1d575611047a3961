// fcmoe_absorbed.hip -- latent attention in its absorbed form over a paged
// cache: all heads of a sequence attend to the same latent rows.
//
//   s_rj = scale * (ql_r . c_j + qr_r . k_j),  out_r = sum_j softmax_j(s_rj) c_j
//
// A row r is a (query token, head) pair; the n * heads rows of a sequence
// share its cached rows (c_j: latent, R values; k_j: rotated key part, P), so
// a cached row is read once for up to 128 of them. With few rows the bound is
// the cache's bytes; with 128 heads a row brings 2 * 128 * (2 R + P) flops to
// 2 (R + P) bytes, 242 a byte, and the matrix units and LDS bound it.
//
// Work split. The keys of a sequence go in tiles of 64; a unit is one tile for
// one group of rows. The units of the whole batch, in order, are divided
// evenly among the workgroups (a few per CU at most), whatever the lengths:
// a workgroup walks a contiguous range of units, and where a row group's keys
// end up with several workgroups each leaves a partial result (normalised O,
// log2-sum-exp) that a second launch joins. Lengths are read on the device, so
// a captured launch serves any lengths.
//
// Products are S^T = K Q^T and O^T = V^T P^T (fcmoe_latent.h). V = c: one LDS
// copy of a tile serves both, read along d for S^T and through transposing
// reads along the keys for O^T.
#include "fcmoe_internal.h"
#include "fcmoe_latent.h"

namespace fcmoe {

namespace {

constexpr int kAbsKeys = 64;  // keys of a tile

struct Absorbed {
  const uint16_t* ql;
  int64_t qlt, qlh;
  const uint16_t* qr;
  int64_t qrt, qrh;
  fcmoe_latent_cache c;
  const int32_t* table;
  int64_t width, table_stride;
  const int32_t* lens;
  const int32_t* q_starts;
  int64_t tokens;
  int batch, heads;
  float scale;
  uint16_t* out;
  int64_t ot, oh;
  float* lse;
  float* part_o;    // [2 * shares slots][rows * R]
  float* part_lse;  // [2 * shares slots][rows], base 2
  int shares;
  int zero_tail;
};

__device__ __forceinline__ SeqSpan absorbed_span(const Absorbed& p, int b) {
  SeqSpan s;
  if (p.q_starts) {
    s.q0 = clamp64(p.q_starts[b], 0, p.tokens);
    s.n = (int)(clamp64(p.q_starts[b + 1], s.q0, p.tokens) - s.q0);
  } else {
    s.q0 = b;
    s.n = b < p.tokens ? 1 : 0;
  }
  const int64_t reach = p.c.pages > 0 ? p.width * p.c.page_size : 0;
  s.k0 = 0;
  s.len = (int)clamp64(p.lens[b], 0, reach < INT32_MAX - 128 ? reach : INT32_MAX - 128);
  return s;
}

__device__ __forceinline__ int row_groups(const Absorbed& p, const SeqSpan& s, int rows) {
  return (int)(((int64_t)s.n * p.heads + rows - 1) / rows);
}
// Tiles of a row group; at least one, so that a sequence without keys still gets its rows written.
__device__ __forceinline__ int key_tiles(const SeqSpan& s) { return s.len > 0 ? (s.len + kAbsKeys - 1) / kAbsKeys : 1; }

__device__ __forceinline__ int absorbed_limit(const SeqSpan& s, int i) {
  const int v = s.len - s.n + i + 1;
  return v < 0 ? 0 : v > s.len ? s.len : v;
}

// Units of the batch (every lane of a wave takes part).
__device__ __forceinline__ int64_t total_units(const Absorbed& p, int rows) {
  int64_t sum = 0;
  for (int b = (int)threadIdx.x % kWave; b < p.batch; b += kWave) {
    const SeqSpan s = absorbed_span(p, b);
    sum += (int64_t)row_groups(p, s, rows) * key_tiles(s);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
  return sum;
}

__device__ __forceinline__ int64_t share_begin(int64_t units, int64_t g, int64_t wgs) { return units * g / wgs; }
// The workgroup whose share holds unit u.
__device__ __forceinline__ int64_t share_of(int64_t units, int64_t u, int64_t wgs) {
  return ((u + 1) * wgs + units - 1) / units - 1;
}

// One range of key tiles of one row group.
struct Segment {
  SeqSpan seq;
  int b;
  int64_t row0;         // first row of the group
  int t_begin, t_end;   // tiles
  bool whole;           // all tiles of the group
  int64_t slot;         // partial slot otherwise
};

// The segment that starts at unit u of workgroup g's share [u, u1).
__device__ __forceinline__ Segment next_segment(const Absorbed& p, int rows, int64_t u, int64_t u1, int64_t g) {
  Segment s;
  int64_t before;
  s.b = find_sequence(
      p.batch, u,
      [&](int b) {
        const SeqSpan q = absorbed_span(p, b);
        return (int64_t)row_groups(p, q, rows) * key_tiles(q);
      },
      &before);
  s.b = __builtin_amdgcn_readfirstlane(s.b);
  s.seq = absorbed_span(p, s.b);
  const int tiles = key_tiles(s.seq);
  const int64_t rel = u - before;
  const int64_t group = rel / tiles;
  s.t_begin = __builtin_amdgcn_readfirstlane((int)(rel - group * tiles));
  const int64_t end = before + (group + 1) * tiles;
  s.t_end = __builtin_amdgcn_readfirstlane(s.t_begin + (int)((end < u1 ? end : u1) - u));
  s.row0 = (int64_t)__builtin_amdgcn_readfirstlane((int)(group * rows));
  s.whole = s.t_begin == 0 && s.t_end == tiles;
  // of a share's segments only the first can start inside a group's tiles and
  // only the last can end inside them: two slots a workgroup
  s.slot = 2 * g + (s.t_begin == 0 ? 1 : 0);
  return s;
}

// LDS swizzles: 16-byte unit u of key row k is stored at u ^ swz(k). bf16 rows
// as in the expanded form; 8-bit rows are read by 8 keys x 16 bytes blocks,
// keys 4 h + (0..3) and 8 + 4 h + (0..3) of a step, and by 8 neighbouring
// keys: both sets map to 8 different values.
template <bool F8>
__device__ __forceinline__ int swz_key(int key) {
  return F8 ? (key & 3) | ((((key >> 2) ^ (key >> 3)) & 1) << 2) : ((key & 3) << 1) | ((key >> 2) & 1) | (key & 8);
}
// The shared key part's rows: 8 units of bf16, 4 of 8-bit values.
template <bool F8>
__device__ __forceinline__ int swz_rope(int key) {
  return F8 ? (key >> 1) & 3 : swz_key<false>(key) & 7;
}

template <int R, int P, bool F8>
struct Tile {
  static constexpr int ELEM = F8 ? 1 : 2;
  static constexpr int LROW = R * ELEM, RROW = P * ELEM;  // bytes of a latent row, of a key-part row
  static constexpr int ROPE = kAbsKeys * LROW;            // key-part rows follow the latent rows
  static constexpr int BYTES = ROPE + kAbsKeys * RROW;
  static constexpr int UNITS = LROW / 16, RUNITS = P > 0 ? RROW / 16 : 1;
  static constexpr int LLOADS = 16 * LROW / 1024;         // 1 KB loads of a wave's 16 keys
  static constexpr int RLOADS = 16 * RROW / 1024;
};

// A value the compiler cannot see through: what depends on it is formed after this point.
__device__ __forceinline__ int opaque(int v) {
  asm volatile("" : "+v"(v));
  return v;
}

// Lane l's value, in scalar registers (l the same for the whole wave).
__device__ __forceinline__ uint64_t lane_value(uint64_t v, int l) {
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, l);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), l);
  return ((uint64_t)hi << 32) | lo;
}

// Brings a wave's 16 keys of a tile into LDS. Lane l knows the cached row of
// the wave's key l % 16: its page id is read one tile ahead (fetch), so that
// the rows' addresses are there when the buffer is free.
template <int R, int P, bool F8>
struct Stager {
  using T = Tile<R, P, F8>;
  const int32_t* table;
  int lane, wave, key_in, last_key;  // key_in: the lane's key of a tile; last_key: of the sequence
  int page_size;
  int32_t id;
  int in;
  bool bad;

  __device__ __forceinline__ void begin(const Absorbed& p, const SeqSpan& s, int b) {
    lane = (int)threadIdx.x % kWave;
    wave = (int)threadIdx.x / kWave;
    key_in = 16 * wave + lane % 16;
    table = p.table + (int64_t)b * p.table_stride;
    page_size = (int)p.c.page_size;
    last_key = s.len - 1;
    bad = false;
  }
  __device__ __forceinline__ void fetch(int tile) {
    int key = tile * kAbsKeys + key_in;
    key = key < last_key ? key : last_key;  // keys past the length re-read its last one; their scores are masked
    const int page = (int)((uint32_t)key / (uint32_t)page_size);
    in = key - page * page_size;
    id = table[page];
  }
  // scl: LDS, 64 scales of the buffer (8-bit rows).
  __device__ __forceinline__ void issue(const Absorbed& p, lds_u8* dst, lds_u8* scl) {
    int64_t page = id;
    if ((uint64_t)page >= (uint64_t)p.c.pages) {
      page = 0;
      bad = true;
    }
    const char* lat = (const char*)p.c.latent + (page * p.c.latent_page_stride + in * p.c.latent_row_stride) * T::ELEM;
    // Lane-dependent parts are formed here, load by load: kept across the tile
    // loop, or all at once, they would take the registers that Q and O need.
    const int ln = opaque(lane);
#pragma unroll
    for (int u = 0; u < T::LLOADS; ++u) {
      lds_u8* to = dst + wave * (16 * T::LROW) + u * 1024;
      if constexpr (T::UNITS == 64) {  // one key a load: its address is the same for the whole wave
        load_lds16((const char*)lane_value((uint64_t)lat, u) + ((ln * 16) ^ (swz_key<F8>(u) * 16)), to);
      } else {
        constexpr int LKEYS = 1024 / T::LROW;
        const int k = u * LKEYS + ln / T::UNITS;
        load_lds16((const char*)__shfl((long long)lat, k) + ((ln % T::UNITS) ^ swz_key<F8>(k)) * 16, to);
      }
      if (u % 2 == 1) __builtin_amdgcn_sched_barrier(0);
    }
    if constexpr (P > 0) {
      const char* rope = (const char*)p.c.rope + (page * p.c.rope_page_stride + in * p.c.rope_row_stride) * T::ELEM;
      constexpr int RKEYS = 1024 / T::RROW;
#pragma unroll
      for (int u = 0; u < T::RLOADS; ++u) {
        const int k = u * RKEYS + ln / T::RUNITS;
        load_lds16((const char*)__shfl((long long)rope, k) + ((ln % T::RUNITS) ^ swz_rope<F8>(k)) * 16,
                   dst + T::ROPE + wave * (16 * T::RROW) + u * 1024);
      }
    }
    if constexpr (F8) {
      const float* s = p.c.scale + page * p.c.scale_page_stride + in;
      if (lane < 16)
        __builtin_amdgcn_global_load_lds((__attribute__((address_space(1))) void*)s,
                                         (__attribute__((address_space(3))) void*)(scl + wave * 64), 4, 0, 0);
    }
  }
};

__device__ __forceinline__ v8bf lds_v8bf(const lds_u8* p) { return *(const __attribute__((address_space(3))) v8bf*)p; }
__device__ __forceinline__ v4i lds_v4i(const lds_u8* p) { return *(const __attribute__((address_space(3))) v4i*)p; }
__device__ __forceinline__ v4f lds_v4f(const lds_u8* p) { return *(const __attribute__((address_space(3))) v4f*)p; }

// ---- the attention kernel ------------------------------------------------------
//
// A workgroup takes 16 NR rows (16, 32 or 64); its four waves split each tile:
// for S^T every wave takes 16 of the 64 keys, for O^T a quarter of the latent
// dimension, both for all rows. So K and V are read from LDS once a workgroup
// however many rows there are (with waves split by rows they are read once a
// wave, and LDS, not the matrix units, bounds 64 rows and more), and a
// fragment feeds NR MFMAs. Q (R + P values of every row) and a quarter of O
// stay in registers: 18 x 4 x NR + 8 x 4 x NR at 512 + 64, all of a SIMD's at
// NR = 4. The row maxima and P go through LDS between the waves.
//
// PAIR: the rows of a sequence fill two workgroups (65 rows and more); these
// two take the same tiles at the same time on the same XCD, whose L2 then
// brings a cached row from memory once for both.
template <int R, int P, bool F8, int NR, int PAIR>
__global__ __launch_bounds__(256, F8&& NR == 1 ? 2 : 1) void absorbed_kernel(const Absorbed p) {
  using T = Tile<R, P, F8>;
  constexpr int ROWS = 16 * NR;       // of this workgroup
  constexpr int GROUP = ROWS * PAIR;  // of the row group that its pair shares
  constexpr int KS = (R + P) / 32, RS = R / 32, DT = R / 64;  // 16x16x32 steps; d tiles of a wave
  constexpr int PROW = 2 * kAbsKeys + 16;                      // bytes of a P row, padded off the banks' period
  constexpr int SCL = 2 * T::BYTES, PBUF = SCL + (F8 ? 2 * 256 : 0), MAXB = PBUF + ROWS * PROW, FLAG = MAXB + 4 * ROWS * 4;
  __shared__ __align__(1024) uint8_t smem[FLAG + 16];
  lds_u8* lds = (lds_u8*)smem;
  const int lane = (int)threadIdx.x % kWave, wave = (int)threadIdx.x / kWave;
  const int q4 = lane / 16, c16 = lane % 16;
  if (p.zero_tail)
    zero_uncovered(p.q_starts, p.batch, p.tokens, p.heads, R, p.out, p.ot, p.oh, p.lse, blockIdx.x, gridDim.x);

  const int64_t units = total_units(p, GROUP);
  const int64_t wgs = units < p.shares ? units : p.shares;
  // workgroups go to the 8 XCDs by blockIdx % 8: a pair's two are 8 apart
  const int member = PAIR == 2 ? (int)(blockIdx.x / 8 % 2) : 0;
  const int64_t g = PAIR == 2 ? blockIdx.x / 16 * 8 + blockIdx.x % 8 : blockIdx.x;
  if (g >= wgs) return;
  int64_t u = share_begin(units, g, wgs);
  const int64_t u1 = share_begin(units, g + 1, wgs);

  // K reads: key krow, unit 4 j + q4 of a window of units that the swizzle
  // stays in (16 units, 8 of an 8-bit row); the key part has one window.
  const int krow = 16 * wave + c16;
  int ka0 = krow * T::LROW + ((q4 ^ swz_key<F8>(krow)) * 16);
  int kra0 = T::ROPE + krow * T::RROW + ((q4 ^ swz_rope<F8>(krow)) * 16);
  // V^T reads: this lane's place in its group's block of keys 8 q4 .. 8 q4 + 7;
  // unit u0 of the wave's quarter, whose other units differ from it in address
  // bits that neither the key nor the lane touches
  const int vkey = F8 ? 8 * q4 + c16 / 2 : 8 * q4 + c16 / 4;
  const int u0 = F8 ? wave * DT : 2 * wave * DT + (c16 % 4) / 2;
  int va0 = vkey * T::LROW + ((u0 ^ swz_key<F8>(vkey)) * 16) + (lane & 1) * 8;
  const float c2 = p.scale * kLog2e;

  while (u < u1) {
    const Segment sg = next_segment(p, GROUP, u, u1, g);
    u += sg.t_end - sg.t_begin;
    const SeqSpan& seq = sg.seq;
    const int64_t rows = (int64_t)seq.n * p.heads;
    const int64_t row0 = sg.row0 + member * ROWS;
    if (PAIR == 2 && row0 >= rows) continue;  // the group's rows end with the other workgroup
    // query token and head of this lane's row of row tile r (rows past the last repeat it and are not stored)
    auto my_row = [&](int r, int& i, int& h) {
      int row = (int)row0 + 16 * r + opaque(c16);
      row = row < (int)rows ? row : (int)rows - 1;
      i = row / p.heads;
      h = row - i * p.heads;
    };
    const int lim_min = absorbed_limit(seq, (int)row0 / p.heads);

    Stager<R, P, F8> st;
    st.begin(p, seq, sg.b);
    __syncthreads();
    if (threadIdx.x == 0) *(__attribute__((address_space(3))) int*)(lds + FLAG) = 0;
    const bool any = seq.len > 0;
    if (any) {
      st.fetch(sg.t_begin);
      st.issue(p, lds, lds + SCL);
      if (sg.t_begin + 1 < sg.t_end) st.fetch(sg.t_begin + 1);
    }
    // Q: B operand. bf16 rows: values 32 ks + 8 q4 ..; 8-bit rows: 64 (ks / 2) + 16 q4 + 8 (ks % 2) ..
    v8bf qf[NR][KS];
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      int i, h;
      my_row(r, i, h);
      const uint16_t* ql = p.ql + (seq.q0 + i) * p.qlt + h * p.qlh;
      const uint16_t* qr = P ? p.qr + (seq.q0 + i) * p.qrt + h * p.qrh : nullptr;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const int k = ks < RS ? ks : ks - RS;
        const int d = F8 ? 64 * (k / 2) + 16 * q4 + 8 * (k % 2) : 32 * k + 8 * q4;
        qf[r][ks] = *(const v8bf*)((ks < RS ? ql : qr) + d);
      }
    }
    float m[NR], l[NR];
    v4f o[NR][DT];
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      m[r] = -INFINITY;
      l[r] = 0.0f;
#pragma unroll
      for (int t = 0; t < DT; ++t) o[r][t] = v4f{0, 0, 0, 0};
    }

    for (int tile = sg.t_begin; any && tile < sg.t_end; ++tile) {
      const int buf = (tile - sg.t_begin) & 1;
      loads_barrier();
      if (tile + 1 < sg.t_end) {
        st.issue(p, lds + (buf ^ 1) * T::BYTES, lds + SCL + (buf ^ 1) * 256);
        if (tile + 2 < sg.t_end) st.fetch(tile + 2);
      }
      const lds_u8* kb = lds + buf * T::BYTES;
      // the addresses below are formed where they are used, an XOR each: hoisted out of the loop they would
      // take the registers that Q and O need
      const int ka = opaque(ka0), kra = opaque(kra0), va = opaque(va0);
      v4f s[NR];
#pragma unroll
      for (int r = 0; r < NR; ++r) s[r] = v4f{0, 0, 0, 0};
      if constexpr (F8) {
#pragma unroll
        for (int kk = 0; kk < KS / 2; ++kk) {
          const int at = kk < RS / 2 ? (ka ^ ((kk & 1) << 6)) + (kk >> 1) * 128 : kra;
          const v4i w = lds_v4i(kb + at);
          const v8bf a0 = widen_e4m3(v2i{w[0], w[1]}), a1 = widen_e4m3(v2i{w[2], w[3]});
#pragma unroll
          for (int r = 0; r < NR; ++r) {
            s[r] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a0, qf[r][2 * kk], s[r], 0, 0, 0);
            s[r] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a1, qf[r][2 * kk + 1], s[r], 0, 0, 0);
          }
        }
      } else {
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          const int at = ks < RS ? (ka ^ ((ks & 3) << 6)) + (ks >> 2) * 256 : kra ^ ((ks - RS) << 6);
          const v8bf a = lds_v8bf(kb + at);
#pragma unroll
          for (int r = 0; r < NR; ++r) s[r] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, qf[r][ks], s[r], 0, 0, 0);
        }
        if constexpr (NR == 4) {
          __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
#pragma unroll
          for (int ks = 0; ks < KS; ++ks) {
            __builtin_amdgcn_sched_group_barrier(0x008, NR, 0);
            if (ks + 4 < KS) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
          }
        }
      }
      // lane: row c16 of each row tile, keys 16 wave + 4 q4 + i
      if constexpr (F8) {
        const v4f sc = lds_v4f(lds + SCL + buf * 256 + (16 * wave + 4 * q4) * 4);
#pragma unroll
        for (int r = 0; r < NR; ++r)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[r][i] *= sc[i];
      }
      if ((tile + 1) * kAbsKeys > lim_min) {
#pragma unroll
        for (int r = 0; r < NR; ++r) {
          int qi, h;
          my_row(r, qi, h);
          const int lim = absorbed_limit(seq, qi) - (tile * kAbsKeys + 16 * wave + 4 * q4);
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (i >= lim) s[r][i] = -INFINITY;
        }
      }
#pragma unroll
      for (int r = 0; r < NR; ++r) {
        float top = fmaxf(fmaxf(s[r][0], s[r][1]), fmaxf(s[r][2], s[r][3]));
        top = fmaxf(top, __shfl_xor(top, 16));
        top = fmaxf(top, __shfl_xor(top, 32));
        if (lane < 16) *(__attribute__((address_space(3))) float*)(lds + MAXB + (wave * ROWS + 16 * r + lane) * 4) = top;
      }
      lds_only_barrier();
      // The reference point m only has to be near the row's maximum (exp2 of up
      // to 2^8 is far inside binary32 and bf16): O is rescaled when some row's
      // maximum has grown past it by more than that, seldom after the first
      // tile. All waves see the same maxima and decide alike.
      float top[NR];
      bool grown = false;
#pragma unroll
      for (int r = 0; r < NR; ++r) {
        top[r] = -INFINITY;
#pragma unroll
        for (int w = 0; w < 4; ++w)
          top[r] = fmaxf(top[r], *(__attribute__((address_space(3))) float*)(lds + MAXB + (w * ROWS + 16 * r + c16) * 4));
        grown = grown || (top[r] - m[r]) * c2 > 8.0f;
      }
      if (__any(grown)) {
#pragma unroll
        for (int r = 0; r < NR; ++r) {
          const float mn = fmaxf(m[r], top[r]);
          const float a = m[r] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((m[r] - mn) * c2);
          m[r] = mn;
          l[r] *= a;
#pragma unroll
          for (int t = 0; t < DT; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[r][t][i] *= a;
        }
      }
      v4f sc = v4f{1, 1, 1, 1};
      if constexpr (F8) sc = lds_v4f(lds + SCL + buf * 256 + opaque((16 * wave + 4 * q4) * 4));
#pragma unroll
      for (int r = 0; r < NR; ++r) {
        const float mc = m[r] == -INFINITY ? 0.0f : m[r] * c2;
        float e[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          e[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r][i], c2, -mc));
          l[r] += e[i];
          if constexpr (F8) e[i] *= sc[i];
        }
        *(__attribute__((address_space(3))) v2i*)(lds + PBUF + (16 * r + c16) * PROW + (16 * wave + 4 * q4) * 2) =
            v2i{(int)pack_bf16(e[0], e[1]), (int)pack_bf16(e[2], e[3])};
      }
      lds_only_barrier();
#pragma unroll
      for (int s2 = 0; s2 < 2; ++s2) {
        v8bf pf[NR];
#pragma unroll
        for (int r = 0; r < NR; ++r) pf[r] = lds_v8bf(lds + PBUF + (16 * r + c16) * PROW + (32 * s2 + 8 * q4) * 2);
#pragma unroll
        for (int t = 0; t < DT; ++t) {
          v8bf vf;
          if constexpr (F8) {
            vf = widen_e4m3(read_tr8(kb + (va ^ (t << 4)) + 32 * s2 * T::LROW));
          } else {
            const v4s lo = read_tr16(kb + (va ^ (t << 5)) + 32 * s2 * T::LROW);
            const v4s hi = read_tr16(kb + (va ^ ((t << 5) | 16)) + (32 * s2 + 4) * T::LROW);  // keys + 4: swizzle bit 0
            vf = join_tr16(lo, hi);
          }
#pragma unroll
          for (int r = 0; r < NR; ++r) o[r][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pf[r], o[r][t], 0, 0, 0);
        }
      }
    }

    if (__any(st.bad) && lane == 0) *(__attribute__((address_space(3))) int*)(lds + FLAG) = 1;
    // the row sums: lanes of a row hold its keys 4 q4 .. of each wave's 16
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      l[r] += __shfl_xor(l[r], 16);
      l[r] += __shfl_xor(l[r], 32);
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < NR; ++r)
      if (lane < 16) *(__attribute__((address_space(3))) float*)(lds + MAXB + (wave * ROWS + 16 * r + lane) * 4) = l[r];
    __syncthreads();
    const bool poisoned = *(__attribute__((address_space(3))) int*)(lds + FLAG) != 0;
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      float sum = 0.0f;
#pragma unroll
      for (int w = 0; w < 4; ++w) sum += *(__attribute__((address_space(3))) float*)(lds + MAXB + (w * ROWS + 16 * r + c16) * 4);
      if (poisoned) sum = __uint_as_float(0x7fc00000u);
      const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
      if (!sg.whole) {
        if (wave == 0 && lane < 16)
          p.part_lse[sg.slot * GROUP + member * ROWS + 16 * r + lane] = sum == 0.0f ? -INFINITY : __builtin_fmaf(m[r], c2, log2f(sum));
        float4* po = (float4*)p.part_o + ((sg.slot * (NR * PAIR) + member * NR + r) * (R / 16) + wave * DT) * 64 + lane;
#pragma unroll
        for (int t = 0; t < DT; ++t) po[t * 64] = make_float4(o[r][t][0] * inv, o[r][t][1] * inv, o[r][t][2] * inv, o[r][t][3] * inv);
        continue;
      }
      if (row0 + 16 * r + c16 >= rows) continue;
      int qi, h;
      my_row(r, qi, h);
      const int64_t token = seq.q0 + qi;
      if (p.lse && wave == 0 && lane < 16)
        p.lse[token * p.heads + h] = sum == 0.0f ? -INFINITY : __builtin_fmaf(m[r], p.scale, logf(sum));
      uint16_t* orow = p.out + token * p.ot + h * p.oh + wave * (R / 4) + 4 * q4;
#pragma unroll
      for (int t = 0; t < DT; ++t)
        *(uint2*)(orow + 16 * t) = make_uint2(pack_bf16(o[r][t][0] * inv, o[r][t][1] * inv), pack_bf16(o[r][t][2] * inv, o[r][t][3] * inv));
    }
  }
}

// ---- joining the partial results ------------------------------------------------
//
// One workgroup a strip of 16 rows and PIECES of its 1 KB pieces (64 lanes x 4
// values: 16 of the latent dimension for each row); its waves split the
// partials, each keeping a running maximum and sum, and meet in LDS.
template <int R, int ROWS, int PIECES>
__global__ __launch_bounds__(256) void absorbed_combine_kernel(const Absorbed p) {
  constexpr int STRIPS = ROWS / 16, ALL = R / 16;
  __shared__ float sm[4][64], sl[4][64];
  __shared__ float4 so[4][PIECES][64];
  const int lane = (int)threadIdx.x % kWave, wave = (int)threadIdx.x / kWave;
  const int64_t units = total_units(p, ROWS);
  const int64_t wgs = units < p.shares ? units : p.shares;
  const int strip = (int)(blockIdx.x % STRIPS);
  int64_t group0;
  // sequence of this row group, and its first unit
  const int64_t item = blockIdx.x / STRIPS;
  const int b = find_sequence(
      p.batch, item, [&](int s) { return (int64_t)row_groups(p, absorbed_span(p, s), ROWS); }, &group0);
  if (b < 0) return;
  const SeqSpan seq = absorbed_span(p, b);
  const int tiles = key_tiles(seq);
  int64_t before = 0;
  for (int s = lane; s < b; s += kWave) {
    const SeqSpan q = absorbed_span(p, s);
    before += (int64_t)row_groups(p, q, ROWS) * key_tiles(q);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) before += __shfl_xor(before, o);
  const int64_t first = before + (item - group0) * tiles;
  const int64_t g0 = share_of(units, first, wgs), g1 = share_of(units, first + tiles - 1, wgs);
  if (g0 == g1) return;  // one workgroup had all tiles and wrote the rows itself
  const int64_t row = (item - group0) * ROWS + strip * 16 + lane % 16;
  const int piece0 = (int)blockIdx.y * PIECES;

  float m = -INFINITY, l = 0.0f;
  float4 acc[PIECES];
#pragma unroll
  for (int k = 0; k < PIECES; ++k) acc[k] = make_float4(0, 0, 0, 0);
#pragma unroll 2
  for (int64_t g = g0 + wave; g <= g1; g += 4) {
    const int64_t slot = 2 * g + (g == g0 ? 1 : 0);
    const float ls = p.part_lse[slot * ROWS + strip * 16 + lane % 16];
    const float4* po = (const float4*)p.part_o + ((slot * STRIPS + strip) * ALL + piece0) * 64 + lane;
    float4 v[PIECES];
#pragma unroll
    for (int k = 0; k < PIECES; ++k) v[k] = po[k * 64];
    const float mn = fmaxf(m, ls);
    const float a = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - mn);
    const float w = ls == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(ls - mn);
    m = mn;
    l = l * a + w;
#pragma unroll
    for (int k = 0; k < PIECES; ++k) {
      acc[k].x = acc[k].x * a + v[k].x * w;
      acc[k].y = acc[k].y * a + v[k].y * w;
      acc[k].z = acc[k].z * a + v[k].z * w;
      acc[k].w = acc[k].w * a + v[k].w * w;
    }
  }
  sm[wave][lane] = m;
  sl[wave][lane] = l;
#pragma unroll
  for (int k = 0; k < PIECES; ++k) so[wave][k][lane] = acc[k];
  __syncthreads();
  float top = -INFINITY, total = 0.0f, w[4];
#pragma unroll
  for (int v = 0; v < 4; ++v) top = fmaxf(top, sm[v][lane]);
#pragma unroll
  for (int v = 0; v < 4; ++v) {
    // a wave that saw no key has l == 0 and nothing in its sums
    w[v] = sl[v][lane] == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(sm[v][lane] - top);
    total += w[v] * sl[v][lane];
  }
  if (row >= (int64_t)seq.n * p.heads) return;
  const float inv = total == 0.0f ? 0.0f : 1.0f / total;
  const int64_t token = seq.q0 + row / p.heads;
  const int h = (int)(row % p.heads);
  if (p.lse && piece0 == 0 && wave == 0 && lane < 16)
    p.lse[token * p.heads + h] = total == 0.0f ? -INFINITY : (top + log2f(total)) * kLn2;
  uint16_t* orow = p.out + token * p.ot + h * p.oh + 4 * (lane / 16);
  for (int k = wave; k < PIECES; k += 4) {
    float4 r = make_float4(0, 0, 0, 0);
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      const float4 x = so[v][k][lane];
      r.x += w[v] * x.x;
      r.y += w[v] * x.y;
      r.z += w[v] * x.z;
      r.w += w[v] * x.w;
    }
    *(uint2*)(orow + (piece0 + k) * 16) = make_uint2(pack_bf16(r.x * inv, r.y * inv), pack_bf16(r.z * inv, r.w * inv));
  }
}

// ---- host ---------------------------------------------------------------------------

struct AbsPlan {
  int rows;        // of a row group: 16, 32, 64, or 128 in two workgroups
  int64_t groups;  // upper bound of the batch's row groups
  int64_t shares;  // the units are divided into
  size_t lse_bytes, bytes;
};

AbsPlan absorbed_plan(const fcmoe_absorbed_args* a) {
  AbsPlan pl{};
  // Rows of a sequence, were the query tokens spread evenly.
  const int64_t per = ceil_div(a->tokens, a->batch) * a->heads;
  pl.rows = per <= 16 ? 16 : per <= 32 ? 32 : per <= 64 ? 64 : 128;
  pl.groups = a->tokens * a->heads / pl.rows + (a->batch < a->tokens ? a->batch : a->tokens);
  int dev = 0, cus = 256;
  if (hipGetDevice(&dev) != hipSuccess || hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess)
    (void)hipGetLastError();
  // One workgroup a CU (two LDS buffers fill it); 8-bit rows of 16 leave room for two.
  const int64_t slots = pl.rows == 128 ? cus / 2 : (int64_t)cus * (a->cache.e4m3 && pl.rows == 16 ? 2 : 1);
  const int64_t most = pl.groups * (a->table_width > 0 ? ceil_div(a->table_width * a->cache.page_size, kAbsKeys) : 1);
  pl.shares = most < slots ? (most > 0 ? most : 1) : slots;
  pl.lse_bytes = (size_t)round_up(2 * pl.shares * pl.rows * 4, 256);
  pl.bytes = pl.lse_bytes + (size_t)(2 * pl.shares) * (size_t)pl.rows * (size_t)a->cache.latent_dim * 4;
  return pl;
}

template <int R, int P, bool F8>
void absorbed_launch(const Absorbed& p, const AbsPlan& pl, hipStream_t stream) {
  const dim3 g((unsigned)pl.shares), b(256);
  if (pl.rows == 16)
    hipLaunchKernelGGL((absorbed_kernel<R, P, F8, 1, 1>), g, b, 0, stream, p);
  else if (pl.rows == 32)
    hipLaunchKernelGGL((absorbed_kernel<R, P, F8, 2, 1>), g, b, 0, stream, p);
  else if (pl.rows == 64)
    hipLaunchKernelGGL((absorbed_kernel<R, P, F8, 4, 1>), g, b, 0, stream, p);
  else  // pairs lie 8 workgroups apart: whole blocks of 16
    hipLaunchKernelGGL((absorbed_kernel<R, P, F8, 4, 2>), dim3((unsigned)(ceil_div(pl.shares, 8) * 16)), b, 0, stream, p);
}

template <int R>
void combine_launch(const Absorbed& p, const AbsPlan& pl, hipStream_t stream) {
  const dim3 b(256);
  const unsigned g = (unsigned)pl.groups;
  if (pl.rows == 128)
    hipLaunchKernelGGL((absorbed_combine_kernel<R, 128, 4>), dim3(g * 8, R / 64), b, 0, stream, p);
  else if (pl.rows == 64)
    hipLaunchKernelGGL((absorbed_combine_kernel<R, 64, 4>), dim3(g * 4, R / 64), b, 0, stream, p);
  else if (pl.rows == 32)
    hipLaunchKernelGGL((absorbed_combine_kernel<R, 32, 4>), dim3(g * 2, R / 64), b, 0, stream, p);
  else if (pl.groups >= 64)
    hipLaunchKernelGGL((absorbed_combine_kernel<R, 16, 4>), dim3(g, R / 64), b, 0, stream, p);
  else
    hipLaunchKernelGGL((absorbed_combine_kernel<R, 16, 1>), dim3(g, R / 16), b, 0, stream, p);
}

int check_absorbed(const fcmoe_absorbed_args* a) {
  if (!a) return fail(FCMOE_EINVAL, "absorbed_attention: NULL args");
  if (const int rc = check_latent_cache(a->cache, "absorbed_attention")) return rc;
  if (a->tokens < 0 || a->batch <= 0 || a->batch > (1 << 20) || a->heads <= 0 || a->heads > 65536 ||
      a->tokens * a->heads > INT32_MAX / 2 || a->table_width < 0 || a->table_width > INT32_MAX ||
      a->page_table_stride < 0)
    return fail(FCMOE_EINVAL, "absorbed_attention: bad shape");
  if (!a->query_starts && a->tokens != a->batch)
    return fail(FCMOE_EINVAL, "absorbed_attention: without query_starts there is one token a sequence");
  return FCMOE_OK;
}

}  // namespace

}  // namespace fcmoe

using namespace fcmoe;

extern "C" size_t fcmoe_absorbed_attention_workspace_bytes(const fcmoe_absorbed_args* a) {
  if (check_absorbed(a) != FCMOE_OK || a->tokens == 0) return 0;
  return absorbed_plan(a).bytes;
}

extern "C" int fcmoe_absorbed_attention(const fcmoe_absorbed_args* a, hipStream_t stream) {
  if (const int rc = check_absorbed(a)) return rc;
  if (!(a->scale > 0.0f) || !(a->scale < INFINITY))
    return fail(FCMOE_EINVAL, "absorbed_attention: scale must be positive and finite");
  if (a->tokens == 0) return FCMOE_OK;
  if (!a->q_latent || (a->cache.rope_dim && !a->q_rope) || !a->kv_lens || !a->out || (a->table_width > 0 && !a->page_table))
    return fail(FCMOE_EINVAL, "absorbed_attention: NULL pointer");
  if (a->q_latent_token_stride % 8 || a->q_latent_head_stride % 8 || (uintptr_t)a->q_latent % 16 ||
      a->q_rope_token_stride % 8 || a->q_rope_head_stride % 8 || (uintptr_t)a->q_rope % 16)
    return fail(FCMOE_EINVAL, "absorbed_attention: query rows must start at multiples of 16 bytes");
  if (a->out_token_stride % 4 || a->out_head_stride % 4 || (uintptr_t)a->out % 8)
    return fail(FCMOE_EINVAL, "absorbed_attention: out rows must start at multiples of 8 bytes");
  const AbsPlan pl = absorbed_plan(a);
  if (!a->workspace || a->workspace_bytes < pl.bytes) return fail(FCMOE_ESPACE, "absorbed_attention: workspace too small");
  if ((uintptr_t)a->workspace % 16) return fail(FCMOE_EINVAL, "absorbed_attention: unaligned workspace");
  Absorbed p{};
  p.ql = a->q_latent, p.qlt = a->q_latent_token_stride, p.qlh = a->q_latent_head_stride;
  p.qr = a->q_rope, p.qrt = a->q_rope_token_stride, p.qrh = a->q_rope_head_stride;
  p.c = a->cache;
  p.table = a->page_table, p.width = a->table_width, p.table_stride = a->page_table_stride;
  p.lens = a->kv_lens, p.q_starts = a->query_starts;
  p.tokens = a->tokens, p.batch = (int)a->batch, p.heads = (int)a->heads;
  p.scale = a->scale;
  p.out = a->out, p.ot = a->out_token_stride, p.oh = a->out_head_stride, p.lse = a->lse;
  p.part_lse = (float*)a->workspace;
  p.part_o = (float*)((char*)a->workspace + pl.lse_bytes);
  p.shares = (int)pl.shares;
  p.zero_tail = a->zero_uncovered && a->query_starts;
  const bool f8 = a->cache.e4m3 != 0;
  if (a->cache.latent_dim == 512) {
    if (a->cache.rope_dim == 64)
      f8 ? absorbed_launch<512, 64, true>(p, pl, stream) : absorbed_launch<512, 64, false>(p, pl, stream);
    else
      f8 ? absorbed_launch<512, 0, true>(p, pl, stream) : absorbed_launch<512, 0, false>(p, pl, stream);
    combine_launch<512>(p, pl, stream);
  } else {
    if (a->cache.rope_dim == 64)
      f8 ? absorbed_launch<256, 64, true>(p, pl, stream) : absorbed_launch<256, 64, false>(p, pl, stream);
    else
      f8 ? absorbed_launch<256, 0, true>(p, pl, stream) : absorbed_launch<256, 0, false>(p, pl, stream);
    combine_launch<256>(p, pl, stream);
  }
  return check_launch("absorbed_attention");
}
