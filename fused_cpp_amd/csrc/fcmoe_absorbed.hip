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
#include <type_traits>

#include "fcmoe_internal.h"
#include "fcmoe_latent.h"

namespace fcmoe {

namespace {

constexpr int kAbsKeys = 64;  // keys of a tile

// A row group whose tiles end up with several shares: left by the share that
// has its first tile for the launch that joins the partial results. Kept by
// group where there are no more groups than shares (every group's is written,
// most not valid), else by share (of which at most one group's last tile lies
// beyond it).
struct Joint {
  int64_t q0;
  int rows, row0;   // of the sequence; first of the group
  int first, last;  // shares with the group's first and last tile
  int valid;
};

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
  Joint* joints;    // [groups] or [shares]
  int* groups;      // [1] groups of the batch
  int by_group;
  int shares;
  int page_shift;  // log2 of a page size that is a power of two, else -1
  int whole;       // pages hold multiples of 16 keys
  int zero_tail;
};

__device__ __forceinline__ SeqSpan absorbed_span(const Absorbed& p, int b) {
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
  s.len = (int)clamp64(p.lens[b], 0, reach < INT32_MAX - 128 ? reach : INT32_MAX - 128);
  return s;
}

__device__ __forceinline__ int row_groups(const Absorbed& p, const SeqSpan& s, int rows) {
  return (int)(((int64_t)s.n * p.heads + rows - 1) / rows);
}
// Tiles of a row group; at least one, so that a sequence without keys still gets its rows written.
__device__ __forceinline__ int key_tiles(const SeqSpan& s) { return s.len > 0 ? (s.len + kAbsKeys - 1) / kAbsKeys : 1; }
// Units of a row group: its tiles, and ahead of them what bringing its queries
// in costs in tiles' time. Times with 0, 1, 3 and 4 of them over those with 2, mean
// of 104 batches (24 to 300 sequences of up to 300 to 6000 keys, 16 to 512 rows
// each, bf16 and e4m3, 512 + 64 and 256): 1.14, 1.05, 0.99, 0.99; with 0 each row
// count and type loses 9 to 29%, with 3 and 4 short batches of 16 rows lose up to 12%
// and long ones of 128 win as much.
constexpr int kGroupCost = 2;
__device__ __forceinline__ int group_units(const SeqSpan& s) { return key_tiles(s) + kGroupCost; }

__device__ __forceinline__ int absorbed_limit(const SeqSpan& s, int i) {
  const int v = s.len - s.n + i + 1;
  return v < 0 ? 0 : v > s.len ? s.len : v;
}

__device__ __forceinline__ int64_t share_begin(int64_t units, int64_t g, int64_t wgs) { return units * g / wgs; }
__device__ __forceinline__ int share_size(int64_t units, int64_t g, int64_t wgs) {
  const int64_t n = share_begin(units, g + 1, wgs) - share_begin(units, g, wgs);
  return n < INT32_MAX ? (int)n : INT32_MAX;
}
// The workgroup whose share holds unit u.
__device__ __forceinline__ int64_t share_of(int64_t units, int64_t u, int64_t wgs) {
  return ((u + 1) * wgs + units - 1) / units - 1;
}

// One range of key tiles of one row group.
struct Segment {
  SeqSpan seq;
  int b;
  int row0;            // first row of the group
  int t_begin, t_end;  // tiles
  int tiles;           // of the group
  int units, ahead;
};

// The segment that starts at unit u, `left` units before the end of its share.
__device__ __forceinline__ Segment next_segment(const Absorbed& p, int rows, int64_t u, int left) {
  Segment s;
  int64_t before;
  s.b = find_sequence(
      p.batch, u, [&](int b) { return absorbed_span(p, b); },
      [&](const SeqSpan& q) { return (int64_t)row_groups(p, q, rows) * group_units(q); }, &s.seq, &before);
  s.tiles = key_tiles(s.seq);
  const uint32_t rel = (uint32_t)(u - before);  // among the sequence's units
  const uint32_t per = (uint32_t)group_units(s.seq), group = rel / per;
  const int first = (int)(rel - group * per);  // among the group's
  s.units = uniform(min((int)per - first, left));
  s.t_begin = uniform(max(first - kGroupCost, 0));
  s.t_end = uniform(max(first + s.units - kGroupCost, 0));
  s.row0 = uniform((int)group * rows);
  s.ahead = uniform(kGroupCost + s.tiles - 1 - first);  // units from u to the group's last
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
  static constexpr int RLOADS = 16 * RROW / 1024;         // 1 KB pieces of a wave's 16 key parts
};

typedef __attribute__((address_space(3))) float lds_f32;
typedef __attribute__((address_space(3))) int lds_i32;
typedef __attribute__((address_space(1))) v4i global_v4i;  // an address from integers is a generic one otherwise

// Brings a wave's 16 keys of a tile into LDS. Lane l knows the cached row of
// the wave's key l % 16: its page id is read one tile ahead (fetch), so that
// the rows' addresses are there when the buffer is free.
//
// Latent rows go from memory straight to LDS, one load a key with its address
// in scalar registers; they are buffer loads, because after a global load to
// LDS the compiler waits for all of a wave's LDS reads wherever it needs one.
// The key parts and scales (rows too short for a load each) pass through
// registers. Where a wave's 16 keys lie in one page and all exist (pages of a
// multiple of 16 keys, tiles before the last), one address serves them all, a
// load brings 1 KB of them whatever the rows' length, and the key parts and
// scales go straight to LDS too: 128 heads, 64 sequences 161 us -> 148.
template <int R, int P, bool F8>
struct Stager {
  using T = Tile<R, P, F8>;
  const int32_t* table;
  int wave, turn, last_key;  // last_key: of the sequence
  int32_t id;
  int in;
  uint64_t lat;  // the tile being brought in
  v4i part[P > 0 ? T::RLOADS : 1];
  float scale;
  // a tile whose 64 keys all exist, in pages of multiples of 16: the wave's 16
  // keys are neighbours in memory, first latent row, key part and scale here
  uint64_t wl, wr, ws;
  uint32_t step, rstep;  // bytes between rows
  bool whole;
  static constexpr int KPL = 1024 / T::LROW;       // keys a load of 1 KB brings
  static constexpr int RKPL = P > 0 ? 1024 / T::RROW : 1;
  static constexpr int WLOADS = 16 / KPL, WRLOADS = P > 0 ? 16 / RKPL : 0;

  __device__ __forceinline__ void begin(const Absorbed& p, const SeqSpan& s, int b, int w, int member) {
    wave = w;
    turn = 8 * member;
    table = p.table + (int64_t)b * p.table_stride;
    last_key = s.len - 1;
  }
  __device__ __forceinline__ void fetch(const Absorbed& p, int tile) {
    int key = tile * kAbsKeys + 16 * wave + lane_now() % 16;
    key = key < last_key ? key : last_key;  // keys past the length re-read its last one; their scores are masked
    uint32_t page;
    if (opaque_uniform(p.page_shift) >= 0) {
      page = (uint32_t)key >> p.page_shift;
      in = key - (int)(page << p.page_shift);
    } else {
      const uint32_t size = (uint32_t)opaque_uniform((int)p.c.page_size);
      page = (uint32_t)key / size;
      in = key - (int)(page * size);
    }
    id = table[page];
  }
  // The fetched tile's latent addresses.
  __device__ __forceinline__ void start(const Absorbed& p, lds_u8* bad_flag) {
    const bool bad = (uint64_t)(int64_t)id >= (uint64_t)p.c.pages;
    if (bad) id = 0;
    if (__any(bad)) *(lds_i32*)bad_flag = 1;  // every lane writes the same
    lat = (uint64_t)p.c.latent + (id * p.c.latent_page_stride + in * p.c.latent_row_stride) * T::ELEM;
  }
  __device__ __forceinline__ void start_whole(const Absorbed& p, lds_u8* bad_flag) {
    uint32_t page = (uint32_t)uniform(id);
    const uint32_t row = (uint32_t)uniform(in);
    if (page >= (uint32_t)p.c.pages) {
      page = 0;
      *(lds_i32*)bad_flag = 1;
    }
    // pages of less than 4 GB: products of 32 bits by 32
    step = (uint32_t)(p.c.latent_row_stride * T::ELEM);
    wl = (uint64_t)p.c.latent + (uint64_t)page * (uint32_t)(p.c.latent_page_stride * T::ELEM) + row * step;
    if constexpr (P > 0) {
      rstep = (uint32_t)(p.c.rope_row_stride * T::ELEM);
      wr = (uint64_t)p.c.rope + (uint64_t)page * (uint32_t)(p.c.rope_page_stride * T::ELEM) + row * rstep;
    }
    if constexpr (F8) ws = (uint64_t)p.c.scale + (uint64_t)page * (uint32_t)(p.c.scale_page_stride * 4) + row * 4;
    wl = (uint64_t)opaque_uniform((int64_t)wl);  // or the compiler merges its store with that of `lat`, through memory
  }
  // Of such a tile: load u of WLOADS + WRLOADS (latent rows, then key parts).
  template <int u>
  static __device__ __forceinline__ void load_whole(lds_u8* dst, uint64_t wl, uint64_t wr, uint32_t step, uint32_t rstep,
                                                    int lane16, int lane_row, int wave, int turn) {
    if constexpr (u < WLOADS) {
      const int half = (KPL * u) & 8 ? turn ^ 8 : turn;  // the first key of the eight that the load is in
      load_lds16(rows_at(wl, 15 * step + T::LROW), dst + (16 * wave + half + KPL * u % 8) * T::LROW,
                 (uint32_t)((lane16 ^ ((swz_key<F8>(KPL * u % 8) * 16) ^ (F8 ? half / 2 : half) * 16)) + lane_row),
                 step * (uint32_t)(half + KPL * u % 8));
    } else if constexpr (P > 0) {
      const int ln = lane_now(), k = ln / T::RUNITS;
      load_lds16(rows_at(wr, 15 * rstep + T::RROW), dst + T::ROPE + (16 * wave + RKPL * (u - WLOADS)) * T::RROW,
                 (uint32_t)(k * (int)rstep + ((ln % T::RUNITS) ^ swz_rope<F8>(k)) * 16), rstep * (uint32_t)(RKPL * (u - WLOADS)));
    }
  }
  __device__ __forceinline__ void scales_whole(lds_u8* scl) const {
    if constexpr (F8) {
      const int ln = lane_now();
      if (ln < 16) load_lds4(rows_at(ws, 64), scl + 64 * wave, (uint32_t)ln * 4);
    }
  }
  static __device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_at(uint64_t base, uint32_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc((void*)base, (short)0, (int)bytes, kBufWord3);
  }
  // Its key parts and scales on their way to registers.
  __device__ __forceinline__ void parts(const Absorbed& p) {
    if constexpr (P > 0) {
      const uint32_t ln = (uint32_t)lane_now();
      const uint64_t rope = (uint64_t)p.c.rope + (id * p.c.rope_page_stride + in * p.c.rope_row_stride) * T::ELEM;
#pragma unroll
      for (int u = 0; u < T::RLOADS; ++u)
        part[u] = *(const global_v4i*)(__shfl((unsigned long long)rope, u * (64 / T::RUNITS) + (int)(ln / T::RUNITS)) +
                                       (ln % T::RUNITS) * 16);
    }
    if constexpr (F8) scale = p.c.scale[id * p.c.scale_page_stride + in];
  }
  // The latent row of key u ^ turn (u 0 .. 15, turn 0 or 8) to its place in
  // buffer `dst`. What its L2 lacks comes to a CU at some 10 bytes a clock
  // (4.9 TB/s over 256 CUs), what it has several times as fast: the two workgroups that share keys bring the halves of their
  // 16 in opposite orders, so that each finds one half fetched by the other.
  __device__ __forceinline__ void load(lds_u8* dst, int u) const {
    const uint32_t ln = (uint32_t)lane_now();
    const int k = u ^ turn;
    const __amdgpu_buffer_rsrc_t row = __builtin_amdgcn_make_buffer_rsrc((void*)lane_value(lat, k), (short)0, T::LROW, kBufWord3);
    const uint32_t x = (uint32_t)swz_key<F8>(u) ^ (uint32_t)(F8 ? turn / 2 : turn);
    if (T::UNITS == 64 || ln < T::UNITS)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(row, (__attribute__((address_space(3))) void*)(dst + (16 * wave + k) * T::LROW), 16,
                                               (ln ^ x) * 16, 0, 0, 0);
  }
  __device__ __forceinline__ void load_all(lds_u8* dst) const {
#pragma unroll
    for (int u = 0; u < 16; ++u) load(dst, u);
  }
  // The key parts and scales from registers to buffer `dst` (scales to `scl`).
  __device__ __forceinline__ void finish(lds_u8* dst, lds_u8* scl) const {
    const uint32_t ln = (uint32_t)lane_now();
    if constexpr (P > 0) {
#pragma unroll
      for (int u = 0; u < T::RLOADS; ++u) {
        const uint32_t k = u * (64 / T::RUNITS) + ln / T::RUNITS;
        *(__attribute__((address_space(3))) v4i*)(dst + T::ROPE + (16 * wave + k) * T::RROW +
                                                  ((ln % T::RUNITS) ^ (uint32_t)swz_rope<F8>(k)) * 16) = part[u];
      }
    }
    if constexpr (F8) {
      if (ln < 16) *(lds_f32*)(scl + (16 * wave + ln) * 4) = scale;
    }
  }
};

// f(integral_constant<int, i>) for an i that unrolling makes known.
template <int N, typename F>
__device__ __forceinline__ void unroll_at(int i, F f) {
  if constexpr (N > 0) {
    if (i == N - 1)
      f(std::integral_constant<int, N - 1>{});
    else
      unroll_at<N - 1>(i, f);
  }
}

__device__ __forceinline__ v8bf lds_v8bf(const lds_u8* p) { return *(const __attribute__((address_space(3))) v8bf*)p; }
__device__ __forceinline__ v4i lds_v4i(const lds_u8* p) { return *(const __attribute__((address_space(3))) v4i*)p; }
__device__ __forceinline__ v4f lds_v4f(const lds_u8* p) { return *(const __attribute__((address_space(3))) v4f*)p; }

// ---- the attention kernel ------------------------------------------------------
//
// A workgroup takes MT row tiles of 16 rows (16, 32 or 64 rows); its four waves
// split each key tile twice: for S^T a wave takes 16 of the 64 keys, for O^T a
// quarter of the latent dimension, both for all rows. So K and V are read from
// LDS once however many rows there are, and a fragment feeds MT MFMAs; S goes
// through LDS as P between the two. Q (R + P values of every row) and a quarter
// of O stay in registers: 72 MT and 32 MT of them at 512 + 64, so that 64 rows
// take all of a SIMD's 512 for its one wave. Half of those are accumulation
// registers, which MFMAs can read as operands; Q lies there, and its MFMAs are
// written out, because the compiler would copy each fragment to an ordinary
// register first. With eight waves instead, Q would leave no registers to read K
// fragments ahead with. A tile of 64 rows takes 6100 clocks: 2200 for S, 800 for the
// weights and their barrier, 2300 for P V, the rest for the next tile's addresses
// and arrival; its products alone are 2200 (128 heads, 64 sequences of 4096 bf16 rows).
//
// PAIR: the rows of a sequence fill two workgroups (65 rows and more); these
// two take the same tiles at the same time on the same XCD, whose L2 then
// brings a cached row from memory once for both.
//
// The reference point m of a row's exponentials only has to be near its maximum
// (exp2 of up to 2^8 is far inside binary32 and bf16), so each wave compares its
// own scores with it; only when one has grown past it by more than that do the
// waves exchange maxima and rescale O, seldom after the first tile.

// acc (+)= K fragment x Q fragment. The compiler does not know these for MFMAs,
// so the waits it would put in stand here: two states between an ordinary
// instruction that wrote the K fragment and the first product that reads it
// (WAIT); a chain's next product comes MT - 1 others later; and qk_done waits
// out the last ones before anything else touches the accumulators.
template <bool ACC, bool FIRST, bool WAIT>
__device__ __forceinline__ void mfma_qk(v4f& acc, const v8bf& k, const v8bf& q) {
  if constexpr (WAIT && FIRST) {
    if constexpr (ACC)
      asm volatile("s_nop 1\n\tv_mfma_f32_16x16x32_bf16 %0, %1, %2, 0" : "=&v"(acc) : "v"(k), "a"(q));
    else
      asm volatile("s_nop 1\n\tv_mfma_f32_16x16x32_bf16 %0, %1, %2, 0" : "=&v"(acc) : "v"(k), "v"(q));
  } else if constexpr (WAIT) {
    if constexpr (ACC)
      asm volatile("s_nop 1\n\tv_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+v"(acc) : "v"(k), "a"(q));
    else
      asm volatile("s_nop 1\n\tv_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+v"(acc) : "v"(k), "v"(q));
  } else if constexpr (FIRST) {
    if constexpr (ACC)
      asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, 0" : "=&v"(acc) : "v"(k), "a"(q));
    else
      asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, 0" : "=&v"(acc) : "v"(k), "v"(q));
  } else {
    if constexpr (ACC)
      asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+v"(acc) : "v"(k), "a"(q));
    else
      asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+v"(acc) : "v"(k), "v"(q));
  }
}
template <int N>
__device__ __forceinline__ void qk_done(v4f* s) {
  if constexpr (N == 2)
    asm volatile("s_nop 11" : "+v"(s[0]), "+v"(s[1]));
  else
    asm volatile("s_nop 11" : "+v"(s[0]), "+v"(s[1]), "+v"(s[2]), "+v"(s[3]));
}

// The kernel's arguments, read anew from the kernarg segment: what only the
// ends of a segment need does not take scalar registers through its tiles.
__device__ __forceinline__ Absorbed args_now() {
#ifdef __HIP_DEVICE_COMPILE__
  auto* k = (const __attribute__((address_space(4))) Absorbed*)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(k));
  return *k;
#else
  return Absorbed{};
#endif
}

template <int R, int P, bool F8, int MT, int PAIR>
__global__ __launch_bounds__(256, MT == 1 && F8 ? 2 : 1) void absorbed_kernel(const Absorbed p) {
  using T = Tile<R, P, F8>;
  constexpr int ROWS = 16 * MT;       // of this workgroup
  constexpr int GROUP = ROWS * PAIR;  // of the row group that its pair shares
  constexpr int KS = (R + P) / 32, RS = R / 32, DT = R / 64;  // 16x16x32 steps; d tiles of a wave in O^T
  constexpr int AKS = MT == 1 ? 0 : MT == 2 ? KS : KS < 16 ? KS : 16;  // steps whose Q lies in accumulation registers
  constexpr int PROW = 2 * kAbsKeys + 16;  // bytes of a P row, padded off the banks' period
  constexpr int SCL = 2 * T::BYTES, PBUF = SCL + (F8 ? 2 * 256 : 0), MAXB = PBUF + ROWS * PROW;
  constexpr int FLAGS = MAXB + 4 * ROWS * 4;  // grown (even, odd tiles), bad page
  constexpr bool QFITS = ROWS * 2 * (R + P) <= T::BYTES;  // Q on its way to registers: in the second buffer, or its own
  constexpr int QOFF = QFITS ? T::BYTES : (FLAGS + 16 + 1023) / 1024 * 1024;
  __shared__ __align__(1024) uint8_t smem[QFITS || MT == 1 ? FLAGS + 16 : QOFF + ROWS * 2 * (R + P)];
  lds_u8* lds = (lds_u8*)smem;
  const int wave = wave_index();
  int64_t units, shares;
  {
    const Absorbed a = args_now();
    if (a.zero_tail)
      zero_uncovered(a.q_starts, a.batch, a.tokens, a.heads, R, a.out, a.ot, a.oh, a.lse, blockIdx.x, gridDim.x);
    units = count_items(
        a.batch, [&](int b) { return absorbed_span(a, b); },
        [&](const SeqSpan& q) { return (int64_t)row_groups(a, q, GROUP) * group_units(q); });
    shares = units < a.shares ? units : a.shares;
  }
  // workgroups go to the 8 XCDs by blockIdx % 8: a pair's two are 8 apart
  const int member = PAIR == 2 ? (int)(blockIdx.x / 8 % 2) : 0;
  const int64_t g = PAIR == 2 ? blockIdx.x / 16 * 8 + blockIdx.x % 8 : blockIdx.x;
  if (g >= shares) {
    if (!p.by_group && member == 0 && g < p.shares && threadIdx.x == 0) p.joints[g].valid = 0;
    if (blockIdx.x == 0 && threadIdx.x == 0) *p.groups = 0;  // no units at all
    return;
  }
  if (blockIdx.x == 0 && p.by_group) {
    const int64_t n = count_items(
        p.batch, [&](int b) { return absorbed_span(p, b); }, [&](const SeqSpan& q) { return (int64_t)row_groups(p, q, GROUP); });
    if (threadIdx.x == 0) *p.groups = (int)n;
  }
  int64_t u = share_begin(units, g, shares);
  int left = share_size(units, g, shares);
  int joint = 0;  // a joint of this share was written
  const float c2 = uniform(p.scale * kLog2e);

  while (left > 0) {
    const Absorbed a = args_now();
    const Segment sg = next_segment(a, GROUP, u, left);
    const SeqSpan& seq = sg.seq;
    const int rows = seq.n * a.heads;
    const int row0 = sg.row0 + member * ROWS;
    const bool whole = sg.t_begin == 0 && sg.t_end == sg.tiles;
    // of a share's segments only the first can start inside a group's tiles and
    // only the last can end inside them: two partial slots a share
    const int64_t slot = 2 * g + (sg.t_begin == 0 ? 1 : 0);
    u += sg.units;
    left -= sg.units;
    if (sg.t_begin == sg.t_end) continue;  // the group's tiles begin in the next share
    if (sg.t_begin == 0 && (a.by_group || !whole)) {
      joint = uniform(joint | (whole ? 0 : 1));
      int64_t at = g;
      if (a.by_group)
        at = sg.row0 / GROUP + count_items(
                                   sg.b, [&](int b) { return absorbed_span(a, b); },
                                   [&](const SeqSpan& q) { return (int64_t)row_groups(a, q, GROUP); });
      if (member == 0 && wave == 0 && lane_now() == 0) {
        const int64_t last = share_of(opaque_uniform(units), u - sg.units + sg.ahead, shares);
        a.joints[at] = Joint{seq.q0, rows, sg.row0, (int)g, (int)last, whole ? 0 : 1};
      }
    }
    if (PAIR == 2 && row0 >= rows) continue;  // the group's rows end with the other workgroup
    // query token and head of row `at` of the workgroup (rows past the last repeat it and are not stored)
    auto my_row = [&](int at, int& i, int& h) {
      int row = row0 + at;
      row = row < rows ? row : rows - 1;
      const int heads = opaque_uniform(p.heads);
      i = row / heads;
      h = row - i * heads;
    };
    const int lim_min = absorbed_limit(seq, row0 / a.heads);

    Stager<R, P, F8> st;
    st.begin(p, seq, sg.b, wave, member);
    const bool any = seq.len > 0;
    if (any) st.fetch(p, sg.t_begin);
    lds_only_barrier();  // the last segment's accesses to LDS have ended
    if (wave == 0) {
      const int ln = lane_now();
      if (ln < 3) *(lds_i32*)(lds + FLAGS + 4 * ln) = 0;
    }
    // Q: B operand. bf16 rows: values 32 ks + 8 (lane / 16) ..; 8-bit rows are
    // read 16 values a lane, two steps at once: 64 (ks / 2) + 16 (lane / 16) + 8 (ks % 2) ..
    v8bf qf[MT][KS];
    if constexpr (MT == 1) {
      const int ql_ = lane_now(), qq = ql_ / 16;
      int i, h;
      my_row(ql_ % 16, i, h);
      const uint16_t* ql = a.ql + (seq.q0 + i) * a.qlt + h * a.qlh;
      const uint16_t* qr = P ? a.qr + (seq.q0 + i) * a.qrt + h * a.qrh : nullptr;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const int k = ks < RS ? ks : ks - RS;
        const int d = F8 ? 64 * (k / 2) + 16 * qq + 8 * (k % 2) : 32 * k + 8 * qq;
        qf[0][ks] = *(const v8bf*)((ks < RS ? ql : qr) + d);
      }
      lds_only_barrier();
      if (any) {
        st.start(p, lds + FLAGS + 8);
        st.load_all(lds);
        st.parts(p);
        st.finish(lds, lds + SCL);
        if (sg.t_begin + 1 < sg.t_end) st.fetch(p, sg.t_begin + 1);
      }
    } else {
      // Through LDS, laid out as a bf16 tile: read straight into fragments, each
      // wave would fetch every row in 64-byte pieces.
      // 16-bit tiles: in the second buffer, which the first iteration fills only
      // once everyone has met at its barrier.
      constexpr int QR = ROWS / 4;  // rows a wave brings
      int i, h;
      const uint32_t ln = (uint32_t)lane_now();
      my_row(QR * wave + (int)(ln % QR), i, h);
      const uint64_t ql = (uint64_t)(a.ql + (seq.q0 + i) * a.qlt + h * a.qlh);
      const uint64_t qr = P ? (uint64_t)(a.qr + (seq.q0 + i) * a.qrt + h * a.qrh) : 0;
#pragma unroll
      for (int k = 0; k < QR; ++k) {
        const __amdgpu_buffer_rsrc_t row = __builtin_amdgcn_make_buffer_rsrc((void*)lane_value(ql, k), (short)0, 2 * R, kBufWord3);
        const uint32_t x = (uint32_t)swz_key<false>(k) ^ (QR == 8 ? 8 * (wave & 1) : 0);
        if (R == 512 || ln < R / 8)
          __builtin_amdgcn_raw_ptr_buffer_load_lds(row, (__attribute__((address_space(3))) void*)(lds + QOFF + (QR * wave + k) * 2 * R),
                                                   16, (ln ^ x) * 16, 0, 0, 0);
      }
      v4i qp[P > 0 ? QR / 8 : 1];
      if constexpr (P > 0) {
#pragma unroll
        for (int k = 0; k < QR / 8; ++k)
          qp[k] = *(const global_v4i*)(__shfl((unsigned long long)qr, 8 * k + (int)(ln / 8)) + (ln % 8) * 16);
      }
      lds_only_barrier();
      if (any) {
        st.start(p, lds + FLAGS + 8);
        st.load_all(lds);
        st.parts(p);
      }
      if constexpr (P > 0) {
#pragma unroll
        for (int k = 0; k < QR / 8; ++k) {
          const uint32_t row = QR * wave + 8 * k + ln / 8;
          *(__attribute__((address_space(3))) v4i*)(lds + QOFF + ROWS * 2 * R + row * 128 +
                                                    ((ln % 8) ^ (uint32_t)swz_rope<false>(row)) * 16) = qp[k];
        }
      }
      // Q's loads came first: its fragments are read while the keys are on their way
      if (any) {
        wait_vm<16 + (P > 0 ? T::RLOADS : 0) + (F8 ? 1 : 0)>();
        lds_only_barrier();
      } else {
        loads_barrier();
      }
      const int ql_ = lane_now(), qq = ql_ / 16, qc = ql_ % 16;
#pragma unroll
      for (int r = 0; r < MT; ++r)
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          const int k = ks < RS ? ks : ks - RS;
          const int unit = F8 ? 8 * (k / 2) + 2 * qq + k % 2 : 4 * k + qq;
          qf[r][ks] = lds_v8bf(lds + QOFF + (ks < RS ? (16 * r + qc) * 2 * R + ((unit ^ swz_key<false>(qc)) * 16)
                                                     : ROWS * 2 * R + (16 * r + qc) * 128 + ((unit ^ swz_rope<false>(qc)) * 16)));
        }
      if (any) {
        st.finish(lds, lds + SCL);
        if (sg.t_begin + 1 < sg.t_end) st.fetch(p, sg.t_begin + 1);
      }
    }
    float m[MT], l[MT];  // the rows' reference points, their sums over this lane's keys
    v4f o[MT][DT];
#pragma unroll
    for (int r = 0; r < MT; ++r) {
      m[r] = -INFINITY;
      l[r] = 0.0f;
#pragma unroll
      for (int t = 0; t < DT; ++t) o[r][t] = v4f{0, 0, 0, 0};
    }

    // what the loads of a tile need, formed at the end of the tile before the one they go among
    auto start = [&](int tile) {
      st.whole = false;
      if (tile >= sg.t_end) return;
      const Absorbed b = args_now();
      st.whole = b.whole && (tile + 1) * kAbsKeys <= seq.len;
      if (st.whole)
        st.start_whole(b, lds + FLAGS + 8);
      else
        st.start(b, lds + FLAGS + 8);
    };
    if (any) start(sg.t_begin + 1);
    for (int tile = sg.t_begin; any && tile < sg.t_end; ++tile) {
      const int buf = (tile - sg.t_begin) & 1;
      const bool more = tile + 1 < sg.t_end;
      loads_barrier();  // the tile has landed; everyone is done with the other buffer
      const bool whole = st.whole;  // the next tile
      const lds_u8* kb = lds + buf * T::BYTES;
      lds_u8* next = lds + (buf ^ 1) * T::BYTES;
      // What depends on the lane is formed here, in each tile, and addresses
      // where they are used, an XOR each: kept across the loop they would take
      // the registers that Q and O need.
      const int tl = lane_now(), tq = tl / 16, tc = tl % 16;
      // K reads: key krow, unit 4 j + tq of a window of units that the swizzle
      // stays in (16 units, 8 of an 8-bit row); the key part has one window
      const int krow = 16 * wave + tc;
      const int ka = krow * T::LROW + ((tq ^ swz_key<F8>(krow)) * 16);
      const int kra = T::ROPE + krow * T::RROW + ((tq ^ swz_rope<F8>(krow)) * 16);
      // One 16-byte read of K a step (an 8-bit row's serves two MFMAs), AHEAD
      // steps before its MFMAs (as many as there are registers for); the next tile's loads go between them.
      constexpr int STEPS = F8 ? KS / 2 : KS, AHEAD = MT < 4 ? 4 : F8 ? PAIR : 3, RING = AHEAD + 1;
      auto k_at = [&](int st_) {
        if constexpr (F8) return st_ < RS / 2 ? (ka ^ ((st_ & 1) << 6)) + (st_ >> 1) * 128 : kra;
        return st_ < RS ? (ka ^ ((st_ & 3) << 6)) + (st_ >> 2) * 256 : kra ^ ((st_ - RS) << 6);
      };
      v4f s[MT];
      // with either kind and without the next tile's loads, as straight-line code
      // each: no branch around every load
      auto scores = [&](auto loads_) {
        constexpr int LOADS = decltype(loads_)::value;
        static_assert(STEPS == Stager<R, P, F8>::WLOADS + Stager<R, P, F8>::WRLOADS, "a load a step");
        using S = Stager<R, P, F8>;
        const uint64_t wl = st.wl, wr = st.wr;
        const uint32_t step = st.step, rstep = st.rstep;
        const int wave = st.wave, turn = st.turn;
        const int part = tl / S::T::UNITS;  // of a load's keys, this lane's
        const int lane16 = ((tl % S::T::UNITS) ^ swz_key<F8>(part)) * 16, lane_row = S::KPL > 1 ? part * (int)step : 0;
        v4i kf[RING];
#pragma unroll
        for (int i = 0; i < AHEAD && i < STEPS; ++i) kf[i] = lds_v4i(kb + k_at(i));
#pragma unroll
        for (int i = 0; i < STEPS; ++i) {
          if (i + AHEAD < STEPS) kf[(i + AHEAD) % RING] = lds_v4i(kb + k_at(i + AHEAD));
          if constexpr (LOADS == 1) {
#pragma unroll
            for (int k = i * 16 / STEPS; k < (i + 1) * 16 / STEPS; ++k) st.load(next, k);
          } else if constexpr (LOADS == 2) {
            unroll_at<STEPS>(i, [&](auto i_) { st.template load_whole<decltype(i_)::value>(next, wl, wr, step, rstep, lane16, lane_row, wave, turn); });
          }
          const v4i w = kf[i % RING];
          auto products = [&](auto ks_, const v8bf& a) {
            constexpr int ks = decltype(ks_)::value;
            if constexpr (MT == 1) {
              s[0] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, qf[0][ks], ks == 0 ? v4f{0, 0, 0, 0} : s[0], 0, 0, 0);
            } else {
#pragma unroll
              for (int r = 0; r < MT; ++r) r == 0 ? mfma_qk<(ks < AKS), ks == 0, true>(s[r], a, qf[r][ks]) : mfma_qk<(ks < AKS), ks == 0, false>(s[r], a, qf[r][ks]);
            }
          };
          unroll_at<STEPS>(i, [&](auto i_) {
            constexpr int ii = decltype(i_)::value;
            if constexpr (F8) {
              products(std::integral_constant<int, 2 * ii>{}, widen_e4m3(v2i{w[0], w[1]}));
              products(std::integral_constant<int, 2 * ii + 1>{}, widen_e4m3(v2i{w[2], w[3]}));
            } else {
              products(std::integral_constant<int, ii>{}, __builtin_bit_cast(v8bf, w));
            }
          });
        }
        if constexpr (MT > 1) qk_done<MT>(s);
      };
      if (whole)
        scores(std::integral_constant<int, 2>{});
      else if (more)
        scores(std::integral_constant<int, 1>{});
      else
        scores(std::integral_constant<int, 0>{});
      if (whole)
        st.scales_whole(lds + SCL + (buf ^ 1) * 256);
      else if (more)
        st.parts(args_now());  // not before: their registers are K's until here
      __builtin_amdgcn_sched_barrier(0);
      // lane: row tc of each row tile, keys 16 wave + 4 tq + i
      if constexpr (F8) {
        const v4f sc = lds_v4f(lds + SCL + buf * 256 + (16 * wave + 4 * tq) * 4);
#pragma unroll
        for (int r = 0; r < MT; ++r)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[r][i] *= sc[i];
      }
      if ((tile + 1) * kAbsKeys > lim_min) {
#pragma unroll
        for (int r = 0; r < MT; ++r) {
          int qi, h;
          my_row(16 * r + lane_now() % 16, qi, h);
          const int lim = absorbed_limit(seq, qi) - (tile * kAbsKeys + 16 * wave + 4 * tq);
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (i >= lim) s[r][i] = -INFINITY;
        }
      }
      float top[MT];
      bool grown = false;
#pragma unroll
      for (int r = 0; r < MT; ++r) {
        top[r] = fmaxf(fmaxf(s[r][0], s[r][1]), fmaxf(s[r][2], s[r][3]));
        grown = grown || (top[r] - m[r]) * c2 > 8.0f;
      }
      if (__any(grown)) *(lds_i32*)(lds + FLAGS + 4 * buf) = 1;  // every lane writes the same
      // The weights go into P V as bf16, off by at most 2^-8 of themselves: a product's operands are of one type, and a
      // second part of each would double the products. An 8-bit cache's scales, which differ by token, go into them first.
      // The sum is of what they were before (of the rounded ones it would leave the output's error as it is, and lse worse):
      // outputs err by 0.0020 to 0.0023 of their size against 64 bits (root mean square), where rounding the output alone
      // leaves 0.0017.
      float sum[MT];
      auto weights = [&]() {
        const int wl = lane_now(), wq = wl / 16, wc = wl % 16;
        v4f sc = v4f{1, 1, 1, 1};
        if constexpr (F8) sc = lds_v4f(lds + SCL + buf * 256 + (16 * wave + 4 * wq) * 4);
#pragma unroll
        for (int r = 0; r < MT; ++r) {
          const float mc = m[r] == -INFINITY ? 0.0f : m[r] * c2;
          float e[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) e[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r][i], c2, -mc));
          sum[r] = (e[0] + e[1]) + (e[2] + e[3]);
          if constexpr (F8) {
#pragma unroll
            for (int i = 0; i < 4; ++i) e[i] *= sc[i];
          }
          *(__attribute__((address_space(3))) v2i*)(lds + PBUF + (16 * r + wc) * PROW + (16 * wave + 4 * wq) * 2) =
              v2i{(int)pack_bf16(e[0], e[1]), (int)pack_bf16(e[2], e[3])};
        }
      };
      weights();
      lds_only_barrier();
      const int far = *(lds_i32*)(lds + FLAGS + 4 * buf);
      // V^T reads: this lane's place in its group's block of keys 8 vq .. 8 vq + 7;
      // unit u0 of the wave's quarter, whose other units differ from it in address
      // bits that neither the key nor the lane touches
      const int vl = lane_now(), vq = vl / 16, vc = vl % 16;
      const int vkey = F8 ? 8 * vq + vc / 2 : 8 * vq + vc / 4;
      const int u0 = F8 ? wave * DT : 2 * wave * DT + (vc % 4) / 2;
      const int va = vkey * T::LROW + ((u0 ^ swz_key<F8>(vkey)) * 16) + (vl & 1) * 8;
      // V fragments are read ahead of their MFMAs (the schedule is pinned: left to
      // itself the compiler reads each where it is used, and every d tile waits out
      // the LDS latency)
      constexpr int VN = 2 * DT, VAHEAD = 4, VRING = VAHEAD + 1;
      v4s vlo[VRING], vhi[VRING];
      v2i v8[VRING];
      auto v_read = [&](int n) {
        const int s2 = n / DT, t = n % DT;
        if constexpr (F8) {
          v8[n % VRING] = read_tr8(kb + (va ^ (t << 4)) + 32 * s2 * T::LROW);
        } else {
          vlo[n % VRING] = read_tr16(kb + (va ^ (t << 5)) + 32 * s2 * T::LROW);
          vhi[n % VRING] = read_tr16(kb + (va ^ ((t << 5) | 16)) + (32 * s2 + 4) * T::LROW);  // keys + 4: swizzle bit 0
        }
      };
      v8bf pf[2][MT];
      auto p_read = [&](int s2, int r0 = 0, int r1 = MT) {
#pragma unroll
        for (int r = r0; r < r1; ++r) pf[s2][r] = lds_v8bf(lds + PBUF + (16 * r + vc) * PROW + (32 * s2 + 8 * vq) * 2);
      };
      // ahead of the decision where there are registers: S is needed until then
      constexpr bool EARLY = MT < 4;
      auto first_reads = [&]() {
        p_read(0);
#pragma unroll
        for (int n = 0; n < VAHEAD; ++n) v_read(n);
      };
      if constexpr (EARLY) first_reads();
      if (__builtin_amdgcn_readfirstlane(far)) {
        // some row's maximum has grown: exchange maxima, rescale, form P again
        const int rl = lane_now();
#pragma unroll
        for (int r = 0; r < MT; ++r) {
          top[r] = fmaxf(top[r], __shfl_xor(top[r], 16));
          top[r] = fmaxf(top[r], __shfl_xor(top[r], 32));
          if (rl < 16) *(lds_f32*)(lds + MAXB + (wave * ROWS + 16 * r + rl) * 4) = top[r];
        }
        lds_only_barrier();
#pragma unroll
        for (int r = 0; r < MT; ++r) {
          float mn = m[r];
#pragma unroll
          for (int w = 0; w < 4; ++w) mn = fmaxf(mn, *(lds_f32*)(lds + MAXB + (w * ROWS + 16 * r + rl % 16) * 4));
          const float a = m[r] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((m[r] - mn) * c2);
          m[r] = mn;
          l[r] *= a;
#pragma unroll
          for (int t = 0; t < DT; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[r][t][i] *= a;
        }
        weights();
        lds_only_barrier();
        if constexpr (EARLY) first_reads();  // anew: not kept through the above
      }
      if constexpr (!EARLY) first_reads();
      if (wave == 0) *(lds_i32*)(lds + FLAGS + 4 * (buf ^ 1)) = 0;  // all have read it before this tile's barriers
#pragma unroll
      for (int r = 0; r < MT; ++r) l[r] += sum[r];
      if (tile + 2 < sg.t_end) st.fetch(p, tile + 2);
#pragma unroll
      for (int n = 0; n < VN; ++n) {
        __builtin_amdgcn_sched_barrier(0);
        if (n + VAHEAD < VN) v_read(n + VAHEAD);
        if (EARLY && n == DT / 2) p_read(1);
        __builtin_amdgcn_sched_barrier(0);
        const v8bf vf = F8 ? widen_e4m3(v8[n % VRING]) : join_tr16(vlo[n % VRING], vhi[n % VRING]);
#pragma unroll
        for (int r = 0; r < MT; ++r) {
          o[r][n % DT] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pf[n / DT][r], o[r][n % DT], 0, 0, 0);
          if (!EARLY && n == DT - 1) p_read(1, r, r + 1);
        }
      }
      if (more) {
        if (!whole) st.finish(next, lds + SCL + (buf ^ 1) * 256);
        start(tile + 2);
      }
    }

    // the row sums: lanes of a row hold its keys 4 (lane / 16) .. of each wave's 16
    const Absorbed e = args_now();
    const int el = lane_now(), eq = el / 16, ec = el % 16;
#pragma unroll
    for (int r = 0; r < MT; ++r) {
      l[r] += __shfl_xor(l[r], 16);
      l[r] += __shfl_xor(l[r], 32);
      if (el < 16) *(lds_f32*)(lds + MAXB + (wave * ROWS + 16 * r + el) * 4) = l[r];
    }
    lds_only_barrier();
    const bool poisoned = *(lds_i32*)(lds + FLAGS + 8) != 0;
#pragma unroll
    for (int r = 0; r < MT; ++r) {
      float sum = 0.0f;
#pragma unroll
      for (int w = 0; w < 4; ++w) sum += *(lds_f32*)(lds + MAXB + (w * ROWS + 16 * r + ec) * 4);
      if (poisoned) sum = __uint_as_float(0x7fc00000u);
      // a row that sees no key has a sum of 0: its output is 0 and its lse -inf
      const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
      if (opaque_uniform(sg.t_begin) != 0 || sg.t_end != sg.tiles) {
        if (wave == 0 && el < 16)
          e.part_lse[slot * GROUP + member * ROWS + 16 * r + el] = sum == 0.0f ? -INFINITY : __builtin_fmaf(m[r], c2, log2f(sum));
        float4* po = (float4*)e.part_o + ((slot * (MT * PAIR) + member * MT + r) * (R / 16) + wave * DT) * 64 + el;
#pragma unroll
        for (int t = 0; t < DT; ++t) po[t * 64] = make_float4(o[r][t][0] * inv, o[r][t][1] * inv, o[r][t][2] * inv, o[r][t][3] * inv);
        continue;
      }
      if (row0 + 16 * r + ec >= rows) continue;
      int qi, h;
      my_row(16 * r + ec, qi, h);
      const int64_t token = seq.q0 + qi;
      if (e.lse && wave == 0 && el < 16)
        e.lse[token * e.heads + h] = sum == 0.0f ? -INFINITY : __builtin_fmaf(m[r], e.scale, logf(sum));
      uint16_t* orow = e.out + token * e.ot + h * e.oh + wave * (16 * DT) + 4 * eq;
#pragma unroll
      for (int t = 0; t < DT; ++t)
        *(uint2*)(orow + 16 * t) = make_uint2(pack_bf16(o[r][t][0] * inv, o[r][t][1] * inv), pack_bf16(o[r][t][2] * inv, o[r][t][3] * inv));
    }
  }
  if (!p.by_group && !joint && member == 0 && wave == 0 && lane_now() == 0) p.joints[g].valid = 0;
}

// ---- joining the partial results ------------------------------------------------
//
// The joint of a strip of 16 rows (workgroup `item` of STRIPS a group), or none.
template <int STRIPS>
__device__ __forceinline__ bool find_joint(const Absorbed& p, int64_t item, Joint* j, int* strip) {
  *strip = (int)(item % STRIPS);
  const int64_t at = item / STRIPS;
  if (p.by_group && at >= *p.groups) return false;
  *j = p.joints[at];
  return j->valid && j->row0 + *strip * 16 < j->rows;
}

// Partial results of many shares: each of the 16 waves takes four at a time, 16
// lanes for the 16 rows' 4 values of one latent piece, so that a strip's
// partials (R / 4 workgroups of them) spread over many CUs: a CU takes some 10
// bytes a clock that its L2 does not have (256 shares of one sequence in 32
// workgroups took 23 us, in 128 6).
template <int R, int ROWS>
__global__ __launch_bounds__(1024) void absorbed_combine_many_kernel(const Absorbed p) {
  constexpr int STRIPS = ROWS / 16, ALL = R / 16, WAVES = 16;
  __shared__ float sm[WAVES][16], sl[WAVES][16];
  __shared__ float4 so[WAVES][16];
  Joint j;
  int strip;
  if (!find_joint<STRIPS>(p, blockIdx.x, &j, &strip)) return;
  const int lane = (int)threadIdx.x % kWave, wave = (int)threadIdx.x / kWave;
  const int row = lane % 16, piece = (int)blockIdx.y / 4, q = (int)blockIdx.y % 4;
  float m = -INFINITY, l = 0.0f;
  float4 acc = make_float4(0, 0, 0, 0);
  auto take = [&](float m2, float l2, const float4& v) {
    const float mn = fmaxf(m, m2);
    const float a = l == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(m - mn);
    const float w = l2 == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(m2 - mn);
    m = mn;
    l = l * a + l2 * w;
    acc.x = acc.x * a + v.x * w;
    acc.y = acc.y * a + v.y * w;
    acc.z = acc.z * a + v.z * w;
    acc.w = acc.w * a + v.w * w;
  };
#pragma unroll 4
  for (int64_t g = j.first + 4 * wave + lane / 16; g <= j.last; g += 4 * WAVES) {
    const int64_t slot = 2 * g + (g == j.first ? 1 : 0);
    const float ls = p.part_lse[slot * ROWS + strip * 16 + row];
    const float4 v = ((const float4*)p.part_o)[((slot * STRIPS + strip) * ALL + piece) * 64 + q * 16 + row];
    take(ls, ls == -INFINITY ? 0.0f : 1.0f, v);
  }
#pragma unroll
  for (int o = 16; o <= 32; o <<= 1) {
    const float4 v = make_float4(__shfl_xor(acc.x, o), __shfl_xor(acc.y, o), __shfl_xor(acc.z, o), __shfl_xor(acc.w, o));
    const float m2 = __shfl_xor(m, o), l2 = __shfl_xor(l, o);
    take(m2, l2, v);
  }
  if (lane < 16) {
    sm[wave][row] = m;
    sl[wave][row] = l;
    so[wave][row] = acc;
  }
  __syncthreads();
  if (wave != 0 || lane >= 16) return;
  for (int w = 1; w < WAVES; ++w) take(sm[w][row], sl[w][row], so[w][row]);
  const int at = j.row0 + strip * 16 + row;
  if (at >= j.rows) return;
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  const int64_t token = j.q0 + at / p.heads;
  const int h = at % p.heads;
  if (p.lse && blockIdx.y == 0) p.lse[token * p.heads + h] = l == 0.0f ? -INFINITY : (m + log2f(l)) * kLn2;
  *(uint2*)(p.out + token * p.ot + h * p.oh + 16 * piece + 4 * q) =
      make_uint2(pack_bf16(acc.x * inv, acc.y * inv), pack_bf16(acc.z * inv, acc.w * inv));
}

// Of a few shares: one workgroup a strip of 16 rows and 4 of its 1 KB pieces (64
// lanes x 4 values: 16 of the latent dimension for each row); its waves split
// the partials, each keeping a running maximum and sum, and meet in LDS.
template <int R, int ROWS>
__global__ __launch_bounds__(256) void absorbed_combine_kernel(const Absorbed p) {
  constexpr int STRIPS = ROWS / 16, ALL = R / 16, PIECES = 4, WAVES = 4;
  __shared__ float sm[WAVES][64], sl[WAVES][64];
  __shared__ float4 so[WAVES][PIECES][64];
  Joint j;
  int strip;
  if (!find_joint<STRIPS>(p, blockIdx.x, &j, &strip)) return;
  const int lane = (int)threadIdx.x % kWave, wave = (int)threadIdx.x / kWave;
  const int row = j.row0 + strip * 16 + lane % 16;
  const int64_t g0 = j.first, g1 = j.last;
  const int piece0 = (int)blockIdx.y * PIECES;

  float m = -INFINITY, l = 0.0f;
  float4 acc[PIECES];
#pragma unroll
  for (int k = 0; k < PIECES; ++k) acc[k] = make_float4(0, 0, 0, 0);
#pragma unroll 2
  for (int64_t g = g0 + wave; g <= g1; g += WAVES) {
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
  float top = -INFINITY, total = 0.0f, w[WAVES];
#pragma unroll
  for (int v = 0; v < WAVES; ++v) top = fmaxf(top, sm[v][lane]);
#pragma unroll
  for (int v = 0; v < WAVES; ++v) {
    // a wave that saw no key has l == 0 and nothing in its sums
    w[v] = sl[v][lane] == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(sm[v][lane] - top);
    total += w[v] * sl[v][lane];
  }
  if (row >= j.rows) return;
  const float inv = total == 0.0f ? 0.0f : 1.0f / total;
  const int64_t token = j.q0 + row / p.heads;
  const int h = row % p.heads;
  if (p.lse && piece0 == 0 && wave == 0 && lane < 16)
    p.lse[token * p.heads + h] = total == 0.0f ? -INFINITY : (top + log2f(total)) * kLn2;
  uint16_t* orow = p.out + token * p.ot + h * p.oh + 4 * (lane / 16);
  for (int k = wave; k < PIECES; k += WAVES) {
    float4 r = make_float4(0, 0, 0, 0);
#pragma unroll
    for (int v = 0; v < WAVES; ++v) {
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
  bool by_group;
  size_t joint_bytes, lse_bytes, bytes;
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
  const int64_t most = pl.groups * ((a->table_width > 0 ? ceil_div(a->table_width * a->cache.page_size, kAbsKeys) : 1) + kGroupCost);
  pl.shares = most < slots ? (most > 0 ? most : 1) : slots;
  pl.by_group = pl.groups <= pl.shares;
  pl.joint_bytes = 256 + (size_t)round_up((pl.by_group ? pl.groups : pl.shares) * (int64_t)sizeof(Joint), 256);
  pl.lse_bytes = (size_t)round_up(2 * pl.shares * pl.rows * 4, 256);
  pl.bytes = pl.joint_bytes + pl.lse_bytes + (size_t)(2 * pl.shares) * (size_t)pl.rows * (size_t)a->cache.latent_dim * 4;
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
  auto go = [&](auto rows_) {
    constexpr int ROWS = decltype(rows_)::value;
    const int64_t strips = (pl.by_group ? pl.groups : pl.shares) * (ROWS / 16);
    // Few strips: their partials are spread over more workgroups, of 16 waves each, which pays while there are no more than
    // two a CU. Attention and join, us, spread and not: 16 rows, 512 + 64, 256 workgroups (one sequence of 60000) 25.0,
    // 44.0, 512 (two of 30000) 27.9, 33.7, 1024 (four of 15000) 32.9, 27.7, 4096 (16 of 4000) 61, 24; 32 rows 512 32.2, 48.4,
    // 1024 37.5, 36.1; 64 rows 1024 44.9, 52.9, 2048 54, 41; latent 256 16 rows 512 21.4, 22.5, 1024 26.5, 19.9, 128 rows
    // 1024 43.9, 42.7.
    constexpr int64_t kSpread = 512;
    if constexpr (ROWS / 16 * (R / 4) <= kSpread) {  // one group's
      if (strips * (R / 4) <= kSpread) {
        hipLaunchKernelGGL((absorbed_combine_many_kernel<R, ROWS>), dim3((unsigned)strips, R / 4), dim3(1024), 0, stream, p);
        return;
      }
    }
    hipLaunchKernelGGL((absorbed_combine_kernel<R, ROWS>), dim3((unsigned)strips, R / 64), dim3(256), 0, stream, p);
  };
  if (pl.rows == 128)
    go(std::integral_constant<int, 128>{});
  else if (pl.rows == 64)
    go(std::integral_constant<int, 64>{});
  else if (pl.rows == 32)
    go(std::integral_constant<int, 32>{});
  else
    go(std::integral_constant<int, 16>{});
}

int check_absorbed(const fcmoe_absorbed_args* a) {
  if (!a) return fail(FCMOE_EINVAL, "absorbed_attention: NULL args");
  if (const int rc = check_latent_cache(a->cache, "absorbed_attention")) return rc;
  if (a->tokens < 0 || a->tokens > INT32_MAX || a->batch <= 0 || a->batch > (1 << 20) || a->heads <= 0 || a->heads > 65536 ||
      a->tokens * a->heads > INT32_MAX / 2 || a->table_width < 0 || a->table_width > INT32_MAX ||
      a->page_table_stride < 0)
    return fail(FCMOE_EINVAL, "absorbed_attention: bad shape");
  // units are counted in 32 bits a sequence
  if (ceil_div(a->tokens * a->heads, 16) + a->batch > INT32_MAX / (ceil_div(a->table_width * a->cache.page_size, kAbsKeys) + kGroupCost + 1))
    return fail(FCMOE_EINVAL, "absorbed_attention: too many rows for a page table of this reach");
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
  p.groups = (int*)a->workspace;
  p.joints = (Joint*)((char*)a->workspace + 256);
  p.by_group = pl.by_group;
  p.part_lse = (float*)((char*)a->workspace + pl.joint_bytes);
  p.part_o = (float*)((char*)a->workspace + pl.joint_bytes + pl.lse_bytes);
  p.shares = (int)pl.shares;
  // a page's rows, and the pages' distances, in 32 bits
  const auto small = [&](int64_t page_stride, int64_t row_stride, int64_t bytes) {
    return page_stride >= 0 && page_stride * bytes < ((int64_t)1 << 32) && row_stride < (1 << 24) &&
           (row_stride * p.c.page_size + 1024) * bytes < ((int64_t)1 << 31);
  };
  const int64_t elem = p.c.e4m3 ? 1 : 2;
  p.whole = p.c.page_size % 16 == 0 && small(p.c.latent_page_stride, p.c.latent_row_stride, elem) &&
            (!p.c.rope_dim || small(p.c.rope_page_stride, p.c.rope_row_stride, elem)) &&
            (!p.c.e4m3 || small(p.c.scale_page_stride, 1, 4));
  p.page_shift = -1;
  for (int i = 0; i <= 20; ++i)
    if (p.c.page_size == (int64_t)1 << i) p.page_shift = i;
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
