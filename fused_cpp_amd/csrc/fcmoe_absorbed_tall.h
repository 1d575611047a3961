// fcmoe_absorbed_tall.h -- the masked absorbed attention of row groups of 128, a
// workgroup each. Spans, segments, tiles and their loads are
// fcmoe_absorbed_kernel.h's.
//
// Each of the four waves takes 32 rows through both products on its own: S^T = K
// Q^T and O^T = V^T P^T in 32x32x16 products, a row one lane in both, so weights
// pass from one to the other in registers and the waves meet once a tile. A lane's
// Q (R + P values of a row, halved between the lanes l and l + 32) and O take
// (R + P) / 4 + R / 2 registers: 400 of a SIMD's 512 at 512 + 64, O all of the
// accumulation registers.
//
// A tile of 64 keys is 2 * 128 * 64 * (2 R + P) flops, 4352 clocks of the matrix
// units at 512 + 64, and as much of LDS in 16-bit rows: each wave reads every key
// row for S and every latent row for O, 1 KB a product. So the softmax has to hide
// among the products. A tile goes in four parts of R / 16 or (R + P) / 16
// products: S of keys 0 .. 31; S of keys 32 .. 63, with the weights of the
// first half taken between its products; P V of the first half, with the weights
// of the second; P V of the second.
//
// Clocks of a tile of 16-bit rows: 2050 + 1750 + 1540 + 1400, 500 for the two
// decisions whether a maximum has grown, 700 for the next tile's addresses. S's
// products, a chain of 36 on one accumulator, come 40 clocks apart instead of 32.
// Of 8-bit rows 9700: a product's 8 values a lane take four conversions of 8
// clocks, more than fits beside it. Two workgroups of 64 rows that share their
// keys' way (the other form) took 6100 and 7500 clocks of two CUs: two query
// tokens of 128 heads, 96 sequences, a window of 1000 of 8-bit rows 134 us ->
// 96; 60 nodes of 16 heads behind 32000 tokens 106 -> 88; 32 trees of up to 9
// nodes of 128 heads 276 -> 207.
#pragma once

#include "fcmoe_absorbed_kernel.h"

namespace fcmoe {

namespace {

constexpr int kTallRows = 128;

// As fcmoe_absorbed_kernel.h's written-out products: the compiler does not know them for MFMAs, so the waits stand
// here. WAIT: an ordinary instruction may just have written the fragment.
template <bool FIRST, bool WAIT>
__device__ __forceinline__ void tall_qk(v16f& acc, const v8bf& k, const v8bf& q) {
  if constexpr (FIRST && WAIT)
    asm volatile("s_nop 1\n\tv_mfma_f32_32x32x16_bf16 %0, %1, %2, 0" : "=&v"(acc) : "v"(k), "v"(q));
  else if constexpr (FIRST)
    asm volatile("v_mfma_f32_32x32x16_bf16 %0, %1, %2, 0" : "=&v"(acc) : "v"(k), "v"(q));
  else if constexpr (WAIT)
    asm volatile("s_nop 1\n\tv_mfma_f32_32x32x16_bf16 %0, %1, %2, %0" : "+v"(acc) : "v"(k), "v"(q));
  else
    asm volatile("v_mfma_f32_32x32x16_bf16 %0, %1, %2, %0" : "+v"(acc) : "v"(k), "v"(q));
}
template <bool WAIT>
__device__ __forceinline__ void tall_pv(v16f& acc, const v8bf& v, const v4u& w) {
  if constexpr (WAIT)
    asm volatile("s_nop 1\n\tv_mfma_f32_32x32x16_bf16 %0, %1, %2, %0" : "+a"(acc) : "v"(v), "v"(w));
  else
    asm volatile("v_mfma_f32_32x32x16_bf16 %0, %1, %2, %0" : "+a"(acc) : "v"(v), "v"(w));
}
// Zeros as a product of zeros: the compiler would hold a vector of them in ordinary registers.
__device__ __forceinline__ void tall_zero(v16f& acc) {
  const v4u zero = v4u{0, 0, 0, 0};
  asm volatile("s_nop 1\n\tv_mfma_f32_32x32x16_bf16 %0, %1, %1, 0" : "=&a"(acc) : "v"(zero));
}
// The last product into S has ended (STATES 24), or will have after four others.
template <int STATES>
__device__ __forceinline__ void tall_qk_done(v16f& s) {
  static_assert(STATES == 24 || STATES == 8, "");
  if constexpr (STATES == 24)
    asm volatile("s_nop 15\n\ts_nop 7" : "+v"(s));
  else
    asm volatile("s_nop 7" : "+v"(s));
}
// Products into O have ended, and what is read of it is read after this.
template <int TO>
__device__ __forceinline__ void tall_pv_done(v16f (&o)[TO]) {
  asm volatile("s_nop 15\n\ts_nop 7" ::: "memory");
#pragma unroll
  for (int t = 0; t < TO; ++t) asm volatile("" : "+a"(o[t]));
}
// The value of lane l ^ 32, without a register for the lane's number.
__device__ __forceinline__ float tall_other_half(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(lane_now() & 32 ? r[0] : r[1]);
}
// Any value, from here on: what is only set on some paths, and only used on those, is not kept from before them.
template <typename T>
__device__ __forceinline__ void tall_any(T& v) {
  asm volatile("" : "=v"(v));
}
template <typename T>
__device__ __forceinline__ void tall_any_uniform(T& v) {
  asm volatile("" : "=s"(v));
}
// One value to the compiler, which would pass its 16 parts around loops and branches one by one.
__device__ __forceinline__ void tall_whole(v16f& v) { asm volatile("" : "+a"(v)); }
template <typename T>
__device__ __forceinline__ void tall_here_one(T& v) {
  asm volatile("" : "+v"(v));
}
// These values are formed here, among the products around.
template <typename... T>
__device__ __forceinline__ void tall_here(T&... v) {
  (tall_here_one(v), ...);
}
// f(integral_constant<int, 0>), f(integral_constant<int, 1>) ..
template <int N, int I = 0, typename F>
__device__ __forceinline__ void tall_unroll(F f) {
  if constexpr (I < N) {
    f(std::integral_constant<int, I>{});
    tall_unroll<N, I + 1>(f);
  }
}
// Step j of `steps` takes items share(j) .. share(j + 1) of n.
constexpr int tall_share(int j, int steps, int n) { return j <= 0 ? 0 : j >= steps ? n : n * j / steps; }

// How the batch is divided. Evenly by units, as in the other form, most shares hold parts of two groups and leave a
// partial result of each: 128 rows of R binary32 values, which cost what some kPartCost tiles do, written and joined. Where
// groups are no more than shares and much alike, each is cut into parts of at most `part` tiles instead, a share each. 28
// batches (1 to 256 sequences of 512 to 131072 keys, 1 to 4 tokens of 128 heads, both types): never by parts, 192 groups of 18
// tiles take 121 us and 150 of 8 73, whole 89 and 54; all others are within 2%. kPartCost of 0 is as never, 3 as 6; 12
// gains once, 150 groups of 18 tiles of 16-bit rows (85 for 100).
struct TallSplit {
  int64_t units, shares;
  int part;  // 0: evenly
};
constexpr int kPartCost = 6;
__device__ __forceinline__ int tall_parts(int tiles, int part) { return (tiles + part - 1) / part; }
__device__ __forceinline__ TallSplit tall_split(const Absorbed& p) {
  int64_t units = 0, groups = 0;
  int high = 0, most = 0;
  for (int b0 = 0; b0 < p.batch; b0 += kWave) {
    const int b = b0 + lane_now();
    SeqSpan s{high, 0, 0, 0};
    if (b < p.batch) s = absorbed_span(p, b);
    high = follow(s, high);
    const int n = b < p.batch ? row_groups(p, s, kTallRows) : 0;
    if (n > 0) {
      const int tiles = key_tiles<true>(p, s, kTallRows);
      groups += n;
      units += (int64_t)n * (tiles + kGroupCost);
      most = max(most, tiles);
    }
  }
  groups = (int64_t)lane_value((uint64_t)wave_scan(groups), kWave - 1);
  units = (int64_t)lane_value((uint64_t)wave_scan(units), kWave - 1);
  most = __builtin_amdgcn_readlane(wave_scan_max(most), kWave - 1);
  TallSplit d{units, units < p.shares ? units : p.shares, 0};
  if (groups == 0 || groups > p.shares) return d;
  const int cuts = p.shares / (int)groups, part = (most + cuts - 1) / cuts;
  if (part + (part < most ? kPartCost : 0) > (int64_t)(units / p.shares) + kPartCost) return d;
  d.part = part;
  d.units = count_items(
      p.batch, [&](int b) { return absorbed_span(p, b); },
      [&](const SeqSpan& q) { return (int64_t)row_groups(p, q, kTallRows) * tall_parts(key_tiles<true>(p, q, kTallRows), part); });
  d.shares = d.units;  // at most groups * cuts
  return d;
}
// The part that is unit u.
__device__ __forceinline__ Segment tall_segment(const Absorbed& p, int64_t u, int part) {
  Segment s;
  int64_t before;
  s.b = find_sequence(
      p.batch, u, [&](int b) { return absorbed_span(p, b); },
      [&](const SeqSpan& q) { return (int64_t)row_groups(p, q, kTallRows) * tall_parts(key_tiles<true>(p, q, kTallRows), part); }, &s.seq, &before);
  s.tiles = key_tiles<true>(p, s.seq, kTallRows);
  const uint32_t rel = (uint32_t)(u - before), parts = (uint32_t)tall_parts(s.tiles, part), group = rel / parts;
  const uint32_t at = rel - group * parts;
  s.units = 1;
  s.t_begin = uniform((int)((uint64_t)(uint32_t)s.tiles * at / parts));
  s.t_end = uniform((int)((uint64_t)(uint32_t)s.tiles * (at + 1) / parts));
  s.row0 = uniform((int)group * kTallRows);
  s.ahead = uniform((int)(parts - 1 - at));
  return s;
}

template <int R, int P, bool F8>
__global__ __launch_bounds__(256, 1) void absorbed_tall_kernel(const Absorbed p) {
  using T = Tile<R, P, F8>;
  using S = Stager<R, P, F8>;
  constexpr int GROUP = kTallRows;
  constexpr int KS = (R + P) / 16, RS = R / 16, TO = R / 32;  // 32x32x16 steps of a key half; d tiles
  constexpr int SCL = 2 * T::BYTES, ONES = SCL + (F8 ? 2 * 256 : 0);
  // of each row the four words of its tree mask that hold the next tile's bits, then its depth
  constexpr int TREE = ONES + (F8 ? 256 : 0), DEPTH = TREE + 16 * GROUP, BAD = DEPTH + 4 * GROUP, END = BAD + 16;
  __shared__ __align__(1024) uint8_t smem[END];
  lds_u8* lds = (lds_u8*)smem;
  const int wave = wave_index();
  int64_t units, shares;
  int part;
  {
    const Absorbed a = args_now();
    if (a.zero_tail)
      zero_uncovered(a.q_starts, a.batch, a.tokens, a.heads, R, a.out, a.ot, a.oh, a.lse, blockIdx.x, gridDim.x);
    const TallSplit d = tall_split(a);
    units = d.units, shares = d.shares, part = d.part;
  }
  const int64_t g = blockIdx.x;
  if (g >= shares) {
    if (!p.by_group && threadIdx.x == 0) p.joints[g].valid = 0;
    if (g == 0 && threadIdx.x == 0) *p.groups = 0;  // no units at all
    return;
  }
  if (g == 0 && p.by_group) {
    const int64_t n = count_items(
        p.batch, [&](int b) { return absorbed_span(p, b); }, [&](const SeqSpan& q) { return (int64_t)row_groups(p, q, GROUP); });
    if (threadIdx.x == 0) *p.groups = (int)n;
  }
  if (F8 && threadIdx.x < 64) *(lds_f32*)(lds + ONES + 4 * threadIdx.x) = 1.0f;
  int64_t u = share_begin(units, g, shares);  // a part: the share itself
  int left = share_size(units, g, shares);
  int joint = 0;  // a joint of this share was written
  const float c2 = uniform(p.scale * kLog2e);

  while (left > 0) {
    const Absorbed a = args_now();
    const Segment sg = part ? tall_segment(a, u, part) : next_segment<true>(a, GROUP, u, left);
    const SeqSpan& seq = sg.seq;
    const int rows = seq.n * a.heads;
    const bool whole_group = sg.t_begin == 0 && sg.t_end == sg.tiles;
    // slots and joints as in the other form
    const int64_t slot = 2 * g + (sg.t_begin == 0 ? 1 : 0);
    u += sg.units;
    left -= sg.units;
    if (sg.t_begin == sg.t_end) continue;  // the group's tiles begin in the next share
    if (sg.t_begin == 0 && (a.by_group || !whole_group)) {
      joint = uniform(joint | (whole_group ? 0 : 1));
      int64_t at = g;
      if (a.by_group)
        at = sg.row0 / GROUP + count_items(
                                   sg.b, [&](int b) { return absorbed_span(a, b); },
                                   [&](const SeqSpan& q) { return (int64_t)row_groups(a, q, GROUP); });
      if (wave == 0 && lane_now() == 0) {
        const int64_t last = share_of(opaque_uniform(units), u - sg.units + sg.ahead, shares);
        a.joints[at] = Joint{seq.q0, rows, sg.row0, (int)g, (int)last, whole_group ? 0 : 1};
      }
    }
    // query token and head of row `at` of this wave's 32 (rows past the last repeat it and are not stored)
    const int row0 = sg.row0 + 32 * wave;
    const bool live = row0 < rows;
    auto my_row = [&](int at, int& i, int& h) {
      const int row = min(row0 + at, rows - 1), heads = args_now().heads;
      i = row / heads;
      h = row - i * heads;
    };
    // keys that all rows of the wave see: those before lim_min, and of these the ones before `sinks` and from lo_max on
    const Seen seen = seen_by(a, seq, sg.row0 / a.heads, min((sg.row0 + GROUP - 1) / a.heads, seq.n - 1));
    const int base = seq.len - seq.n;
    const int lim_min = a.tree ? max(base, 0) : absorbed_limit(seq, min(row0, rows - 1) / a.heads);
    const int lo_max = window_low(base + (a.tree ? seq.n - 1 : min((row0 + 31) / a.heads, seq.n - 1)), a.window);
    const int t_end = min(sg.t_end, seen.tiles);
    const bool any = sg.t_begin < t_end;

    S st;
    st.begin(a, seen.hi, sg.b, wave, 0);
    auto fetch = [&](int t) { st.template fetch<true>(args_now(), seen.tile(t), seen.head, seen.lo); };
    if (any) fetch(sg.t_begin);

    // Q: B operand, column lane % 32. bf16 rows: values 16 ks + 8 (lane / 32) ..; 8-bit rows are read 16 values a
    // lane, two steps at once: 32 (ks / 2) + 16 (lane / 32) + 8 (ks % 2) ..
    v8bf qf[KS];
    {
      const int ln = lane_now(), half = ln / 32;
      int i, h;
      my_row(ln % 32, i, h);
      const uint16_t* ql = a.ql + (seq.q0 + i) * a.qlt + h * a.qlh;
      const uint16_t* qr = P ? a.qr + (seq.q0 + i) * a.qrt + h * a.qrh : nullptr;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const int k = ks < RS ? ks : ks - RS;
        const int d = F8 ? 32 * (k / 2) + 16 * half + 8 * (k % 2) : 16 * k + 8 * half;
        qf[ks] = *(const v8bf*)((ks < RS ? ql : qr) + d);
      }
    }
    lds_only_barrier();  // the last segment's accesses to LDS have ended
    if (wave == 0) *(lds_i32*)(lds + BAD) = 0;
    lds_only_barrier();
    if (any) {
      st.start(a, lds + BAD);
      st.load_all(lds);
      st.template parts<true>(a);
      st.finish(lds, lds + SCL);
      if (sg.t_begin + 1 < t_end) fetch(sg.t_begin + 1);
    }
    // what the loads of a tile need, formed at the end of the tile before the one they go among
    auto start = [&](int t) {
      st.whole = false;
      tall_any(st.lat);
      tall_any_uniform(st.wl), tall_any_uniform(st.wr), tall_any_uniform(st.ws);
      tall_any_uniform(st.step), tall_any_uniform(st.rstep);
      if (t >= t_end) return;
      const Absorbed b = args_now();
      const int first = seen.tile(t) * kAbsKeys, last = first + kAbsKeys;
      st.whole = b.whole && (last <= seen.head || (first >= seen.lo && last <= seen.hi));
      if (st.whole)
        st.start_whole(b, lds + BAD);
      else
        st.start(b, lds + BAD);
    };
    // The words of the rows' tree masks from the one on that has the first bit of
    // tile t, straight to LDS: they arrive with the tile, and words past a mask's
    // end are zeros. Lane l: rows l / 4 and 16 + l / 4 of the wave's, word l % 4.
    auto tree_word = [&](int t) { return max(seen.tile(t) * kAbsKeys - base, 0) >> 5; };
    auto tree_load = [&](int t) {
      const Absorbed b = args_now();
      if (!b.tree || (seen.tile(t) + 1) * kAbsKeys <= base) return;
      const int ln = lane_now(), word = tree_word(t) + ln % 4;
      const __amdgpu_buffer_rsrc_t masks = __builtin_amdgcn_make_buffer_rsrc((void*)b.tree, (short)0, (int)b.tree_bytes, kBufWord3);
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        int i, h;
        my_row(16 * k + ln / 4, i, h);
        const uint32_t at = word < b.tree_words ? (uint32_t)(((seq.q0 + i) * b.tree_stride + word) * 4) : 0xffffff00u;
        load_lds4(masks, lds + TREE + 512 * wave + 256 * k, at);
      }
    };
    if (any) {
      start(sg.t_begin + 1);
      tree_load(sg.t_begin);
      const Absorbed b = args_now();
      const int ln = lane_now();
      if (b.tree && ln < 32) {
        int i, h;
        my_row(ln, i, h);
        load_lds4(__builtin_amdgcn_make_buffer_rsrc((void*)b.tree_depths, (short)0, (int)(b.tokens * 4), kBufWord3), lds + DEPTH + 128 * wave,
                  (uint32_t)((seq.q0 + i) * 4));
      }
    }

    // m: a row's reference point in units of log2, -inf while it has seen no key; mz the same with 0 for that. It
    // only has to be near the maximum, so it stays until the weights of a tile's half show that some row has grown far past
    // it (a lane's sum beyond 2^14, far inside binary32 and bf16) and they are taken anew.
    float m = -INFINITY, mz = 0.0f, l = 0.0f;  // l: over this lane's keys
    bool unset = true;
    v16f o[TO];
#pragma unroll
    for (int t = 0; t < TO; ++t) tall_zero(o[t]);

    for (int tile = sg.t_begin; any && tile < t_end; ++tile) {
      const int buf = (tile - sg.t_begin) & 1;
      const bool more = tile + 1 < t_end;
      loads_barrier();  // the tile has landed; everyone is done with the other buffer
      const bool whole = st.whole;  // the next tile
      const lds_u8* kb = lds + buf * T::BYTES;
      lds_u8* next = lds + (buf ^ 1) * T::BYTES;
      const lds_u8* scl = lds + SCL + buf * 256;
      lds_u8* next_scl = lds + SCL + (buf ^ 1) * 256;
      const int first_key = seen.tile(tile) * kAbsKeys;
      const bool masked = first_key + kAbsKeys > lim_min || (first_key < lo_max && first_key + kAbsKeys > seen.head);
      if (!live) {
        if (whole) {
          const uint64_t wl = (uint64_t)uniform((int64_t)st.wl), wr = (uint64_t)uniform((int64_t)st.wr);
          const uint32_t step = (uint32_t)uniform((int)st.step), rstep = (uint32_t)uniform((int)st.rstep);
          const int tl = lane_now(), part = tl / T::UNITS;
          const int lane16 = ((tl % T::UNITS) ^ swz_key<F8>(part)) * 16, lane_row = S::KPL > 1 ? part * (int)step : 0;
          tall_unroll<S::WLOADS + S::WRLOADS>(
              [&](auto u_) { st.template load_whole<decltype(u_)::value>(next, wl, wr, step, rstep, lane16, lane_row, wave, 0); });
          st.scales_whole(next_scl);
        } else if (more) {
          st.load_all(next);
          st.template parts<true>(args_now());
          st.finish(next, next_scl);
        }
        if (tile + 2 < t_end) fetch(tile + 2);
        if (more) start(tile + 2);
        continue;
      }
      // What depends on the lane is formed here, in each tile, and addresses where they are used, an XOR each.
      const int tl = lane_now(), half = tl / 32, tc = tl % 32;
      const int ka = tc * T::LROW + ((half ^ swz_key<F8>(tc)) * 16);
      const int kra = T::ROPE + tc * T::RROW + ((half ^ swz_rope<F8>(tc)) * 16);
      // One 16-byte read of K a step (an 8-bit row's serves two), AHEAD before its products.
      constexpr int READS = F8 ? KS : 2 * KS, PER = READS / 2, AHEAD = F8 ? 2 : 4, RING = AHEAD + 1;
      v4i kf[RING];
      auto k_read = [&](auto n_) {
        constexpr int n = decltype(n_)::value, hf = n / PER, k = n % PER, LS = F8 ? RS / 2 : RS;
        constexpr int WIN = F8 ? 4 : 8;  // reads of the window of units that the swizzle stays in
        if constexpr (k < LS)
          kf[n % RING] = lds_v4i(kb + (ka ^ ((k % WIN) << 5)) + k / WIN * (WIN * 32) + hf * 32 * T::LROW);
        else
          kf[n % RING] = lds_v4i(kb + (kra ^ ((k - LS) << 5)) + hf * 32 * T::RROW);
      };
      // V^T reads. 16-bit rows: 4 keys x 16 values a group of 16 lanes, keys 4 (lane / 32) .. and 8 beyond; 8-bit rows:
      // both sets of keys at once.
      int va;
      {
        const int g16 = tl / 16, i = tl % 16;
        if constexpr (F8) {
          const int key = 4 * half + i / 2 % 4 + 8 * (i / 8);
          va = key * T::LROW + (((g16 & 1) ^ swz_key<F8>(key)) * 16) + (i & 1) * 8;
        } else {
          const int key = 4 * half + i / 4, e = 2 * (g16 & 1) + i % 4 / 2;
          va = key * T::LROW + ((e ^ swz_key<F8>(key)) * 16) + (i & 1) * 8;
        }
      }
      constexpr int VN = 4 * TO, VAHEAD = F8 ? 3 : 4, VRING = VAHEAD + 1;
      v4s vlo[VRING], vhi[VRING];
      v2i v8[VRING];
      auto v_read = [&](auto n_) {
        constexpr int n = decltype(n_)::value, s4 = n / TO, t = n % TO;
        if constexpr (F8) {
          v8[n % VRING] = read_tr8(kb + (va ^ ((t & 3) << 5)) + (t >> 2) * 128 + 16 * s4 * T::LROW);
        } else {
          vlo[n % VRING] = read_tr16(kb + (va ^ ((t & 3) << 6)) + (t >> 2) * 256 + 16 * s4 * T::LROW);
          vhi[n % VRING] = read_tr16(kb + (va ^ (((t & 3) ^ 2) << 6)) + (t >> 2) * 256 + (16 * s4 + 8) * T::LROW);  // keys + 8: swizzle bit 3
        }
      };
      v16f s[2];
      v8bf wide[2];  // 8-bit rows: fragments widened one product ahead
      auto widen_k = [&](auto j_) {
        constexpr int j = decltype(j_)::value;
        const v4i w = kf[j / 2 % RING];
        wide[j & 1] = j & 1 ? widen_e4m3(v2i{w[2], w[3]}) : widen_e4m3(v2i{w[0], w[1]});
      };
      // Products j0 .. j0 + KS - 1 of S; between(k) follows the k-th.
      auto scores = [&](auto hf_, auto between) {
        constexpr int hf = decltype(hf_)::value;
        tall_unroll<KS>([&](auto ks_) {
          constexpr int ks = decltype(ks_)::value, j = hf * KS + ks;
          if constexpr (F8) {
            if constexpr (j % 2 == 0 && j / 2 + AHEAD < READS) k_read(std::integral_constant<int, j / 2 + AHEAD>{});
          } else {
            if constexpr (j + AHEAD < READS) k_read(std::integral_constant<int, j + AHEAD>{});
          }
          __builtin_amdgcn_sched_barrier(0);
          if constexpr (F8)
            tall_qk<ks == 0, true>(s[hf], wide[j & 1], qf[ks]);
          else
            tall_qk<ks == 0, false>(s[hf], __builtin_bit_cast(v8bf, kf[j % RING]), qf[ks]);
          __builtin_amdgcn_sched_barrier(0);
          if constexpr (F8 && j + 1 < 2 * KS) widen_k(std::integral_constant<int, j + 1>{});
          between(ks_);
        });
      };
      // Lane: row tc, keys 32 hf + 8 (i / 4) + 4 half + i % 4 of the tile in s[hf][i].
      auto mask = [&](auto hf_) {
        constexpr int hf = decltype(hf_)::value;
        const Absorbed b = args_now();
        const int ml = lane_now(), mh = ml / 32, j0 = first_key + 32 * hf + 4 * mh;
        int pos, up, h;
        my_row(ml % 32, pos, h);
        uint32_t bits = 0;  // bit k: key j0 + k is a node that the row sees
        if (b.tree) {
          const int off = j0 - base - 32 * tree_word(tile);
          if (off > -32) {
            const lds_u8* w = lds + TREE + (32 * wave + ml % 32) * 16 + max(off, 0) / 32 * 4;
            const uint32_t lo = *(const __attribute__((address_space(3))) uint32_t*)w;
            const uint32_t hi = *(const __attribute__((address_space(3))) uint32_t*)(w + 4);
            bits = off < 0 ? lo << -off : __builtin_amdgcn_alignbit(hi, lo, off);
          }
          pos = node_depth(seq, *(lds_i32*)(lds + DEPTH + (32 * wave + ml % 32) * 4));
          up = base;
        } else {
          up = absorbed_limit(seq, pos);
        }
        // bit k: the row sees key j0 + k
        auto below = [](int n) { return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1; };
        const uint32_t before = below(up - j0), low = below(window_low(base + pos, b.window) - j0);
        const uint32_t sinks = below((int)clamp64((int64_t)b.sinks - j0, 0, 32));
        const uint32_t sees = (before & (~low | sinks)) | (bits & ~before & below(seq.len - j0));
#pragma unroll
        for (int g4 = 0; g4 < 4; ++g4) {
          v4f sc = v4f{1, 1, 1, 1};
          if constexpr (F8) sc = lds_v4f(scl + (32 * hf + 8 * g4 + 4 * mh) * 4);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t all = (uint32_t)((int)(sees << (31 - 8 * g4 - i)) >> 31);  // the bit in every place
            const uint32_t v = __float_as_uint(F8 ? s[hf][4 * g4 + i] * sc[i] : s[hf][4 * g4 + i]);
            s[hf][4 * g4 + i] = __uint_as_float((v & all) | (0xff800000u & ~all));
          }
        }
        asm volatile("" : "+v"(s[hf]));
      };
      // The weights of a half in 16 operations: of each group of four keys the exponents, two exponentials twice, and
      // their sum and rounding to bf16 (an 8-bit cache's scales, which differ by token, go into them before it; the sum
      // is of what they were: as in the other form).
      v4u w[2][2];
      float e[4], sum = 0.0f;
      v4f sc[2], by[2];
      const lds_u8* in_scores = masked ? (const lds_u8*)lds + ONES : scl;  // a masked tile's scores have the scales already
      auto scales_read = [&](auto hf_, auto g_) {
        constexpr int hf = decltype(hf_)::value, g4 = decltype(g_)::value;
        if constexpr (F8 && g4 < 4) {
          const int at = (32 * hf + 8 * g4 + 4 * (lane_now() / 32)) * 4;
          by[g4 & 1] = lds_v4f(in_scores + at);
          sc[g4 & 1] = lds_v4f(scl + at);
        }
      };
      auto weigh = [&](auto hf_, auto op_) {
        constexpr int hf = decltype(hf_)::value, op = decltype(op_)::value, g4 = op / 4, kind = op % 4;
        if constexpr (kind == 0) {
          if constexpr (F8) {
#pragma unroll
            for (int i = 0; i < 4; ++i) s[hf][4 * g4 + i] *= by[g4 & 1][i];
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) s[hf][4 * g4 + i] = __builtin_fmaf(s[hf][4 * g4 + i], c2, -mz);
        } else if constexpr (kind < 3) {
#pragma unroll
          for (int i = 2 * kind - 2; i < 2 * kind; ++i) e[i] = __builtin_amdgcn_exp2f(s[hf][4 * g4 + i]);
          if constexpr (kind == 1) scales_read(hf_, std::integral_constant<int, g4 + 1>{});
          tall_here(e[2 * kind - 2], e[2 * kind - 1]);
        } else {
          sum += (e[0] + e[1]) + (e[2] + e[3]);
          if constexpr (F8) {
#pragma unroll
            for (int i = 0; i < 4; ++i) e[i] *= sc[g4 & 1][i];
          }
          uint32_t w0 = pack_bf16(e[0], e[1]), w1 = pack_bf16(e[2], e[3]);
          tall_here(w0, w1, sum);
          w[hf][g4 / 2][2 * (g4 % 2)] = w0;
          w[hf][g4 / 2][2 * (g4 % 2) + 1] = w1;
        }
      };
      // some row's maximum has grown far past its reference point: rescale, and the half's weights anew
      auto settle = [&](auto hf_) {
        constexpr int hf = decltype(hf_)::value;
        if (unset || __any(sum > 16384.0f)) {
          float top = s[hf][0];
#pragma unroll
          for (int i = 1; i < 16; ++i) top = fmaxf(top, s[hf][i]);
          top = fmaxf(top, tall_other_half(top));
          const float mn = fmaxf(m, mz + top), r = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - mn);
          const float mnz = mn == -INFINITY ? 0.0f : mn, by = mnz - mz;
          if (__any(m != -INFINITY)) {  // else O is still zeros
            tall_pv_done<TO>(o);
#pragma unroll
            for (int t = 0; t < TO; ++t) {
#pragma unroll
              for (int i = 0; i < 16; ++i) o[t][i] *= r;
              tall_whole(o[t]);  // back before the next: few ordinary registers pass between
              __builtin_amdgcn_sched_barrier(0);
            }
          }
          m = mn, mz = mnz;
          l *= r;
          sum = 0.0f;
#pragma unroll
          for (int g4 = 0; g4 < 4; ++g4) {
            v4f again = v4f{1, 1, 1, 1};
            if constexpr (F8) again = lds_v4f(scl + (32 * hf + 8 * g4 + 4 * (lane_now() / 32)) * 4);
            float v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = __builtin_amdgcn_exp2f(s[hf][4 * g4 + i] - by);
            sum += (v[0] + v[1]) + (v[2] + v[3]);
            w[hf][g4 / 2][2 * (g4 % 2)] = pack_bf16(v[0] * again[0], v[1] * again[1]);
            w[hf][g4 / 2][2 * (g4 % 2) + 1] = pack_bf16(v[2] * again[2], v[3] * again[3]);
          }
          unset = __any(m == -INFINITY);
        }
        l += sum;
        sum = 0.0f;
        asm volatile("s_nop 1" : "+v"(w[hf][0]), "+v"(w[hf][1]));  // before a product reads them
      };
      constexpr std::integral_constant<int, 0> kFirst{};
      constexpr std::integral_constant<int, 1> kSecond{};

      tall_unroll<AHEAD>([&](auto n_) { k_read(n_); });
      if constexpr (F8) widen_k(kFirst);
      // the next tile's loads go among the products, of a whole one as straight-line code
      if (whole) {
        const uint64_t wl = (uint64_t)uniform((int64_t)st.wl), wr = (uint64_t)uniform((int64_t)st.wr);
        const uint32_t step = (uint32_t)uniform((int)st.step), rstep = (uint32_t)uniform((int)st.rstep);
        const int part = tl / T::UNITS;
        const int lane16 = ((tl % T::UNITS) ^ swz_key<F8>(part)) * 16, lane_row = S::KPL > 1 ? part * (int)step : 0;
        constexpr int LOADS = S::WLOADS + S::WRLOADS;
        scores(kFirst, [&](auto ks_) {
          constexpr int ks = decltype(ks_)::value, at = tall_share(ks, KS, LOADS);
          tall_unroll<tall_share(ks + 1, KS, LOADS) - at>([&](auto k_) {
            st.template load_whole<at + decltype(k_)::value>(next, wl, wr, step, rstep, lane16, lane_row, wave, 0);
          });
        });
        st.scales_whole(next_scl);
      } else {
        scores(kFirst, [&](auto ks_) {
          constexpr int ks = decltype(ks_)::value, at = tall_share(ks, KS, 16);
          if (more) tall_unroll<tall_share(ks + 1, KS, 16) - at>([&](auto k_) { st.load(next, at + decltype(k_)::value); });
        });
        asm volatile("s_nop 11" : "+v"(s[0]));  // the branches around may pass what follows here by a register of S
      }
      __builtin_amdgcn_sched_barrier(0);
      if (masked) {
        tall_qk_done<24>(s[0]);
        mask(kFirst);
      }
      scores(kSecond, [&](auto ks_) {
        constexpr int ks = decltype(ks_)::value;
        if constexpr (ks == 0) scales_read(kFirst, kFirst);
        if constexpr (ks == 3) tall_qk_done<8>(s[0]);
        if constexpr (ks >= 4 && ks < KS - 1) {
          constexpr int at = tall_share(ks - 4, KS - 5, 16);
          tall_unroll<tall_share(ks - 3, KS - 5, 16) - at>([&](auto k_) { weigh(kFirst, std::integral_constant<int, at + decltype(k_)::value>{}); });
        }
        if constexpr (ks >= KS - VAHEAD) v_read(std::integral_constant<int, ks - (KS - VAHEAD)>{});
      });
      __builtin_amdgcn_sched_barrier(0);
      settle(kFirst);
      if (masked) {
        tall_qk_done<24>(s[1]);
        mask(kSecond);
      }
      auto values = [&](auto hf_, auto between) {
        constexpr int hf = decltype(hf_)::value;
        tall_unroll<2 * TO>([&](auto k_) {
          constexpr int k = decltype(k_)::value, n = 2 * TO * hf + k;
          if constexpr (n + VAHEAD < VN) v_read(std::integral_constant<int, n + VAHEAD>{});
          const v8bf vf = F8 ? widen_e4m3(v8[n % VRING]) : join_tr16(vlo[n % VRING], vhi[n % VRING]);
          __builtin_amdgcn_sched_barrier(0);
          tall_pv<F8>(o[n % TO], vf, w[hf][k / TO]);
          __builtin_amdgcn_sched_barrier(0);
          between(k_);
        });
      };
      values(kFirst, [&](auto k_) {
        constexpr int k = decltype(k_)::value;
        if constexpr (k == 0) scales_read(kSecond, kFirst);
        if constexpr (k == 3) tall_qk_done<8>(s[1]);
        if constexpr (k >= 4 && k < 2 * TO - 1) {
          constexpr int at = tall_share(k - 4, 2 * TO - 5, 16);
          tall_unroll<tall_share(k - 3, 2 * TO - 5, 16) - at>([&](auto i_) { weigh(kSecond, std::integral_constant<int, at + decltype(i_)::value>{}); });
        }
      });
      __builtin_amdgcn_sched_barrier(0);
      settle(kSecond);
      if constexpr (P > 0) {
#pragma unroll
        for (int i = 0; i < T::RLOADS; ++i) tall_any(st.part[i]);
      }
      if constexpr (F8) tall_any(st.scale);
      if (more && !whole) st.template parts<true>(args_now());  // not before: there are no registers for them
      tall_any(st.id), tall_any(st.in);
      if (tile + 2 < t_end) fetch(tile + 2);
      values(kSecond, [](auto) {});
      if (more) {
        if (!whole) st.finish(next, next_scl);
        start(tile + 2);
        tree_load(tile + 1);
      }
    }

    tall_pv_done<TO>(o);
    if (!live) continue;
    const Absorbed z = args_now();
    const int el = lane_now(), half = el / 32;
    l += tall_other_half(l);
    if (*(lds_i32*)(lds + BAD) != 0) l = __uint_as_float(0x7fc00000u);
    // a row that sees no key has a sum of 0: its output is 0 and its lse -inf
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    if (opaque_uniform(sg.t_begin) != 0 || sg.t_end != sg.tiles) {
      // as the launch that joins them reads them: strips of 16 rows, pieces of 16 d x 16 rows, 4 values of one row a lane
      const int row = 32 * wave + el % 32;
      if (el < 32) z.part_lse[slot * GROUP + row] = l == 0.0f ? -INFINITY : m + log2f(l);
      float4* po = (float4*)z.part_o + (slot * (GROUP / 16) + row / 16) * (R / 16) * 64 + 16 * half + row % 16;
#pragma unroll
      for (int t = 0; t < TO; ++t)
#pragma unroll
        for (int k = 0; k < 4; ++k)
          po[(2 * t + k / 2) * 64 + k % 2 * 32] = make_float4(o[t][4 * k] * inv, o[t][4 * k + 1] * inv, o[t][4 * k + 2] * inv, o[t][4 * k + 3] * inv);
      continue;
    }
    if (row0 + el % 32 >= rows) continue;
    int qi, h;
    my_row(el % 32, qi, h);
    const int64_t token = seq.q0 + qi;
    if (z.lse && el < 32) z.lse[token * z.heads + h] = l == 0.0f ? -INFINITY : __builtin_fmaf(m, kLn2, logf(l));
    // Lanes l and l + 32 hold 4 values each of 8 neighbouring ones: swapped, l has 8 of the first of two eights and l + 32
    // of the second, a store of 16 bytes each where rows start at multiples of that.
    uint16_t* orow = z.out + token * z.ot + h * z.oh;
    const bool sixteen = ((z.ot | z.oh) & 7) == 0 && ((uintptr_t)z.out & 15) == 0;
#pragma unroll
    for (int t = 0; t < TO; ++t) {
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int k = 0; k < 4; k += 2) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = pack_bf16(o[t][4 * k + 2 * i] * inv, o[t][4 * k + 2 * i + 1] * inv);
        if (sixteen) {
          const auto a0 = __builtin_amdgcn_permlane32_swap(w[0], w[2], false, false), a1 = __builtin_amdgcn_permlane32_swap(w[1], w[3], false, false);
          *(uint4*)(orow + 32 * t + 8 * (k + half)) = make_uint4(a0[0], a1[0], a0[1], a1[1]);
        } else {
          *(uint2*)(orow + 32 * t + 8 * k + 4 * half) = make_uint2(w[0], w[1]);
          *(uint2*)(orow + 32 * t + 8 * (k + 1) + 4 * half) = make_uint2(w[2], w[3]);
        }
      }
    }
  }
  if (!args_now().by_group && !joint && wave == 0 && lane_now() == 0) args_now().joints[g].valid = 0;
}

template <int R, int P, bool F8>
void tall_launch(const Absorbed& p, const AbsPlan& pl, hipStream_t stream) {
  hipLaunchKernelGGL((absorbed_tall_kernel<R, P, F8>), dim3((unsigned)pl.shares), dim3(256), 0, stream, p);
}

}  // namespace

}  // namespace fcmoe
