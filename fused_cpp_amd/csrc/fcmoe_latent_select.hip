// fcmoe_latent_select.hip -- what lies between attentions over a part of a
// latent cache: the masks of a tree of drafted tokens, the positions that a
// sequence keeps, and the move of cached rows.
#include "fcmoe_internal.h"
#include "fcmoe_latent.h"

namespace fcmoe {

namespace {

typedef __attribute__((address_space(3))) int32_t lds_i32;

// ---- trees of drafted tokens --------------------------------------------------
//
// Node i of a sequence's n has parent[i] < i among them, or none. Its mask has
// the bits of its line up to the root, its own included; its depth is the length
// of that line but one. A workgroup a sequence: the parents go to LDS, and each
// thread walks the line of one (node, mask word) pair until it lies before that
// word: bound by the latency of a line's LDS reads.
constexpr int kTreeNodes = 1024, kTreeThreads = 256;

struct Tree {
  const int32_t* parents;
  const int32_t* starts;
  int64_t tokens;
  int batch, words;
  uint64_t* masks;  // [tokens, words]
  int32_t* depths;
};

__global__ __launch_bounds__(kTreeThreads) void draft_tree_kernel(const Tree p) {
  __shared__ int parent[kTreeNodes];
  __shared__ int tops[kTreeThreads / kWave];
  const int b = (int)blockIdx.x, tid = (int)threadIdx.x;
  // the sequence's span: a start below an earlier one counts as that one
  int top = 0;
  for (int k = tid; k <= b; k += kTreeThreads) top = max(top, (int)clamp64(p.starts[k], 0, p.tokens));
#pragma unroll
  for (int o = 1; o < kWave; o <<= 1) top = max(top, __shfl_xor(top, o));
  if (tid % kWave == 0) tops[tid / kWave] = top;
  __syncthreads();
  for (int w = 0; w < kTreeThreads / kWave; ++w) top = max(top, tops[w]);
  const int64_t q0 = top, end = max((int64_t)top, clamp64(p.starts[b + 1], 0, p.tokens));
  // tokens before the first and behind the last sequence see nothing
  auto clear = [&](int64_t from, int64_t to) {
    for (int64_t k = from * p.words + tid; k < to * p.words; k += kTreeThreads) p.masks[k] = 0;
    for (int64_t k = from + tid; k < to; k += kTreeThreads) p.depths[k] = 0;
  };
  if (b == 0) clear(0, q0);
  if (b == p.batch - 1) clear(end, p.tokens);
  const int64_t n = end - q0;
  const int nodes = (int)(n < 64 * p.words ? n : 64 * p.words);  // nodes past them see the context alone
  if (nodes < n) clear(q0 + nodes, end);
  for (int i = tid; i < nodes; i += kTreeThreads) {
    const int v = p.parents[q0 + i];
    parent[i] = v >= 0 && v < i ? v : -1;
  }
  __syncthreads();
  for (int k = tid; k < nodes * p.words; k += kTreeThreads) {
    const int i = k / p.words, w = k - i * p.words;
    uint64_t bits = 0;
    int depth = -1;
    for (int at = i; at >= (w == 0 ? 0 : 64 * w); at = parent[at]) {
      if (at < 64 * w + 64) bits |= (uint64_t)1 << (at % 64);
      ++depth;
    }
    p.masks[(q0 + i) * p.words + w] = bits;
    if (w == 0) p.depths[q0 + i] = depth;
  }
}

// ---- the positions that stay ----------------------------------------------------
//
// Of a sequence of len > keep tokens: its first `sinks`, its last `recent`, and of
// the others the keep - sinks - recent with the largest weights, ties to the
// lower position (NaN counts as the largest, -0 as 0), in ascending order.
//
// The m-th largest weight is found from its bits, as integers in the same
// order, 11, 11 and 10 at a time from the top: a histogram in LDS of those that
// agree so far, then the bin that the m-th falls into. What stays is counted wave
// by wave and written in order.
//
// A workgroup holds kSlice weights in registers. Sequences of up to that many columns
// are one launch, a workgroup each, that reads the weights once. Longer ones are cut into
// slices, a workgroup each, in three launches (a CU alone takes some 10 bytes a
// clock from memory): histograms of the first digit by slice; the weights of
// the bin that they lead to, in one list (the histograms say where a slice's
// begin); the other digits from that list, every workgroup for itself, and what
// stays of the slice behind what stays of those before it.
constexpr int kHeavyWaves = 16, kHeavyThreads = kHeavyWaves * kWave, kBins = 2048;
// Histograms of the three digits, several of each that waves share: many weights have one first digit.
constexpr int kCopies = 8;
__device__ constexpr int copy_of(int round) { return round == 0 ? 0 : 2 + 2 * round; }
__device__ constexpr int copies_of(int round) { return round == 0 ? 4 : 2; }
constexpr int kHold = 8, kSlice = kHold * kHeavyThreads;

struct Heavy {
  const float* weights;
  int64_t positions, stride;
  const int32_t* lens;
  int64_t keep;
  int sinks, recent;
  int32_t* out;  // [batch, keep], -1 behind the count
  int32_t* counts;
  float* kept;   // [batch, keep], 0 behind the count
  int slices;    // of a sequence's columns; 1: one launch
  int* hist;       // [batch, slices][kBins], first digits
  uint32_t* list;  // [batch][slices * kSlice], the weights of the chosen bin, in their positions' order
  struct FirstDigit* first;  // [batch, slices]
};

__device__ __forceinline__ uint32_t order_of(float w) {
  if (w != w) return 0xffffffffu;
  const uint32_t u = __float_as_uint(w + 0.0f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Sum over the lanes before this one, and in *total over all.
__device__ __forceinline__ int lanes_before(int v, int* total) {
  const int upto = (int)wave_scan(v);
  *total = __builtin_amdgcn_readlane(upto, kWave - 1);
  return upto - v;
}

struct HeavyLds {
  alignas(16) int hist[kCopies][kBins];
  alignas(16) int waves[2][kHeavyWaves];
  int found[2];  // digit, how many of its bin
};

// Sum of the waves' values before this wave's.
__device__ __forceinline__ int waves_before(const int (&of)[kHeavyWaves]) {
  const int wave = (int)threadIdx.x / kWave;
  int sum = 0;
#pragma unroll
  for (int v = 0; v < kHeavyWaves; v += 4) {
    const int4 n = *(const int4*)&of[v];
    sum += (v < wave ? n.x : 0) + (v + 1 < wave ? n.y : 0) + (v + 2 < wave ? n.z : 0) + (v + 3 < wave ? n.w : 0);
  }
  return sum;
}

__device__ __forceinline__ void clear_bins(HeavyLds& l) {
  for (int k = (int)threadIdx.x; k < kCopies * kBins / 4; k += kHeavyThreads) ((int4*)l.hist[0])[k] = make_int4(0, 0, 0, 0);
  __syncthreads();
}
// The bin that the need-th largest falls into, from the highest down; need becomes how many of that bin. The thread's
// two bins hold n0 (bin 2047 - 2 thread) and n1 (the one below).
__device__ __forceinline__ int pick_bin(HeavyLds& l, int n0, int n1, int& need) {
  const int tid = (int)threadIdx.x, lane = tid % kWave, wave = tid / kWave;
  int total;
  int before = lanes_before(n0 + n1, &total);
  if (lane == 0) l.waves[0][wave] = total;
  __syncthreads();
  before += waves_before(l.waves[0]);
  if (before < need && before + n0 + n1 >= need) {
    const bool upper = before + n0 >= need;
    l.found[0] = kBins - 1 - 2 * tid - (upper ? 0 : 1);
    l.found[1] = need - before - (upper ? 0 : n0);
  }
  __syncthreads();
  need = l.found[1];
  return l.found[0];
}
__device__ __forceinline__ int pick_bin(HeavyLds& l, int round, int& need) {
  __syncthreads();
  const int lo = kBins - 2 - 2 * (int)threadIdx.x;
  int n0 = 0, n1 = 0;
#pragma unroll
  for (int c = 0; c < copies_of(round); ++c) {
    const int2 n = *(const int2*)&l.hist[copy_of(round) + c][lo];
    n1 += n.x;
    n0 += n.y;
  }
  return pick_bin(l, n0, n1, need);
}
__device__ __forceinline__ void add_to_bin(HeavyLds& l, int round, uint32_t digit) {
  atomicAdd(&l.hist[copy_of(round) + (int)threadIdx.x / kWave % copies_of(round)][digit], 1);
}

// A sequence's span of weights that are compared, and how many of them stay (0: nothing to choose).
struct HeavySpan {
  int len, first, last, need;
};
__device__ __forceinline__ HeavySpan heavy_span(const Heavy& p, int64_t b) {
  HeavySpan s;
  s.len = (int)clamp64(p.lens[b], 0, p.positions);
  s.first = p.sinks, s.last = s.len - p.recent;
  s.need = s.len > p.keep ? (int)p.keep - p.sinks - p.recent : 0;
  return s;
}

// This workgroup's slice of the compared weights begins here; -1: it has none. (First tokens and columns together may pass
// 32 bits: the grid covers all columns, whatever the first tokens leave of them.)
__device__ __forceinline__ int slice_begin(const HeavySpan& s) {
  const int64_t at = s.first + (int64_t)blockIdx.x * kSlice;
  return s.need > 0 && at < s.last ? (int)at : -1;
}

// Weight i of this thread among the slice from position `from` on: a wave has 64 kHold neighbours, 64 of them at a time.
__device__ __forceinline__ int held_at(int from, int i) {
  return from + ((int)threadIdx.x / kWave * kHold + i) * kWave + (int)threadIdx.x % kWave;
}
__device__ __forceinline__ void hold(const float* w, int from, int last, float (&v)[kHold]) {
#pragma unroll
  for (int i = 0; i < kHold; ++i) v[i] = held_at(from, i) < last ? w[held_at(from, i)] : 0.0f;
}

// Everything of a sequence but the weights that are compared.
__device__ __forceinline__ void write_ends(const Heavy& p, int64_t b, const HeavySpan& s) {
  const int tid = (int)threadIdx.x;
  const float* w = p.weights + b * p.stride;
  int32_t* out = p.out + b * p.keep;
  float* kept = p.kept + b * p.keep;
  const int count = (int)(s.len < p.keep ? s.len : p.keep);
  if (tid == 0) p.counts[b] = count;
  for (int64_t k = count + tid; k < p.keep; k += kHeavyThreads) {
    out[k] = -1;
    kept[k] = 0.0f;
  }
  const int head = s.len > p.keep ? p.sinks : s.len;
  for (int k = tid; k < head; k += kHeavyThreads) {
    out[k] = k;
    kept[k] = w[k];
  }
  if (s.len <= p.keep) return;
  for (int k = tid; k < p.recent; k += kHeavyThreads) {
    out[p.keep - p.recent + k] = s.last + k;
    kept[p.keep - p.recent + k] = w[s.last + k];
  }
}

// Writes the held weights above `bound` and the first of those that equal it, `need` less the `ties` before this
// slice, from place `at` on.
__device__ __forceinline__ void write_kept(HeavyLds& l, const Heavy& p, int64_t b, const float (&v)[kHold], int from, int last,
                                           uint32_t bound, int need, int ties, int at) {
  const int lane = (int)threadIdx.x % kWave, wave = (int)threadIdx.x / kWave;
  int above = 0, same = 0;
#pragma unroll
  for (int i = 0; i < kHold; ++i) {
    const bool in = held_at(from, i) < last;
    const uint32_t u = order_of(v[i]);
    above += __popcll(__ballot(in && u > bound));
    same += __popcll(__ballot(in && u == bound));
  }
  if (lane == 0) {
    l.waves[0][wave] = above;
    l.waves[1][wave] = same;
  }
  __syncthreads();
  const int ties_before = waves_before(l.waves[1]);
  at += waves_before(l.waves[0]) + min(need, ties + ties_before) - min(need, ties);
  ties += ties_before;
  const uint64_t lower = ((uint64_t)1 << lane) - 1;
#pragma unroll
  for (int i = 0; i < kHold; ++i) {
    const int j = held_at(from, i);
    const uint32_t u = order_of(v[i]);
    const uint64_t eq = __ballot(j < last && u == bound);
    const bool stays = j < last && (u > bound || (u == bound && ties + __popcll(eq & lower) < need));
    const uint64_t all = __ballot(stays);
    if (stays) {
      const int64_t to = b * p.keep + at + __popcll(all & lower);
      p.out[to] = j;
      p.kept[to] = v[i];
    }
    at += __popcll(all);
    ties += __popcll(eq);
  }
}

__global__ __launch_bounds__(kHeavyThreads) void heaviest_kernel(const Heavy p) {
  __shared__ HeavyLds l;
  const int64_t b = blockIdx.x;
  const HeavySpan s = heavy_span(p, b);
  float v[kHold];
  if (s.need > 0) hold(p.weights + b * p.stride, s.first, s.last, v);
  if (s.need > 0) clear_bins(l);
  write_ends(p, b, s);
  if (s.need <= 0) return;
  int need = s.need;
  uint32_t bound = 0, mask = 0;
#pragma unroll
  for (int round = 0; round < 3; ++round) {
    const int shift = round == 0 ? 21 : round == 1 ? 10 : 0;
    const uint32_t digits = round == 2 ? 1023u : 2047u;
#pragma unroll
    for (int i = 0; i < kHold; ++i) {
      const uint32_t u = order_of(v[i]);
      if (held_at(s.first, i) < s.last && (u & mask) == bound) add_to_bin(l, round, u >> shift & digits);
    }
    bound |= (uint32_t)pick_bin(l, round, need) << shift;
    mask |= digits << shift;
  }
  write_kept(l, p, b, v, s.first, s.last, bound, need, 0, p.sinks);
}

// The first digits of a slice.
__global__ __launch_bounds__(kHeavyThreads) void heaviest_count_kernel(const Heavy p) {
  __shared__ HeavyLds l;
  const int64_t b = blockIdx.y;
  const HeavySpan s = heavy_span(p, b);
  const int from = slice_begin(s);
  if (blockIdx.x == 0) write_ends(p, b, s);
  if (from < 0) return;
  float v[kHold];
  hold(p.weights + b * p.stride, from, s.last, v);
  clear_bins(l);
#pragma unroll
  for (int i = 0; i < kHold; ++i)
    if (held_at(from, i) < s.last) add_to_bin(l, 0, order_of(v[i]) >> 21);
  __syncthreads();
  int* to = p.hist + (b * p.slices + blockIdx.x) * kBins;
  for (int k = (int)threadIdx.x; k < kBins; k += kHeavyThreads) {
    int n = 0;
#pragma unroll
    for (int c = 0; c < copies_of(0); ++c) n += l.hist[copy_of(0) + c][k];
    to[k] = n;
  }
}

// The bin of the first digit from all slices' histograms, and what those say of the weights in it and above it.
struct FirstDigit {
  uint32_t digit;
  int above, before, all;  // weights above the bin in the slices before this one; in the bin there, in all slices
  int need;                // of the bin's
};
__device__ __forceinline__ FirstDigit first_digit(HeavyLds& l, const Heavy& p, int64_t b, const HeavySpan& s) {
  __shared__ int sums[3];
  int need = s.need;
  const int used = (s.last - s.first + kSlice - 1) / kSlice, lo = kBins - 2 - 2 * (int)threadIdx.x;
  const int* h = p.hist + b * p.slices * kBins + lo;
  int n0 = 0, n1 = 0, m0 = 0, m1 = 0;
#pragma unroll 8
  for (int k = 0; k < used; ++k) {
    const int2 n = *(const int2*)(h + (int64_t)k * kBins);
    n1 += n.x;
    n0 += n.y;
    m1 += k < (int)blockIdx.x ? n.x : 0;
    m0 += k < (int)blockIdx.x ? n.y : 0;
  }
  if (threadIdx.x < 3) sums[threadIdx.x] = 0;
  const int digit = pick_bin(l, n0, n1, need);
  int above = (lo + 1 > digit ? m0 : 0) + (lo > digit ? m1 : 0);
  if (lo == digit || lo + 1 == digit) {
    sums[1] = lo == digit ? m1 : m0;
    sums[2] = lo == digit ? n1 : n0;
  }
#pragma unroll
  for (int o = 1; o < kWave; o <<= 1) above += __shfl_xor(above, o);
  if ((int)threadIdx.x % kWave == 0 && above) atomicAdd(&sums[0], above);
  __syncthreads();
  return FirstDigit{(uint32_t)digit, sums[0], sums[1], sums[2], need};
}

__global__ __launch_bounds__(kHeavyThreads) void heaviest_list_kernel(const Heavy p) {
  __shared__ HeavyLds l;
  const int64_t b = blockIdx.y;
  const int lane = (int)threadIdx.x % kWave, wave = (int)threadIdx.x / kWave;
  const HeavySpan s = heavy_span(p, b);
  const int from = slice_begin(s);
  if (from < 0) return;
  float v[kHold];
  hold(p.weights + b * p.stride, from, s.last, v);
  const FirstDigit f = first_digit(l, p, b, s);
  if (threadIdx.x == 0) p.first[b * p.slices + blockIdx.x] = f;
  int in_bin = 0;
#pragma unroll
  for (int i = 0; i < kHold; ++i) in_bin += __popcll(__ballot(held_at(from, i) < s.last && order_of(v[i]) >> 21 == f.digit));
  if (lane == 0) l.waves[1][wave] = in_bin;
  __syncthreads();
  int at = f.before + waves_before(l.waves[1]);
  uint32_t* to = p.list + b * p.slices * kSlice;
#pragma unroll
  for (int i = 0; i < kHold; ++i) {
    const uint32_t u = order_of(v[i]);
    const bool in = held_at(from, i) < s.last && u >> 21 == f.digit;
    const uint64_t which = __ballot(in);
    if (in) to[at + __popcll(which & (((uint64_t)1 << lane) - 1))] = u;
    at += __popcll(which);
  }
}

__global__ __launch_bounds__(kHeavyThreads) void heaviest_write_kernel(const Heavy p) {
  __shared__ HeavyLds l;
  __shared__ int sums[2];
  const int64_t b = blockIdx.y;
  const int tid = (int)threadIdx.x, lane = tid % kWave;
  const HeavySpan s = heavy_span(p, b);
  const int from = slice_begin(s);
  if (from < 0) return;
  float v[kHold];
  hold(p.weights + b * p.stride, from, s.last, v);
  const FirstDigit f = p.first[b * p.slices + blockIdx.x];
  const uint32_t* list = p.list + b * p.slices * kSlice;
  // the list's first kHold a thread stay in registers: most lists have no more
  uint32_t held[kHold];
#pragma unroll
  for (int i = 0; i < kHold; ++i) held[i] = i * kHeavyThreads + tid < f.all ? list[i * kHeavyThreads + tid] : 0;
  auto each = [&](int end, auto use) {
#pragma unroll
    for (int i = 0; i < kHold; ++i)
      if (i * kHeavyThreads + tid < end) use(held[i]);
#pragma unroll 4
    for (int i = kHold * kHeavyThreads + tid; i < end; i += kHeavyThreads) use(list[i]);
  };
  clear_bins(l);
  int need = f.need;
  uint32_t bound = f.digit << 21, mask = 2047u << 21;
#pragma unroll
  for (int round = 1; round < 3; ++round) {
    const int shift = round == 1 ? 10 : 0;
    const uint32_t digits = round == 2 ? 1023u : 2047u;
    each(f.all, [&](uint32_t u) {
      if ((u & mask) == bound) add_to_bin(l, round, u >> shift & digits);
    });
    bound |= (uint32_t)pick_bin(l, round, need) << shift;
    mask |= digits << shift;
  }
  // what stays of the slices before this one
  if (tid < 2) sums[tid] = 0;
  __syncthreads();
  int above = 0, same = 0;
  each(f.before, [&](uint32_t u) {
    above += u > bound;
    same += u == bound;
  });
#pragma unroll
  for (int o = 1; o < kWave; o <<= 1) {
    above += __shfl_xor(above, o);
    same += __shfl_xor(same, o);
  }
  if (lane == 0) {
    atomicAdd(&sums[0], above);
    atomicAdd(&sums[1], same);
  }
  __syncthreads();
  write_kept(l, p, b, v, from, s.last, bound, need, sums[1], p.sinks + f.above + sums[0] + min(need, sums[1]));
}

int heavy_slices(int64_t positions) { return (int)ceil_div(positions > 0 ? positions : 1, kSlice); }
size_t heavy_list_bytes(int64_t batch, int64_t slices) { return (size_t)batch * (size_t)slices * kSlice * 4; }
size_t heavy_first_bytes(int64_t batch, int64_t slices) { return (size_t)batch * (size_t)slices * sizeof(FirstDigit); }
size_t heavy_hist_bytes(int64_t batch, int64_t slices) { return (size_t)batch * (size_t)slices * kBins * 4; }

int check_heavy(int64_t batch, int64_t positions, int64_t stride, int64_t keep, int64_t sinks, int64_t recent) {
  if (batch < 0 || batch > 65535 || positions < 0 || positions > INT32_MAX - 4 * kSlice || stride < 0 || keep < 1 || keep > INT32_MAX - 4096 ||
      sinks < 0 || recent < 0 || sinks > keep || recent > keep - sinks)
    return fail(FCMOE_EINVAL, "heaviest_positions: bad shape (keep at least 1, and no fewer than sinks + recent)");
  return FCMOE_OK;
}

// ---- moving cached rows ---------------------------------------------------------
//
// Row positions[b, k] of sequence b becomes its row starts[b] + k, for k < counts[b].
// Bound by the rows' bytes, read once and written once.
struct Move {
  fcmoe_latent_cache c;
  const int32_t* from;
  int64_t from_width, from_stride;
  const int32_t* to;
  int64_t to_width, to_stride;
  const int32_t* positions;  // [batch, most]
  int64_t most, positions_stride;
  const int32_t* counts;
  const int32_t* starts;
  int64_t batch;
};

__device__ __forceinline__ int move_count(const Move& p, int64_t b) { return (int)clamp64(p.counts[b], 0, p.most); }
// The page and row of a position, or -1: none there.
__device__ __forceinline__ int2 cached_at(const Move& p, const int32_t* table, int64_t width, int64_t at) {
  const int64_t page = at / p.c.page_size;
  if (at < 0 || page >= width) return make_int2(-1, 0);
  const int32_t id = table[page];
  if ((uint64_t)(int64_t)id >= (uint64_t)p.c.pages) return make_int2(-1, 0);
  return make_int2(id, (int)(at - page * p.c.page_size));
}

// Rows of a workgroup, us with 16, 32, 64: 64 sequences of up to 2048 kept rows, rows from memory, 72.7, 63.0, 65.7; of 512 to
// 2048 53.9, 47.8, 50.2, of 8 bits 28.5, 36.2, 29.3; 16 of 2048 21.4, 18.1, 16.9; 8 of up to 300 4.9, 5.1, 7.5.
constexpr int kMoveRows = 32;
// To rows that no row of the call is read from: every 16 bytes on their own.
template <int R, int P, bool F8>
__global__ __launch_bounds__(256) void move_apart_kernel(const Move p) {
  constexpr int ELEM = F8 ? 1 : 2, LU = R * ELEM / 16, UNITS = LU + P * ELEM / 16, ROWS = kMoveRows;
  __shared__ int2 src[ROWS], dst[ROWS];
  const int64_t b = blockIdx.y;
  const int count = move_count(p, b), k0 = (int)blockIdx.x * ROWS, tid = (int)threadIdx.x;
  if (k0 >= count) return;
  if (tid < ROWS) {
    const int k = k0 + tid;
    int2 s = make_int2(-1, 0), d = make_int2(-1, 0);
    if (k < count) {
      s = cached_at(p, p.from + b * p.from_stride, p.from_width, p.positions[b * p.positions_stride + k]);
      d = cached_at(p, p.to + b * p.to_stride, p.to_width, (p.starts ? (int64_t)p.starts[b] : 0) + k);
    }
    if (d.x < 0) s.x = -1;
    src[tid] = s, dst[tid] = d;
    if (F8 && s.x >= 0) p.c.scale[d.x * p.c.scale_page_stride + d.y] = p.c.scale[s.x * p.c.scale_page_stride + s.y];
  }
  __syncthreads();
  constexpr int EACH = (ROWS * UNITS + 255) / 256;
  v4i v[EACH];
  auto place = [&](int2 at, int unit) {
    return unit < LU ? (char*)p.c.latent + (at.x * p.c.latent_page_stride + at.y * p.c.latent_row_stride) * ELEM + unit * 16
                     : (char*)p.c.rope + (at.x * p.c.rope_page_stride + at.y * p.c.rope_row_stride) * ELEM + (unit - LU) * 16;
  };
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const int at = i * 256 + tid, row = at / UNITS;
    if (row < ROWS && src[row].x >= 0) v[i] = *(const v4i*)place(src[row], at % UNITS);
  }
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const int at = i * 256 + tid, row = at / UNITS;
    if (row < ROWS && src[row].x >= 0) *(v4i*)place(dst[row], at % UNITS) = v[i];
  }
}

// Within a sequence: positions ascend and none lies before its new place, so a
// row's place is only ever read for an earlier one (or itself). A workgroup takes
// 128 bytes of every row of a sequence (the last one the key part and the
// scales), 1024 rows at a time in order: they are all read before any is written.
// That is 9 workgroups a sequence (5 of 8-bit rows), each with one chunk's latency
// behind the other: 1 sequence of 4096 kept rows 48 us (62 of 8 bits), 8 of them 72,
// 64 of 512 to 2048 99 (68), where the bytes take 2, 16 and 38 (20); up to 5
// accepted drafts of 32 sequences 4.2.
template <int R, int P, bool F8>
__global__ __launch_bounds__(1024) void move_within_kernel(const Move p) {
  constexpr int ELEM = F8 ? 1 : 2, PIECES = R * ELEM / 128, RU = P * ELEM / 16, HOLD = 8;
  const int64_t b = blockIdx.y;
  const int count = move_count(p, b), piece = (int)blockIdx.x, unit = (int)threadIdx.x % 8;
  const int64_t first = p.starts ? p.starts[b] : 0;
  const bool latent = piece < PIECES, rope = !latent && unit < RU, scale = F8 && !latent && unit == 7;
  for (int k0 = 0; k0 < count; k0 += 128 * HOLD) {
    v4i v[HOLD];
    int2 to[HOLD];
#pragma unroll
    for (int i = 0; i < HOLD; ++i) {
      const int k = k0 + i * 128 + (int)threadIdx.x / 8;
      to[i] = make_int2(-1, 0);
      if (k >= count) continue;
      const int64_t at = p.positions[b * p.positions_stride + k];
      if (at == first + k) continue;
      const int2 s = cached_at(p, p.from + b * p.from_stride, p.from_width, at);
      if (s.x >= 0) to[i] = cached_at(p, p.from + b * p.from_stride, p.from_width, first + k);
      if (to[i].x < 0) continue;
      if (latent)
        v[i] = *(const v4i*)((const char*)p.c.latent + (s.x * p.c.latent_page_stride + s.y * p.c.latent_row_stride) * ELEM + piece * 128 + unit * 16);
      else if (rope)
        v[i] = *(const v4i*)((const char*)p.c.rope + (s.x * p.c.rope_page_stride + s.y * p.c.rope_row_stride) * ELEM + unit * 16);
      else if (scale)
        v[i][0] = __float_as_int(p.c.scale[s.x * p.c.scale_page_stride + s.y]);
    }
    loads_barrier();  // all of them are here before the first is overwritten
#pragma unroll
    for (int i = 0; i < HOLD; ++i) {
      if (to[i].x < 0) continue;
      if (latent)
        *(v4i*)((char*)p.c.latent + (to[i].x * p.c.latent_page_stride + to[i].y * p.c.latent_row_stride) * ELEM + piece * 128 + unit * 16) = v[i];
      else if (rope)
        *(v4i*)((char*)p.c.rope + (to[i].x * p.c.rope_page_stride + to[i].y * p.c.rope_row_stride) * ELEM + unit * 16) = v[i];
      else if (scale)
        p.c.scale[to[i].x * p.c.scale_page_stride + to[i].y] = __int_as_float(v[i][0]);
    }
  }
}

template <int R, int P, bool F8>
void move_launch(const Move& p, hipStream_t stream) {
  if (p.to)
    hipLaunchKernelGGL((move_apart_kernel<R, P, F8>), dim3((unsigned)ceil_div(p.most, kMoveRows), (unsigned)p.batch), dim3(256), 0, stream, p);
  else
    hipLaunchKernelGGL((move_within_kernel<R, P, F8>), dim3((unsigned)(R * (F8 ? 1 : 2) / 128 + (P || F8 ? 1 : 0)), (unsigned)p.batch),
                       dim3(1024), 0, stream, p);
}

}  // namespace

}  // namespace fcmoe

using namespace fcmoe;

extern "C" int fcmoe_draft_tree(const int32_t* parents, int64_t tokens, const int32_t* query_starts, int64_t batch,
                                int64_t mask_words, uint64_t* masks, int32_t* depths, hipStream_t stream) {
  if (tokens < 0 || tokens > INT32_MAX || batch <= 0 || batch > (1 << 20) || mask_words < 1 || mask_words > kTreeNodes / 64)
    return fail(FCMOE_EINVAL, "draft_tree: bad shape (1 to 16 mask words)");
  if (tokens == 0) return FCMOE_OK;
  if (!parents || !query_starts || !masks || !depths) return fail(FCMOE_EINVAL, "draft_tree: NULL pointer");
  Tree p{parents, query_starts, tokens, (int)batch, (int)mask_words, masks, depths};
  hipLaunchKernelGGL(draft_tree_kernel, dim3((unsigned)batch), dim3(kTreeThreads), 0, stream, p);
  return check_launch("draft_tree");
}

extern "C" size_t fcmoe_heaviest_positions_workspace_bytes(int64_t batch, int64_t positions, int64_t keep, int64_t sinks, int64_t recent) {
  if (check_heavy(batch, positions, 0, keep, sinks, recent) != FCMOE_OK || batch == 0) return 0;
  const int64_t slices = heavy_slices(positions);
  return slices == 1 ? 0 : heavy_list_bytes(batch, slices) + heavy_hist_bytes(batch, slices) + heavy_first_bytes(batch, slices);
}

extern "C" int fcmoe_heaviest_positions(const float* weights, int64_t batch, int64_t positions, int64_t stride,
                                        const int32_t* kv_lens, int64_t keep, int64_t sinks, int64_t recent,
                                        int32_t* out_positions, int32_t* counts, float* kept, void* workspace,
                                        size_t workspace_bytes, hipStream_t stream) {
  if (const int rc = check_heavy(batch, positions, stride, keep, sinks, recent)) return rc;
  if (batch == 0) return FCMOE_OK;
  if ((positions > 0 && !weights) || !kv_lens || !out_positions || !counts || !kept)
    return fail(FCMOE_EINVAL, "heaviest_positions: NULL pointer");
  Heavy p{};
  p.weights = weights, p.positions = positions, p.stride = stride, p.lens = kv_lens, p.keep = keep;
  p.sinks = (int)sinks, p.recent = (int)recent, p.out = out_positions, p.counts = counts, p.kept = kept;
  p.slices = heavy_slices(positions);
  if (p.slices == 1) {
    hipLaunchKernelGGL(heaviest_kernel, dim3((unsigned)batch), dim3(kHeavyThreads), 0, stream, p);
    return check_launch("heaviest_positions");
  }
  if (!workspace || workspace_bytes < fcmoe_heaviest_positions_workspace_bytes(batch, positions, keep, sinks, recent))
    return fail(FCMOE_ESPACE, "heaviest_positions: workspace too small");
  if ((uintptr_t)workspace % 16) return fail(FCMOE_EINVAL, "heaviest_positions: unaligned workspace");
  p.list = (uint32_t*)workspace;
  p.hist = (int*)((char*)workspace + heavy_list_bytes(batch, p.slices));
  p.first = (FirstDigit*)((char*)p.hist + heavy_hist_bytes(batch, p.slices));
  const dim3 g((unsigned)p.slices, (unsigned)batch), t(kHeavyThreads);
  hipLaunchKernelGGL(heaviest_count_kernel, g, t, 0, stream, p);
  hipLaunchKernelGGL(heaviest_list_kernel, g, t, 0, stream, p);
  hipLaunchKernelGGL(heaviest_write_kernel, g, t, 0, stream, p);
  return check_launch("heaviest_positions");
}

extern "C" int fcmoe_latent_cache_move(const fcmoe_latent_move_args* a, hipStream_t stream) {
  if (!a) return fail(FCMOE_EINVAL, "latent_cache_move: NULL args");
  if (const int rc = check_latent_cache(a->cache, "latent_cache_move")) return rc;
  if (a->batch < 0 || a->batch > 65535 || a->most < 0 || a->most > INT32_MAX - 4096 || a->positions_stride < 0 || a->table_width < 0 ||
      a->table_width > INT32_MAX || a->page_table_stride < 0 || a->to_width < 0 || a->to_width > INT32_MAX || a->to_stride < 0)
    return fail(FCMOE_EINVAL, "latent_cache_move: bad shape");
  if (a->batch == 0 || a->most == 0 || a->cache.pages == 0 || a->table_width == 0) return FCMOE_OK;
  if (!a->page_table || !a->positions || !a->counts) return fail(FCMOE_EINVAL, "latent_cache_move: NULL pointer");
  Move p{};
  p.c = a->cache;
  p.from = a->page_table, p.from_width = a->table_width, p.from_stride = a->page_table_stride;
  p.to = a->to_table, p.to_width = a->to_width, p.to_stride = a->to_stride;
  p.positions = a->positions, p.most = a->most, p.positions_stride = a->positions_stride;
  p.counts = a->counts, p.starts = a->starts, p.batch = a->batch;
  const bool f8 = a->cache.e4m3 != 0;
  if (a->cache.latent_dim == 512) {
    if (a->cache.rope_dim == 64)
      f8 ? move_launch<512, 64, true>(p, stream) : move_launch<512, 64, false>(p, stream);
    else
      f8 ? move_launch<512, 0, true>(p, stream) : move_launch<512, 0, false>(p, stream);
  } else {
    if (a->cache.rope_dim == 64)
      f8 ? move_launch<256, 64, true>(p, stream) : move_launch<256, 64, false>(p, stream);
    else
      f8 ? move_launch<256, 0, true>(p, stream) : move_launch<256, 0, false>(p, stream);
  }
  return check_launch("latent_cache_move");
}
