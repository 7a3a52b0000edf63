// Scores of given tokens and distillation from a teacher's top alternatives on
// rows of logits in device memory, and their gradients.
//
// With z a row of V logits, T the temperature, m = max z, c = log2(e) / T:
//   t_j = (z_j - m) c,  e_j = 2^t_j,  r = sum of e over all but one maximum,
//   L = log(1 + r),     log p_j = (z_j - m) / T - L.
// Keeping the maximum out of r lets the log probability of a token that is
// nearly certain keep its digits (log(1 + 1e-9) is not formed from 1 + 1e-9).
//
// Nothing here feeds the codec, whose integer CDFs repeat the reference's
// arithmetic operation by operation (../csrc); these kernels have none to
// repeat and use fused multiply-adds and the hardware's 2^x (1 ulp), with 32-bit
// sums inside a segment and 64-bit ones across segments.
#include "dtl_scores.h"

#include "dtl_rows.h"

namespace dtl {
namespace {

constexpr int kJoinThreads = 512;
constexpr int kPartThreads = 256;
constexpr int kPer = kScoreSeg / 64;  // logits a lane holds of a segment
constexpr int kMostWaves = 16;        // of a row's workgroup
constexpr double kLog2E = 1.4426950408889634074;
constexpr double kLn2 = 0.6931471805599453094;

// ---- a segment in registers ------------------------------------------------

template <int DT>
struct Seg {  // a lane's logits of a segment: packets of 16 bytes, 64 lanes apart
  static constexpr int kPackets = kPer / Type<DT>::kInPacket;
  packet w[kPackets];
};
using dtl::value;  // of a packet
template <int DT>
__device__ __forceinline__ float value(const Seg<DT>& s, int i) {
  return value<DT>(s.w[i / Type<DT>::kInPacket], i % Type<DT>::kInPacket);
}

// ONCE: past the caches' usual policy, for logits that do not fit the 256 MB
// memory-side cache anyway (see read_past).
template <int DT, bool ONCE>
__device__ __forceinline__ void load_seg(Seg<DT>& s, const char* row, int seg, int lane, int V) {
  constexpr int n = Type<DT>::kInPacket;
  const int at = seg * kScoreSeg + lane * n;
  if (seg * kScoreSeg + kScoreSeg <= V) {
#pragma unroll
    for (int q = 0; q < Seg<DT>::kPackets; q++) {
      const auto* p = reinterpret_cast<const typename Type<DT>::mem*>(row + (size_t)(at + q * 64 * n) * Type<DT>::kBytes);
      s.w[q] = ONCE ? __builtin_nontemporal_load(p) : *p;
    }
  } else {
#pragma unroll
    for (int q = 0; q < Seg<DT>::kPackets; q++) s.w[q] = load_packet<DT>(row, at + q * 64 * n, V);
  }
}

// Masks the lane's logits whose bit is set.
template <int DT>
__device__ __forceinline__ void mask_seg(Seg<DT>& s, uint32_t bits) {
#pragma unroll
  for (int q = 0; q < Seg<DT>::kPackets; q++)
#pragma unroll
    for (int d = 0; d < 4; d++) {
      uint32_t m;
      if constexpr (DT == DTL_F32) {
        m = bits >> (q * 4 + d) & 1 ? ~0u : 0u;
      } else {
        const uint32_t b = bits >> (q * 8 + 2 * d);
        m = (b & 1 ? 0xffffu : 0u) | (b & 2 ? 0xffff0000u : 0u);
      }
      s.w[q][d] = (s.w[q][d] & ~m) | (Type<DT>::kMasked & m);
    }
}

// ---- a segment -----------------------------------------------------------------

struct Part {  // of a segment: the maximum, sum of e, sum of e t, both relative to it
  float m, s, u;
};

// e t needs t kept off -inf (0 times that is no number); 2^-200 is 0 anyway.
// e itself is formed from t, so that a logit that is no number makes s none.
constexpr float kLowest = -200.0f;

template <int DT>
__device__ __forceinline__ float lane_max(const Seg<DT>& z) {
  float m = value<DT>(z, 0);
#pragma unroll
  for (int i = 1; i < kPer; i++) m = fmaxf(m, value<DT>(z, i));
  return m;
}

// The sums of a segment.  NEAR: t from one fused z c - mc, mc the rounded m c
// (the sums are then relative to mc and are brought back to m c at the end by
// 2^-d, d = m c - mc of up to half an ulp of mc); otherwise from z - m.
template <int DT, bool ENT, bool NEAR>
__device__ __forceinline__ void seg_sums(const Seg<DT>& z, float m, float c, float& sum, float& weighted) {
  float s[4] = {}, u[4] = {};
  const float mc = m * c;
#pragma unroll
  for (int i = 0; i < kPer; i++) {
    const float v = value<DT>(z, i), t = NEAR ? __builtin_fmaf(v, c, -mc) : (v - m) * c;
    const float e = __builtin_amdgcn_exp2f(t);
    s[i & 3] += e;
    if (ENT) u[i & 3] = __builtin_fmaf(e, fmaxf(t, kLowest), u[i & 3]);
  }
  sum = wave_sum((s[0] + s[1]) + (s[2] + s[3]));
  weighted = ENT ? wave_sum((u[0] + u[1]) + (u[2] + u[3])) : 0.0f;
  if (NEAR) {
    const float d = __builtin_fmaf(m, c, -mc), f = __builtin_amdgcn_exp2f(-d);
    weighted = (weighted - d * sum) * f;
    sum *= f;
  }
}

template <int DT, bool ENT>
__device__ __forceinline__ Part seg_part(const Seg<DT>& z, float most, float c) {
  Part p{wave_max(most), 0.0f, 0.0f};
  const float m = p.m == -__builtin_inff() ? 0.0f : p.m;
  // |d| <= 2^-5 there, so that taking it through the sums costs less than a
  // rounding.  From |m c| = 2^32 on it can pass 128, where 2^d overflows.
  if (__builtin_fabsf(m * c) < 0x1p20f)
    seg_sums<DT, ENT, true>(z, m, c, p.s, p.u);
  else
    seg_sums<DT, ENT, false>(z, m, c, p.s, p.u);
  return p;
}

// ---- a row, its segments' parts in LDS -------------------------------------------

struct RowStats {
  float m;      // the largest logit; -inf: every logit is masked
  double r, u;  // over the row, relative to m
  bool bad;     // a logit is NaN or +inf
};

// A row's maximum and the first segment that holds it, by a whole wave.
struct RowMax {
  float m;
  int first;
  bool none;  // nothing to sum: a NaN or +inf (bad), or every logit masked
  bool bad;
};
__device__ __forceinline__ RowMax find_max(const Part* parts, int nseg, int lane) {
  const float no = -__builtin_inff();
  const Part a = lane < nseg ? parts[lane] : Part{no, 0.0f, 0.0f};
  const Part b = lane + 64 < nseg ? parts[lane + 64] : Part{no, 0.0f, 0.0f};
  RowMax x;
  x.m = wave_max(fmaxf(a.m, b.m));
  x.bad = __ballot(!(a.s == a.s) || !(b.s == b.s)) != 0 || x.m == __builtin_inff();
  x.none = x.bad || x.m == no;
  const uint64_t in_a = __ballot(a.m == x.m), in_b = __ballot(b.m == x.m);
  x.first = x.none ? 0 : in_a ? __builtin_ctzll(in_a) : 64 + __builtin_ctzll(in_b);
  return x;
}

// A lane's sums of e and of e t over the segment that holds the maximum m, one
// such logit left out.
template <int DT, bool ENT>
__device__ __forceinline__ void sums_without_max(const Seg<DT>& z, float m, float c, int lane, float& s, float& w) {
  const uint64_t have = __ballot(lane_max<DT>(z) == m);
  bool out = lane == __builtin_ctzll(have);  // this lane's first maximum stays out
  s = w = 0.0f;
#pragma unroll
  for (int i = 0; i < kPer; i++) {
    const float v = value<DT>(z, i), t = (v - m) * c;
    const bool skip = out && v == m;
    out = out && !skip;
    const float e = skip ? 0.0f : __builtin_amdgcn_exp2f(t);
    s += e;
    if (ENT) w = __builtin_fmaf(e, fmaxf(t, kLowest), w);
  }
}

// The row's sums from its parts, with those of the maximum's segment as above.
template <bool ENT>
__device__ __forceinline__ RowStats join_parts(const RowMax& x, const Part* parts, int nseg, float s, float w, float c,
                                               int lane) {
  RowStats st{x.m, 0.0, 0.0, x.bad};
  if (x.none) return st;
  double r = s, u = w;
#pragma unroll
  for (int i = 0; i < 2; i++) {
    const int seg = lane + 64 * i;
    if (seg >= nseg || seg == x.first || parts[seg].m == -__builtin_inff()) continue;
    const Part p = parts[seg];
    const float d = fmaxf((p.m - x.m) * c, -1000.0f);
    const double f = __builtin_amdgcn_exp2f(d);
    r += f * p.s;
    if (ENT) u += f * ((double)p.u + (double)d * p.s);
  }
  st.r = wave_sum(r);
  if (ENT) st.u = wave_sum(u);
  return st;
}

// Both by one wave, the maximum's segment read again.  `mask` (may be null): per
// segment and lane the logits that the parts left out.
template <int DT, bool ENT>
__device__ __forceinline__ RowStats join_row(const char* row, int V, int nseg, const Part* parts, const uint32_t* mask, float c, int lane) {
  const RowMax x = find_max(parts, nseg, lane);
  float s = 0.0f, w = 0.0f;
  if (!x.none) {
    Seg<DT> z;
    load_seg<DT, false>(z, row, x.first, lane, V);
    if (mask) mask_seg<DT>(z, mask[x.first * 64 + lane]);
    sums_without_max<DT, ENT>(z, x.m, c, lane, s, w);
  }
  return join_parts<ENT>(x, parts, nseg, s, w, c, lane);
}

// ---- the largest logits of a row ---------------------------------------------------

// Logits in their order as unsigned numbers; masked ones are 0, -0 equals 0.
__device__ __forceinline__ uint32_t order_of(float v) {
  const uint32_t b = __builtin_bit_cast(uint32_t, v + 0.0f);
  if (v == -__builtin_inff() || !(v == v)) return 0;
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float of_order(uint32_t k) {
  return __builtin_bit_cast(float, k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

struct alignas(16) TopLds {
  uint32_t bins[4][256];
  uint32_t low[kMostWaves], high[kMostWaves];
  uint32_t counts[2][kMostWaves];
  uint32_t buckets, candidates, chosen;
  uint16_t ties[kScoreMaxSegs];
  uint16_t bucket[kScoreMaxTop + 64];
  uint64_t best[kScoreMaxTop];
};
// Candidates: every logit of K + 64 buckets at most.
constexpr size_t candidate_bytes(size_t top) { return (top + 64) * kPer * sizeof(uint64_t); }

// Places for each lane's n entries at the end of a list, by a whole wave.
__device__ __forceinline__ uint32_t append(uint32_t* length, uint32_t n, int lane) {
  const uint32_t sum = wave_scan(n), all = __builtin_amdgcn_readlane((int)sum, 63);
  uint32_t base = 0;
  if (all != 0) {
    if (lane == 0) base = atomicAdd(length, all);
    base = __builtin_amdgcn_readfirstlane((int)base);
  }
  return base + sum - n;
}

// How many of the workgroup's flags are set, for step `step` of a loop: the two
// sets of counts let one barrier a step do.
template <int WAVES>
__device__ __forceinline__ int group_count(TopLds& t, int step, int in_wave, int wave, int lane) {
  if (lane == 0) t.counts[step & 1][wave] = in_wave;
  __syncthreads();
  int n = 0;
#pragma unroll
  for (int w = 0; w < WAVES; w++) n += t.counts[step & 1][w];
  return n;
}

// A thread's keys: those of its lane in segments wave, wave + WAVES, ...
template <int WAVES>
struct Keys {
  uint32_t k[kScoreMaxSegs / WAVES];
};
// Before the barrier that precedes select_top: the keys into registers from
// keys[nseg * 64], the order of the largest logit of each bucket (a lane's share
// of a segment), and what the workgroup's threads say of them.
template <int WAVES>
__device__ __forceinline__ void take_keys(Keys<WAVES>& key, const uint32_t* keys, int nseg, TopLds& t) {
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  uint32_t most = 0;
#pragma unroll
  for (int i = 0; i < kScoreMaxSegs / WAVES; i++) {
    key.k[i] = i * WAVES + wave < nseg ? keys[i * (WAVES * 64) + tid] : 0;
    most = max(most, key.k[i]);
  }
  const uint32_t low = ~wave_max(~most), high = wave_max(most);
  if ((tid & 63) == 0) {
    t.low[wave] = low;
    t.high[wave] = high;
  }
  for (int i = tid; i < 4 * 256; i += WAVES * 64) (&t.bins[0][0])[i] = 0;
  if (tid == 0) t.buckets = t.candidates = t.chosen = 0;
}

// The `top` largest logits of a row in order (value, then the lower index), by
// the whole workgroup.  Put the buckets in the order of their largest logits: the
// row's `top` largest lie in the first `top` buckets, since each of those holds
// one that is as large.  So:
//   1. tau, such that at least `top` buckets reach it and few more, by counting
//      keys in 256 equal steps of an interval, then of the step that holds key
//      `top`, four times at most, mostly once.  It starts at a key that a whole
//      wave's threads reach (each by the largest of its keys): 64 keys are no less;
//   2. the buckets from tau on.  If many equal tau, those only up to the segment
//      where there are enough: the lowest indices among equals lie no further;
//   3. their logits from tau on, read again (32 a bucket);
//   4. these ranked by counting, each against each.
// All but 3 is in LDS and registers, whatever the logits hold: rows of equal
// logits take the same steps.  `memory` holds the candidates; it may be the keys'.
// `aside` is the first wave's, which takes no part in 3; its results are there
// when `emit` is called.
template <int DT, int WAVES, typename Aside, typename Emit>
__device__ __forceinline__ void select_top(const char* row, int V, int nseg, int top, const Keys<WAVES>& keys,
                                           uint64_t* memory, TopLds& t, Aside&& aside, Emit&& emit) {
  constexpr int threads = WAVES * 64, per_thread = kScoreMaxSegs / WAVES;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const auto& key = keys.k;

  uint32_t lo = 0, second = 0, hi = 0;
#pragma unroll
  for (int w = 0; w < WAVES; w++) {
    const uint32_t x = t.low[w];
    second = max(second, min(lo, x));
    lo = max(lo, x);
    hi = max(hi, t.high[w]);
  }
  lo = top == 1 ? hi : top > 64 ? second : lo;
  lo = max(lo, 1u);  // 0 is masked
  static_assert(kScoreMaxTop <= 128, "two waves' keys");
  int above = 0, equal = 0;  // keys past the interval, and in the last one
  uint32_t tau = lo;
  for (int step = 0; step < 4 && lo <= hi; step++) {
    const int bits = 32 - __builtin_clz((hi - lo) | 1u), shift = bits > 8 ? bits - 8 : 0;
#pragma unroll
    for (int i = 0; i < per_thread; i++)
      if (key[i] >= lo && key[i] <= hi) atomicAdd(&t.bins[step][(key[i] - lo) >> shift], 1u);
    __syncthreads();
    // lane 0 has the four highest bins
    const uint4 b = *reinterpret_cast<const uint4*>(&t.bins[step][252 - 4 * lane]);
    const uint32_t sum = wave_scan(b.x + b.y + b.z + b.w);
    const uint64_t reach = __ballot((int)sum >= top - above);
    if (reach == 0) {  // fewer than `top` buckets hold anything unmasked
      equal = __builtin_amdgcn_readlane((int)sum, 63);
      tau = lo;
      break;
    }
    uint32_t over = sum - (b.x + b.y + b.z + b.w), bin = 252 - 4 * lane + 3, in = b.w;
    const uint32_t c[3] = {b.z, b.y, b.x};
#pragma unroll
    for (int i = 0; i < 3; i++)
      if ((int)(over + in) < top - above) {
        over += in;
        in = c[i];
        bin--;
      }
    const int at = __builtin_ctzll(reach);
    above += __builtin_amdgcn_readlane((int)over, at);
    equal = __builtin_amdgcn_readlane((int)in, at);
    lo += (uint32_t)__builtin_amdgcn_readlane((int)bin, at) << shift;
    hi = lo + min(hi - lo, (1u << shift) - 1u);
    tau = lo;
    if (shift == 0 || above + equal <= top + top / 4 + 8) break;
  }

  int last = nseg;  // the segment up to which keys equal to tau count
  if (above + equal > top + 64) {  // then the interval is one key wide
#pragma unroll
    for (int i = 0; i < per_thread; i++)
      if (i * WAVES + wave < nseg) {
        const int same = __popcll(__ballot(key[i] == tau));
        if (lane == 0) t.ties[i * WAVES + wave] = same;
      }
    __syncthreads();
    last = 0;
    for (int have = above; last < nseg; last++) {
      have += t.ties[last];
      if (have >= top) break;
    }
  }
  uint32_t mine = 0;
#pragma unroll
  for (int i = 0; i < per_thread; i++)
    if (key[i] > tau || (key[i] == tau && i * WAVES + wave <= last)) mine |= 1u << i;
  uint32_t at = append(&t.buckets, __popc(mine), lane);
  for (uint32_t m = mine; m; m &= m - 1)
    t.bucket[at++] = (uint16_t)((__builtin_ctz(m) * WAVES + wave) * 64 + lane);
  __syncthreads();
  if (wave == 0) aside();

  constexpr int np = Seg<DT>::kPackets, in = Type<DT>::kInPacket;
  const int work = (int)t.buckets * np;
  for (int first = wave == 0 ? work : 0; first < work; first += threads - 64) {
    const int w = first + tid - 64;
    int j = 0;
    uint32_t k[in], have = 0;
    if (w < work) {
      const int b = t.bucket[w / np];
      j = (b >> 6) * kScoreSeg + (w % np) * (64 * in) + (b & 63) * in;
      const packet p = load_packet<DT>(row, j, V);
#pragma unroll
      for (int i = 0; i < in; i++) {
        k[i] = order_of(value<DT>(p, i));
        have += k[i] >= tau;
      }
    }
    uint32_t to = append(&t.candidates, have, lane);
    if (have)
#pragma unroll
      for (int i = 0; i < in; i++)
        if (k[i] >= tau) memory[to++] = (uint64_t)k[i] << 18 | (uint32_t)(kScoreMaxVocab - 1 - (j + i));
  }
  __syncthreads();

  const uint64_t* list = memory;
  int n = t.candidates;
  if (n > 512) {  // many equal or neighbouring ones: the `top` best by their 50 bits first
    uint64_t floor = 0;
    for (int bit = 49; bit >= 0; bit--) {
      const uint64_t trial = floor | (uint64_t)1 << bit;
      int in_wave = 0;
      for (int i = tid - lane; i < n; i += threads) in_wave += __popcll(__ballot(i + lane < n && memory[i + lane] >= trial));
      const int got = group_count<WAVES>(t, bit, in_wave, wave, lane);
      if (got >= top) floor = trial;
      if (got == top) break;
    }
    for (int i = tid; i < n; i += threads)
      if (memory[i] >= floor) t.best[atomicAdd(&t.chosen, 1u)] = memory[i];
    __syncthreads();
    list = t.best;
    n = top;
  }
  // eight threads count for one candidate
  for (int first = 0; first < n; first += threads / 8) {
    const int i = first + tid / 8;
    const uint64_t one = list[min(i, n - 1)];
    int rank = 0;
    for (int j = tid & 7; j < n; j += 8) rank += list[j] > one;
    rank += __shfl_xor(rank, 1);
    rank += __shfl_xor(rank, 2);
    rank += __shfl_xor(rank, 4);
    if (i < n && rank < top && (tid & 7) == 0)
      emit(rank, kScoreMaxVocab - 1 - (int)(one & (kScoreMaxVocab - 1)), of_order((uint32_t)(one >> 18)));
  }
  if (tid < top && tid >= n) emit(tid, -1, -__builtin_inff());
}

// ---- reading a row ------------------------------------------------------------------

// Segments seg0 + wave, seg0 + wave + waves, ... below seg1: their parts, and
// with KEYS their buckets' largest logits.  The next segment's loads are in
// flight while one is reduced.
template <int DT, bool ENT, bool KEYS, bool ONCE>
__device__ __forceinline__ void read_segs_as(const char* row, int V, int seg0, int seg1, int wave, int waves, int lane,
                                             float c, Part* parts, uint32_t* keys, const uint32_t* mask) {
  int seg = seg0 + wave;
  if (seg >= seg1) return;
  Seg<DT> z, next;
  load_seg<DT, ONCE>(z, row, seg, lane, V);
  for (; seg < seg1; seg += waves) {
    if (seg + waves < seg1) load_seg<DT, ONCE>(next, row, seg + waves, lane, V);
    if (mask) {
      const uint32_t bits = mask[seg * 64 + lane];
      if (__ballot(bits != 0)) mask_seg<DT>(z, bits);
    }
    const float most = lane_max<DT>(z);
    if (KEYS) keys[seg * 64 + lane] = order_of(most);
    const Part p = seg_part<DT, ENT>(z, most, c);
    if (lane == 0) parts[seg] = p;
    z = next;
  }
}
template <int DT, bool ENT, bool KEYS>
__device__ __forceinline__ void read_segs(const char* row, int V, int seg0, int seg1, int wave, int waves, int lane,
                                          float c, bool once, Part* parts, uint32_t* keys, const uint32_t* mask) {
  if (once)
    read_segs_as<DT, ENT, KEYS, true>(row, V, seg0, seg1, wave, waves, lane, c, parts, keys, mask);
  else
    read_segs_as<DT, ENT, KEYS, false>(row, V, seg0, seg1, wave, waves, lane, c, parts, keys, mask);
}

// Whole rows by one workgroup each, or for few rows one part of a row each
// (PARTS) and a second launch that joins them (JOIN).
enum Phase { WHOLE, PARTS, JOIN };

// ---- scores ---------------------------------------------------------------------------

struct ScoreK {
  const char* z;
  size_t row_bytes, row0;  // the launch's first row
  bool once;               // read past the caches
  int V, nseg, groups;
  const void* tokens;
  int wide, top;
  float c;
  double inv_t;
  float *log_probs, *entropy, *stats;
  int32_t* top_ids;
  float* top_log_probs;
  Part* parts;     // [rows][nseg], PARTS and JOIN
  uint32_t* keys;  // [rows][nseg * 64]
};

template <int DT, bool TOP, int PHASE, int THREADS>
__global__ __launch_bounds__(THREADS) void k_scores(ScoreK a) {
  extern __shared__ uint64_t memory[];
  __shared__ Part lds_parts[PHASE == PARTS ? 1 : kScoreMaxSegs];
  __shared__ TopLds tl;
  __shared__ float row_m;
  __shared__ double row_log;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  constexpr int waves = THREADS / 64;
  const float no = -__builtin_inff();

  if constexpr (PHASE == PARTS) {
    const size_t row = blockIdx.x / a.groups;
    const int g = (int)(blockIdx.x % a.groups), per = (a.nseg + a.groups - 1) / a.groups;
    read_segs<DT, true, TOP>(a.z + row * a.row_bytes, a.V, g * per, min(a.nseg, (g + 1) * per), wave, waves, lane, a.c,
                             false, a.parts + row * a.nseg, TOP ? a.keys + row * a.nseg * 64 : nullptr, nullptr);
    return;
  }

  const size_t row = a.row0 + blockIdx.x;
  const char* z = a.z + row * a.row_bytes;
  long y = -1;
  float zy = 0.0f;
  if (wave == 0 && a.tokens) {
    y = load_index(a.tokens, a.wide, row);
    if (y >= 0 && y < a.V) zy = load_one<DT>(z, (int)y);
  }
  Keys<TOP ? waves : kScoreMaxSegs> key;
  if constexpr (PHASE == WHOLE) {
    uint32_t* keys = reinterpret_cast<uint32_t*>(memory);
    read_segs<DT, true, TOP>(z, a.V, 0, a.nseg, wave, waves, lane, a.c, a.once, lds_parts, keys, nullptr);
    if constexpr (TOP) take_keys(key, keys, a.nseg, tl);  // each thread its own
  } else {
    for (int i = threadIdx.x; i < a.nseg; i += THREADS) lds_parts[i] = a.parts[row * a.nseg + i];
    if constexpr (TOP) take_keys(key, a.keys + row * a.nseg * 64, a.nseg, tl);
  }
  __syncthreads();
  auto join = [&]() __attribute__((always_inline)) {
    const RowStats st = join_row<DT, true>(z, a.V, a.nseg, lds_parts, nullptr, a.c, lane);
    const double l = st.bad ? (double)__builtin_nanf("") : log1p(st.r);
    const float m = st.bad ? __builtin_nanf("") : st.m;
    if (lane != 0) return;
    row_m = m;
    row_log = l;
    if (a.stats) {
      a.stats[2 * row] = m;
      a.stats[2 * row + 1] = st.bad ? m : (float)st.r;
    }
    if (a.entropy) a.entropy[row] = st.m == no && !st.bad ? 0.0f : (float)(l - kLn2 * st.u / (1.0 + st.r));
    if (a.log_probs) {
      float lp = 0.0f;
      if (y >= a.V)
        lp = __builtin_nanf("");
      else if (y >= 0)
        lp = m == no ? no : (float)(((double)zy - m) * a.inv_t - l);
      a.log_probs[row] = lp;
    }
  };
  if constexpr (!TOP) {
    if (wave == 0) join();
  } else {
    int32_t* ids = a.top_ids + row * a.top;
    float* lps = a.top_log_probs + row * a.top;
    select_top<DT>(z, a.V, a.nseg, a.top, key, memory, tl, join, [&](int at, int id, float v) __attribute__((always_inline)) {
      const float m = row_m;
      const bool bad = !(m == m);
      ids[at] = bad ? -1 : id;
      lps[at] = bad ? m : id < 0 ? no : (float)(((double)v - m) * a.inv_t - row_log);
    });
  }
}

// dz = ( g (delta_y - p) - h p (log p + H) ) / T for the gradients g of the
// token's log probability and h of the entropy.  With p = e / (1 + r) that is
// e (A + B t) per logit, and at the token 1 - p = -expm1(log p).
struct ScoreGradK {
  const char* z;
  char* grad;
  size_t row_bytes, grad_bytes, row0;
  int V, nseg, chunks;
  bool past;  // write past the caches
  const void* tokens;
  int wide;
  float c;
  double inv_t;
  const float *stats, *entropy, *g, *h;
};

// Waves of a gradient's workgroup, each with one segment: us of 4096 rows of 151936
// bf16 with one / two / four segments a wave 450 / 471 / 478.
constexpr int kGradWaves = 4;

// PAST: past the caches' usual policy, see write_past.
template <int DT, bool PAST, typename F>
__device__ __forceinline__ void write_seg_as(const Seg<DT>& z, char* out, int seg, int lane, int V, F&& f) {
  constexpr int in = Type<DT>::kInPacket;
  const bool whole = seg * kScoreSeg + kScoreSeg <= V;
#pragma unroll
  for (int q = 0; q < Seg<DT>::kPackets; q++) {
    const int j = seg * kScoreSeg + (q * 64 + lane) * in;
    float v[in];
#pragma unroll
    for (int i = 0; i < in; i++) v[i] = f(value<DT>(z.w[q], i), j + i);
    packet p;
#pragma unroll
    for (int d = 0; d < 4; d++)
      p[d] = DT == DTL_F32 ? bits_of<DT>(v[d]) : bits_of<DT>(v[2 * d % in]) | bits_of<DT>(v[(2 * d + 1) % in]) << 16;
    if (whole || j + in <= V) {
      auto* to = reinterpret_cast<typename Type<DT>::mem*>(out + (size_t)j * Type<DT>::kBytes);
      if (PAST)
        __builtin_nontemporal_store(p, to);
      else
        *to = p;
    } else {
#pragma unroll
      for (int i = 0; i < in; i++)
        if (j + i < V) store_one<DT>(out, j + i, v[i]);
    }
  }
}

template <int DT, typename F>
__device__ __forceinline__ void write_seg(const Seg<DT>& z, char* out, int seg, int lane, int V, bool past, F&& f) {
  if (past)
    write_seg_as<DT, true>(z, out, seg, lane, V, f);
  else
    write_seg_as<DT, false>(z, out, seg, lane, V, f);
}

template <int DT, bool ENT>
__global__ __launch_bounds__(kGradWaves * 64) void k_scores_grad(ScoreGradK a) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const float no = -__builtin_inff();
  const size_t row = a.row0 + (gridDim.x - 1 - blockIdx.x) / a.chunks;  // the forward's last rows first
  const int seg = (int)(blockIdx.x % a.chunks) * kGradWaves + wave;
  if (seg >= a.nseg) return;
  const char* z = a.z + row * a.row_bytes;
  char* out = a.grad + row * a.grad_bytes;
  const long y = a.tokens ? load_index(a.tokens, a.wide, row) : -1;
  const double g = a.g && y >= 0 ? a.g[row] : 0.0f, h = ENT && a.h ? a.h[row] : 0.0f;
  const float m = a.stats[2 * row];
  const double r = a.stats[2 * row + 1], p0 = 1.0 / (1.0 + r);
  // padding, and rows whose mask leaves nothing: zeros, whatever they hold
  const bool zero = (g == 0.0 && h == 0.0) || m == no;
  const bool bad = y >= a.V, here = y >= 0 && !bad && !zero && (int)(y / kScoreSeg) == seg;
  double l = 0.0, hh = 0.0;
  if (ENT || here) {
    l = log1p(r);
    hh = ENT ? (double)a.entropy[row] - l : 0.0;
  }
  const float A = bad ? __builtin_nanf("") : (float)(-a.inv_t * p0 * (g + h * hh)), B = (float)(-a.inv_t * p0 * h * kLn2);
  float at_y = 0.0f;
  if (here) {
    const double t = ((double)load_one<DT>(z, (int)y) - m) * a.inv_t, lp = t - l;
    // log p of a masked token is -inf and its p log p is 0
    at_y = (float)(a.inv_t * (-g * expm1(lp) - (ENT && h != 0.0 && lp > -1e30 ? h * exp(lp) * (t + hh) : 0.0)));
  }
  Seg<DT> s;
  if (zero) {
    write_seg<DT>(s, out, seg, lane, a.V, a.past, [](float, int) { return 0.0f; });
    return;
  }
  load_seg<DT, false>(s, z, seg, lane, a.V);
  auto value_of = [&](float v) {
    const float t = (v - m) * a.c, e = __builtin_amdgcn_exp2f(t);
    return e * (ENT ? __builtin_fmaf(B, fmaxf(t, kLowest), A) : A);
  };
  if (here)
    write_seg<DT>(s, out, seg, lane, a.V, a.past, [&](float v, int j) { return j == (int)y ? at_y : value_of(v); });
  else
    write_seg<DT>(s, out, seg, lane, a.V, a.past, [&](float v, int) { return value_of(v); });
}

// ---- distillation ------------------------------------------------------------------------

// A row's teacher: up to 256 slots (id, log probability v).
//   renormalised: p_k = e^(v_k) / sum;  rest: p_k = e^(v_k), and what is left of
//   one is the teacher's mass outside the list.
// loss = w T^2 (sum p_k (log p_k - log q_k) + rest (log rest - log q_rest)); the
// last term only where a logit outside the list is unmasked.
// dz_j = w T (e_j share - p_j) with share = (sum p + rest) / sum of e.  For j
// outside the list both terms are relative to the largest logit there, which may
// lie far below the list's: with e'_j = 2^((z_j - out_m) c) <= 1 and out_a =
// share e^((out_m - m) / T) - rest / sum of e', dz_j = w T e'_j out_a.
// The slots' terms are formed in 64 bits: the loss is a small difference of
// large ones.
struct DistillK {
  const char* z;
  char* grad;
  size_t row_bytes, grad_bytes, row0;
  int V, nseg, groups;
  bool once, past;  // read (a loss alone), write past the caches
  const void* ids;
  int wide, k;
  const float* teacher;
  const float* weights;
  float c, T;
  double inv_t;
  float* loss;
  float* stats;  // [rows][kDistillStats]: put_stats
  Part* parts;
};

// The row's slots and their logits.
struct alignas(16) Slots {
  int32_t id[kDistillMaxK];  // -1: empty
  float v[kDistillMaxK];
  float z[kDistillMaxK];
  int bits[kDistillMaxK / 64];
};
enum { USED = 1, BROKEN = 2 };

// Loads the slots: one for each of 256 threads.  After the barrier that follows,
// slots_state tells whether the row has a slot in use and whether one is broken:
// an id past the vocabulary, a log probability that is NaN or +inf (or with
// rest such a logit, which the pass over the row leaves out).
template <int DT, bool REST>
__device__ __forceinline__ void load_slots(Slots& s, const DistillK& a, size_t row, const char* z) {
  const int k = threadIdx.x;
  if (k >= kDistillMaxK) return;
  int id = -1, bits = 0;
  float v = -__builtin_inff(), zk = v;
  if (k < a.k) {
    const long j = load_index(a.ids, a.wide, row * a.k + k);
    v = a.teacher[row * a.k + k];
    if (j >= 0 && v != -__builtin_inff()) {
      bits = USED;
      if (j >= a.V || !(v < __builtin_inff())) {
        bits |= BROKEN;
      } else {
        id = (int)j;
        zk = load_one<DT>(z, id);
        if (REST && !(zk < __builtin_inff())) bits |= BROKEN;
      }
    }
  }
  s.id[k] = id;
  s.v[k] = v;
  s.z[k] = zk;
  const int any = (__ballot(bits & USED) ? USED : 0) | (__ballot(bits & BROKEN) ? BROKEN : 0);
  if ((k & 63) == 0) s.bits[k >> 6] = any;
}
__device__ __forceinline__ int slots_state(const Slots& s) {
  int bits = 0;
#pragma unroll
  for (int i = 0; i < kDistillMaxK / 64; i++) bits |= s.bits[i];
  return __builtin_amdgcn_readfirstlane(bits);
}

// Which lane's which logit of a segment an id is: the bit of the segments' mask.
template <int DT>
__device__ __forceinline__ void mask_bit(uint32_t* mask, int id) {
  constexpr int in = Type<DT>::kInPacket;
  const int seg = id / kScoreSeg, at = id % kScoreSeg;
  const int q = at / (64 * in), lane = at / in % 64;
  atomicOr(&mask[seg * 64 + lane], 1u << (q * in + at % in));
}

// What the slots alone give, a wave's share: with p proportional to e^(v - v0),
// v0 the share's largest v (0 with rest, where p = e^v), z0 its largest logit.
struct SlotSums {
  double v0, sum, sum_v, sum_z;  // of e^(v - v0), and of it times v - v0 and times z - z0
  double z0, in;                 // rest: sum of e^((z - z0) / T) over distinct ids
};

template <bool REST>
__device__ __forceinline__ void sum_slots(const Slots& s, SlotSums* sums, int waves, double inv_t) {
  const float no = -__builtin_inff();
  for (int w = threadIdx.x >> 6; w < kDistillMaxK / 64; w += waves) {
    const int lane = threadIdx.x & 63, k = w * 64 + lane, id = s.id[k];
    const float v = s.v[k], z = s.z[k];
    SlotSums t{};
    if (!REST) {
      const float most = wave_max(id >= 0 ? v : no);
      t.v0 = most == no ? 0.0 : most;
    }
    const double e = id >= 0 ? exp((double)v - t.v0) : 0.0;
    t.sum = wave_sum(e);
    t.sum_v = wave_sum(e > 0.0 ? e * ((double)v - t.v0) : 0.0);
    const float z0 = wave_max(id >= 0 ? z : no);
    t.z0 = z0;
    t.sum_z = wave_sum(!(e > 0.0) ? 0.0 : z == no ? (double)no : e * ((double)z - z0));
    if (REST) {
      bool first = id >= 0;
      const int4* ids = reinterpret_cast<const int4*>(s.id);
      for (int j = 0; j < w * 16; j++) {
        const int4 x = ids[j];
        first = first && x.x != id && x.y != id && x.z != id && x.w != id;
      }
      for (int j = 0; j < 64; j++) first = first && (j >= lane || __builtin_amdgcn_readlane(id, j) != id);
      t.in = wave_sum(first && z != no ? exp(((double)z - z0) * inv_t) : 0.0);
    }
    if (lane == 0) sums[w] = t;
  }
}

// What a row's gradient needs besides its logits: m and share for the list's,
// out_m and out_a for the others, and for p = e^(v - v0) / sum the list's largest v
// and the log of the sum as a float and what it leaves (with rest all 0: p = e^v).
// v0 is not joined with the log, which a v0 of any size would swallow.
struct RowGrad {
  float m, share, out_m, out_a, v0, log_hi, log_lo;
};

// From the forward to the backward: without rest out_m is m and out_a is share.
template <bool REST>
__device__ __forceinline__ void put_stats(float* stats, size_t row, const RowGrad& g) {
  float* s = stats + row * kDistillStats;
  s[0] = g.m;
  s[1] = g.share;
  s[2] = REST ? g.out_m : g.v0;
  s[3] = REST ? g.out_a : g.log_hi;
  s[4] = REST ? 0.0f : g.log_lo;
}
template <bool REST>
__device__ __forceinline__ RowGrad get_stats(const float* stats, size_t row) {
  const float* s = stats + row * kDistillStats;
  return REST ? RowGrad{s[0], s[1], s[2], s[3], 0.0f, 0.0f, 0.0f} : RowGrad{s[0], s[1], s[0], s[1], s[2], s[3], s[4]};
}

// The row's loss (times T^2) and what its gradient needs, from the row's stats
// (with rest those outside the list) and the slots' sums.
template <bool REST>
__device__ __forceinline__ RowGrad join_distill(const DistillK& a, const RowStats& st, const SlotSums* sums, int state, float* loss) {
  const float no = -__builtin_inff(), nan = __builtin_nanf("");
  if (!(state & USED)) {
    *loss = 0.0f;
    return RowGrad{};
  }
  if (st.bad || (state & BROKEN)) {
    *loss = nan;
    return RowGrad{nan, nan, nan, nan, nan, nan, nan};
  }
  constexpr int n = kDistillMaxK / 64;
  double v0 = no, z0 = no;
#pragma unroll
  for (int i = 0; i < n; i++) {
    if (sums[i].sum > 0.0) v0 = fmax(v0, sums[i].v0);
    z0 = fmax(z0, sums[i].z0);
  }
  // total of e relative to m, the row's largest logit.  With rest st has the sums
  // without the list; down: from its maximum to m, and log left, the log of what
  // the others have of the total, without down's underflow.
  double total = 1.0 + st.r, down = 1.0, log_left = 0.0, m = st.m;
  if (REST) {
    m = fmax(m, z0);
    down = st.m == no ? 0.0 : exp((st.m - m) * a.inv_t);
    log_left = (st.m - m) * a.inv_t + log1p(st.r);
    total = down * (1.0 + st.r);
  }
  if (m == no) {  // every logit masked: no q to compare with, nothing to move
    *loss = __builtin_inff();
    return RowGrad{no, 0.0f, no, 0.0f, 0.0f, 0.0f, 0.0f};
  }
  double mass = 0.0, own = 0.0, cross = 0.0;  // sum of p, p (v - v0) and p (z - m)
#pragma unroll
  for (int i = 0; i < n; i++) {
    const SlotSums& x = sums[i];
    if (REST && x.z0 > no) total += x.in * exp((x.z0 - m) * a.inv_t);
    const double f = x.sum > 0.0 ? exp(x.v0 - v0) : 0.0;
    if (f > 0.0) {
      mass += f * x.sum;
      own += f * (x.sum_v + x.sum * (x.v0 - v0));
      cross += f * (x.sum_z + x.sum * (x.z0 - m));
    }
  }
  const double log_total = REST ? log(total) : log1p(st.r);
  double log_sum = 0.0;
  if (!REST) {
    log_sum = log(mass);
    cross /= mass;
    own = own / mass - log_sum;
    mass = 1.0;
  }
  double term = own - cross * a.inv_t + mass * log_total;
  double rest = 0.0;
  if (REST && st.m != no) {
    rest = fmax(0.0, 1.0 - mass);
    if (rest > 0.0) term += rest * (log(rest) - (log_left - log_total));
  }
  *loss = (float)((double)a.T * a.T * term);
  RowGrad g;
  g.m = (float)m;
  g.share = (float)((mass + rest) / total);
  // where every logit outside is masked e' is 0 as long as out_m is finite
  g.out_m = REST && st.m == no ? g.m : st.m;
  g.out_a = (float)(down * ((mass + rest) / total) - rest / (1.0 + st.r));
  g.v0 = REST ? 0.0f : (float)v0;
  g.log_hi = (float)log_sum;
  g.log_lo = (float)(log_sum - g.log_hi);
  return g;
}

// Gradient of a segment for every j as if outside the list (a listed logit's may
// be anything: its slot writes it again).
template <int DT>
__device__ __forceinline__ void grad_seg(const DistillK& a, const Seg<DT>& s, char* out, const RowGrad& g, float scale,
                                         int seg, int lane) {
  const float A = scale * g.out_a;
  write_seg<DT>(s, out, seg, lane, a.V, a.past,
                [&](float v, int) { return __builtin_amdgcn_exp2f((v - g.out_m) * a.c) * A; });
}
template <int DT>
__device__ __forceinline__ void zero_seg(char* out, int seg, int lane, int V) {
  Seg<DT> s;
  write_seg_as<DT, false>(s, out, seg, lane, V, [](float, int) { return 0.0f; });
}
__device__ __forceinline__ bool grad_is_zero(const RowGrad& g, float scale) {
  return scale == 0.0f || g.m == -__builtin_inff();
}

// The gradient at slot k's id, by the first slot of each distinct id.  Its
// logit is the slots': the gradient may lie over the logits.
template <int DT>
__device__ __forceinline__ void grad_slot(const DistillK& a, char* out, const Slots& s, const RowGrad& g, float scale,
                                          int k) {
  const int id = s.id[k];
  const int4* ids = reinterpret_cast<const int4*>(s.id);
  int before = 0, behind = 0;  // other slots of this id
  for (int j = 0; 4 * j < a.k; j++) {
    const int4 x = ids[j];
    const int n = (x.x == id) + (x.y == id) + (x.z == id) + (x.w == id);
    before += 4 * j < (k & ~3) ? n : 0;
    behind += 4 * j > k ? n : 0;
    if (j == k / 4) {
      before += (x.x == id && (k & 3) > 0) + (x.y == id && (k & 3) > 1) + (x.z == id && (k & 3) > 2);
      behind += (x.y == id && (k & 3) < 1) + (x.z == id && (k & 3) < 2) + (x.w == id && (k & 3) < 3);
    }
  }
  if (before) return;  // an earlier slot of the same id writes it
  const auto p_of = [&](float v) { return exp(((double)v - g.v0) - g.log_hi - g.log_lo); };
  double p = p_of(s.v[k]);
  for (int j = k + 1; behind && j < a.k; j++)
    if (s.id[j] == id) p += p_of(s.v[j]);
  const float e = __builtin_amdgcn_exp2f((s.z[k] - g.m) * a.c);
  store_one<DT>(out, id, (float)((double)scale * ((double)e * g.share - p)));
}

// Losses, by whole rows or from parts.
template <int DT, bool REST, int PHASE, int THREADS>
__global__ __launch_bounds__(THREADS) void k_distill(DistillK a) {
  extern __shared__ uint32_t mask[];  // REST: [nseg * 64]
  __shared__ Part lds_parts[PHASE == PARTS ? 1 : kScoreMaxSegs];
  __shared__ Slots s;
  __shared__ SlotSums sums[kDistillMaxK / 64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  constexpr int waves = THREADS / 64;
  const size_t row = PHASE == PARTS ? blockIdx.x / a.groups : a.row0 + blockIdx.x;
  const char* z = a.z + row * a.row_bytes;
  const float w = a.weights ? a.weights[row] : 1.0f;

  // a row that does not count, or has no slots in use, is not read
  int state = 0;
  if (w != 0.0f) {
    if (REST)
      for (int i = threadIdx.x; i < a.nseg * 64; i += THREADS) mask[i] = 0;
    load_slots<DT, REST>(s, a, row, z);
    __syncthreads();
    state = slots_state(s);
  }
  if (state) {
    if (REST) {
      if (threadIdx.x < kDistillMaxK && s.id[threadIdx.x] >= 0) mask_bit<DT>(mask, s.id[threadIdx.x]);
      __syncthreads();
    }
    if constexpr (PHASE == PARTS) {
      const int g = (int)(blockIdx.x % a.groups), per = (a.nseg + a.groups - 1) / a.groups;
      read_segs<DT, false, false>(z, a.V, g * per, min(a.nseg, (g + 1) * per), wave, waves, lane, a.c, false,
                                  a.parts + row * a.nseg, nullptr, REST ? mask : nullptr);
      return;
    }
    sum_slots<REST>(s, sums, waves, a.inv_t);
    if constexpr (PHASE == WHOLE) {
      read_segs<DT, false, false>(z, a.V, 0, a.nseg, wave, waves, lane, a.c, a.once, lds_parts, nullptr,
                                  REST ? mask : nullptr);
    } else {
      for (int i = threadIdx.x; i < a.nseg; i += THREADS) lds_parts[i] = a.parts[row * a.nseg + i];
    }
  }
  if constexpr (PHASE == PARTS) return;
  __syncthreads();
  if (wave != 0) return;
  RowStats st{};
  if (state) st = join_row<DT, false>(z, a.V, a.nseg, lds_parts, REST ? mask : nullptr, a.c, lane);
  float loss;
  const RowGrad g = join_distill<REST>(a, st, sums, state, &loss);
  if (lane == 0) {
    a.loss[row] = state ? w * loss : 0.0f;
    if (a.stats) put_stats<REST>(a.stats, row, g);
  }
}

// A loss and its gradient.  Between the two a wave keeps its first NS segments of
// the row in registers, so that they are read once; of longer rows (LONGER) the
// rest is read again.
template <int DT, bool REST, int NS, bool LONGER, int THREADS>
__global__ __launch_bounds__(THREADS) void k_distill_step(DistillK a) {
  extern __shared__ uint32_t mask[];  // REST: [nseg * 64]
  constexpr int waves = THREADS / 64;
  __shared__ Part lds_parts[kScoreMaxSegs];
  __shared__ Slots s;
  __shared__ SlotSums sums[kDistillMaxK / 64];
  __shared__ RowGrad row_grad;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const size_t row = a.row0 + blockIdx.x;
  const char* z = a.z + row * a.row_bytes;
  char* out = a.grad + row * a.grad_bytes;
  const float w = a.weights ? a.weights[row] : 1.0f;
  if (w == 0.0f) {  // a row that does not count is not read
    for (int seg = wave; seg < a.nseg; seg += waves) zero_seg<DT>(out, seg, lane, a.V);
    if (threadIdx.x == 0) a.loss[row] = 0.0f;
    return;
  }
  Seg<DT> held[NS];
#pragma unroll
  for (int i = 0; i < NS; i++)
    if (i * waves + wave < a.nseg) load_seg<DT, false>(held[i], z, i * waves + wave, lane, a.V);
  if (REST)
    for (int i = threadIdx.x; i < a.nseg * 64; i += THREADS) mask[i] = 0;
  load_slots<DT, REST>(s, a, row, z);
  __syncthreads();
  const int state = slots_state(s);
  if (REST) {
    if (threadIdx.x < kDistillMaxK && s.id[threadIdx.x] >= 0) mask_bit<DT>(mask, s.id[threadIdx.x]);
    __syncthreads();
  }
  sum_slots<REST>(s, sums, waves, a.inv_t);
  auto reduce = [&](Seg<DT>& x, int seg) {
    if (REST) {  // the listed logits' gradients are written by their slots
      const uint32_t bits = mask[seg * 64 + lane];
      if (__ballot(bits != 0)) mask_seg<DT>(x, bits);
    }
    const Part p = seg_part<DT, false>(x, lane_max<DT>(x), a.c);
    if (lane == 0) lds_parts[seg] = p;
    __builtin_amdgcn_sched_barrier(0);  // one segment's temporaries at a time
  };
#pragma unroll
  for (int i = 0; i < NS; i++)
    if (i * waves + wave < a.nseg) reduce(held[i], i * waves + wave);
  if (LONGER)
    for (int seg = NS * waves + wave; seg < a.nseg; seg += waves) {
      Seg<DT> x;
      load_seg<DT, false>(x, z, seg, lane, a.V);
      reduce(x, seg);
    }
  __syncthreads();

  // the wave that has the maximum's segment joins the row
  const RowMax top = find_max(lds_parts, a.nseg, lane);
  if (wave == top.first % waves) {
    float rs = 0.0f, rw = 0.0f;
    if (!top.none) {
#pragma unroll
      for (int i = 0; i < NS; i++)
        if (top.first == i * waves + wave) sums_without_max<DT, false>(held[i], top.m, a.c, lane, rs, rw);
      if (LONGER && top.first >= NS * waves) {
        Seg<DT> y;
        load_seg<DT, false>(y, z, top.first, lane, a.V);
        if (REST) mask_seg<DT>(y, mask[top.first * 64 + lane]);
        sums_without_max<DT, false>(y, top.m, a.c, lane, rs, rw);
      }
    }
    float loss;
    const RowGrad g =
        join_distill<REST>(a, join_parts<false>(top, lds_parts, a.nseg, rs, rw, a.c, lane), sums, state, &loss);
    if (lane == 0) {
      row_grad = g;
      a.loss[row] = state ? w * loss : 0.0f;
    }
  }
  __syncthreads();
  const RowGrad g = row_grad;
  const float scale = state ? w * a.T : 0.0f;
  const bool zero = grad_is_zero(g, scale);
#pragma unroll
  for (int i = 0; i < NS; i++) {
    const int seg = i * waves + wave;
    if (seg < a.nseg) {
      if (zero)
        zero_seg<DT>(out, seg, lane, a.V);
      else
        grad_seg<DT>(a, held[i], out, g, scale, seg, lane);
    }
    __builtin_amdgcn_sched_barrier(0);
  }
  if (LONGER)
    for (int seg = NS * waves + wave; seg < a.nseg; seg += waves) {
      if (zero) {
        zero_seg<DT>(out, seg, lane, a.V);
      } else {
        Seg<DT> x;
        load_seg<DT, false>(x, z, seg, lane, a.V);
        grad_seg<DT>(a, x, out, g, scale, seg, lane);
      }
    }
  wait_for_stores();
  const int k = threadIdx.x;
  if (!zero && k < a.k && s.id[k] >= 0) grad_slot<DT>(a, out, s, g, scale, k);
}

// The gradient alone, from the stats of the forward: workgroups of four segments
// of a row each (2048 rows of 151936 f32: 447 us, 467 with sixteen).
template <int DT, bool REST>
__global__ __launch_bounds__(kGradWaves * 64) void k_distill_grad(DistillK a) {
  __shared__ Slots s;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const size_t row = a.row0 + (gridDim.x - 1 - blockIdx.x) / a.groups;  // the forward's last rows first
  const int seg0 = (int)(blockIdx.x % a.groups) * kGradWaves, seg = seg0 + wave;
  const char* z = a.z + row * a.row_bytes;
  char* out = a.grad + row * a.grad_bytes;
  const float weight = a.weights ? a.weights[row] : 1.0f;
  if (weight == 0.0f) {  // a row that does not count is not read
    if (seg < a.nseg) zero_seg<DT>(out, seg, lane, a.V);
    return;
  }
  const RowGrad g = get_stats<REST>(a.stats, row);
  load_slots<DT, false>(s, a, row, z);
  __syncthreads();
  const float scale = slots_state(s) ? weight * a.T : 0.0f;
  const bool zero = grad_is_zero(g, scale);
  if (seg < a.nseg) {
    if (zero) {
      zero_seg<DT>(out, seg, lane, a.V);
    } else {
      Seg<DT> x;
      load_seg<DT, false>(x, z, seg, lane, a.V);
      grad_seg<DT>(a, x, out, g, scale, seg, lane);
    }
  }
  wait_for_stores();
  const int k = threadIdx.x, id = s.id[k];
  if (!zero && id >= seg0 * kScoreSeg && id < (seg0 + kGradWaves) * kScoreSeg) grad_slot<DT>(a, out, s, g, scale, k);
}
static_assert(kGradWaves * 64 == kDistillMaxK && kPartThreads >= kDistillMaxK,
              "a thread a slot");

// ---- launches ---------------------------------------------------------------------------

// Whether a row is one workgroup's.  Few long rows would leave compute units idle
// and go to several workgroups each, with a second launch to join them.  us on the
// device by whole rows / in parts, scores of bf16: 1 row of 32000 5.6 / 6.6, of
// 60000 7.9 / 6.7 (and one launch less on the host), of 151936 13.3 / 6.7; of
// 151936 64 rows 14.0 / 10.0, 100 rows 14.8 / 11.8, 128 rows 15.5 / 15.1, 159 rows
// 16.5 / 17.5; with 20 alternatives 128 rows 21.1 / 21.3; losses of 128 rows 14.3 /
// 15.0, of f32 18.1 / 20.4.
bool whole_rows(size_t rows, int nseg) { return nseg <= 32 || rows >= 128; }

int segments(size_t vocab) { return (int)((vocab + kScoreSeg - 1) / kScoreSeg); }

// Workgroups of four waves for a row in the split form: as many as its segments
// keep busy, until the chip has enough.
int part_groups(size_t rows, int nseg) {
  const size_t most = (nseg + kPartThreads / 64 - 1) / (kPartThreads / 64);
  const size_t enough = (2048 + rows - 1) / rows;
  return (int)(most < enough ? most : enough);
}

// Logits larger than the memory-side cache of 256 MB are read past it: 7.0 TB/s
// instead of 6.2 on 1.24 GB.  Smaller ones are not: it leaves nothing behind, and a
// backward pass over 32 MB then takes 18.6 us instead of 15.0.  (Leaving the last 192
// MB of larger ones to a backward pass made the forward as much slower, 238 instead
// of 205 us, as the backward faster.)
bool read_past(size_t rows, size_t row_bytes) { return rows * row_bytes > (size_t)256 << 20; }

// Whole rows go to workgroups of one, four or eight waves by their length (us of
// 16384 rows of 1000 bf16 with one / four / eight: scores 30 / - / 80, with 20
// alternatives - / 149 / 225, losses - / 57 / 93), and of sixteen where there are
// too few rows for several workgroups a compute unit, which reads faster the more
// waves it has (64 rows of 32000 f32 6.6 instead of 7.1).  Scores of many rows of
// middle length take four waves too, more rows side by side for the selection to
// hide behind: 4096 rows with 20 alternatives, four / eight waves: of 16000 f32 63 /
// 87, of 32000 f32 104 / 131, of 49152 bf16 96 / 101, 100000 bf16 159 / 157; 400 rows of
// 32000 bf16 17.7 / 15.8; with 128 alternatives the candidates' LDS leaves room for
// too few (of 151936 bf16 360 / 269).  Calls without alternatives follow the same
// rule; they were not measured.
bool wide_rows(size_t rows, int nseg) { return rows <= 256 && nseg > 8; }


}  // namespace

size_t score_scratch_bytes(size_t rows, size_t vocab, size_t top) {
  const size_t nseg = segments(vocab);
  if (whole_rows(rows, (int)nseg)) return 0;
  return round256(rows * nseg * sizeof(Part)) + (top ? rows * nseg * 64 * 4 : 0);
}

void launch_token_scores(const ScoreArgs& a, hipStream_t s) {
  if (a.rows == 0) return;
  ScoreK k{};
  k.z = static_cast<const char*>(a.z);
  k.row_bytes = a.stride * type_bytes(a.dtype);
  k.V = a.vocab;
  k.nseg = segments(a.vocab);
  k.tokens = a.tokens;
  k.wide = a.wide;
  k.top = a.top;
  k.c = (float)(kLog2E / a.temperature);
  k.inv_t = 1.0 / a.temperature;
  k.log_probs = a.log_probs;
  k.entropy = a.entropy;
  k.stats = a.stats;
  k.top_ids = a.top_ids;
  k.top_log_probs = a.top_log_probs;
  size_t lds = 0;
  if (a.top) {
    lds = candidate_bytes(a.top);
    if (lds > (size_t)k.nseg * kScoreSeg * 8) lds = (size_t)k.nseg * kScoreSeg * 8;  // a short row has no more
    if (lds < (size_t)k.nseg * 256) lds = (size_t)k.nseg * 256;
  }
  by_type(a.dtype, [&](auto dt) {
    by_bool(a.top != 0, [&](auto with_top) {
      constexpr int DT = decltype(dt)::value;
      constexpr bool TOP = decltype(with_top)::value;
      if (whole_rows(a.rows, k.nseg)) {
        k.once = read_past(a.rows, k.row_bytes);
        if (!TOP && k.nseg == 1) {
          if constexpr (!TOP) launch_rows(k_scores<DT, false, WHOLE, 64>, a.rows, 1, 64, lds, s, k);
        } else if (k.nseg <= 4 || (a.rows >= 1024 && k.nseg <= 48 && a.top <= 32)) {
          launch_rows(k_scores<DT, TOP, WHOLE, 256>, a.rows, 1, 256, lds, s, k);
        } else if (wide_rows(a.rows, k.nseg)) {
          launch_rows(k_scores<DT, TOP, WHOLE, 1024>, a.rows, 1, 1024, lds, s, k);
        } else {
          launch_rows(k_scores<DT, TOP, WHOLE, 512>, a.rows, 1, 512, lds, s, k);
        }
        return;
      }
      k.groups = part_groups(a.rows, k.nseg);
      k.parts = static_cast<Part*>(a.scratch);
      k.keys = reinterpret_cast<uint32_t*>(static_cast<char*>(a.scratch) + round256(a.rows * k.nseg * sizeof(Part)));
      launch_rows(k_scores<DT, TOP, PARTS, kPartThreads>, a.rows, k.groups, kPartThreads, 0, s, k);
      launch_rows(k_scores<DT, TOP, JOIN, kJoinThreads>, a.rows, 1, kJoinThreads, lds, s, k);
    });
  });
}

void launch_token_scores_grad(const ScoreGradArgs& a, hipStream_t s) {
  if (a.rows == 0) return;
  ScoreGradK k{};
  k.z = static_cast<const char*>(a.z);
  k.grad = static_cast<char*>(a.grad);
  k.row_bytes = a.stride * type_bytes(a.dtype);
  k.grad_bytes = a.grad_stride * type_bytes(a.dtype);
  k.V = a.vocab;
  k.nseg = segments(a.vocab);
  k.chunks = (k.nseg + kGradWaves - 1) / kGradWaves;
  k.past = write_past(a.rows, k.grad_bytes);
  k.tokens = a.tokens;
  k.wide = a.wide;
  k.c = (float)(kLog2E / a.temperature);
  k.inv_t = 1.0 / a.temperature;
  k.stats = a.stats;
  k.entropy = a.entropy;
  k.g = a.g_log_probs;
  k.h = a.g_entropy;
  by_type(a.dtype, [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    launch_rows(a.g_entropy ? k_scores_grad<DT, true> : k_scores_grad<DT, false>, a.rows, k.chunks, kGradWaves * 64, 0,
                s, k);
  });
}

namespace {
DistillK distill_kernel_args(const DistillArgs& a) {
  DistillK k{};
  k.z = static_cast<const char*>(a.z);
  k.grad = static_cast<char*>(a.grad);
  k.row_bytes = a.stride * type_bytes(a.dtype);
  k.grad_bytes = a.grad_stride * type_bytes(a.dtype);
  k.V = a.vocab;
  k.nseg = segments(a.vocab);
  k.ids = a.ids;
  k.wide = a.wide;
  k.k = a.k;
  k.teacher = a.teacher;
  k.weights = a.weights;
  k.c = (float)(kLog2E / a.temperature);
  k.T = a.temperature;
  k.inv_t = 1.0 / a.temperature;
  k.loss = a.loss;
  k.stats = a.stats;
  k.past = write_past(a.rows, k.grad_bytes);
  return k;
}
}  // namespace

// Parts, and for a step of few rows the stats between its launches.
size_t distill_scratch_bytes(size_t rows, size_t vocab, bool step) {
  if (whole_rows(rows, segments(vocab))) return 0;
  return round256(rows * segments(vocab) * sizeof(Part)) + (step ? rows * kDistillStats * sizeof(float) : 0);
}

void launch_distill_grad(const DistillArgs& a, hipStream_t s) {
  if (a.rows == 0) return;
  DistillK k = distill_kernel_args(a);
  k.groups = (k.nseg + kGradWaves - 1) / kGradWaves;
  by_type(a.dtype, [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    launch_rows(a.rest ? k_distill_grad<DT, true> : k_distill_grad<DT, false>, a.rows, k.groups, kGradWaves * 64, 0, s,
                k);
  });
}

namespace {
template <int DT, bool REST, int NS, bool LONGER, int THREADS>
void launch_step_as(const DistillK& k, size_t rows, hipStream_t s) {
  launch_rows(k_distill_step<DT, REST, NS, LONGER, THREADS>, rows, 1, THREADS, REST ? (size_t)k.nseg * 256 : 0, s, k);
}
// A step of whole rows, by their length alone (the figures are of 2048 rows and
// more; fewer were not compared).  Workgroups that hold only part of a long row
// leave room for two or three of them a compute unit, one reading while another
// writes; us by segments held a wave x waves:
//   4096 rows of 32000 bf16   2 x 8 (all) 109, 4 x 4 (all) 111, 1 x 16 (all) 175
//   4096 rows of 49152 bf16   2 x 8 158, 3 x 8 (all) 158, 1 x 8 168, 2 x 16 225
//   4096 rows of 151936 bf16  4 x 8 515, 3 x 8 523, 2 x 8 543, 1 x 8 562, 5 x 16 (all) 601
//   4096 rows of 32000 f32    2 x 8 (all) 188, 4 x 4 (all) 203, 1 x 16 (all) 234
//   4096 rows of 49152 f32    2 x 8 308, 1 x 8 317, 3 x 8 323, 2 x 16 320
//   2048 rows of 151936 f32   2 x 16 509, 3 x 8 520, 2 x 8 547, 1 x 8 546, 2 x 4 683
template <int DT, bool REST>
void launch_step(const DistillK& k, size_t rows, hipStream_t s) {
  if (k.nseg <= 4) return launch_step_as<DT, REST, 1, false, 256>(k, rows, s);
  if (k.nseg <= 8) return launch_step_as<DT, REST, 1, false, 512>(k, rows, s);
  if (k.nseg <= 16) return launch_step_as<DT, REST, 2, false, 512>(k, rows, s);
  if (k.nseg <= 32) return launch_step_as<DT, REST, 2, true, 512>(k, rows, s);
  if constexpr (DT == DTL_F32)
    launch_step_as<DT, REST, 2, true, 1024>(k, rows, s);
  else
    launch_step_as<DT, REST, 4, true, 512>(k, rows, s);
}
}  // namespace

void launch_distill(const DistillArgs& a, hipStream_t s) {
  if (a.rows == 0) return;
  DistillK k = distill_kernel_args(a);
  const size_t lds = a.rest ? (size_t)k.nseg * 256 : 0;
  k.once = read_past(a.rows, k.row_bytes);
  by_type(a.dtype, [&](auto dt) {
    by_bool(a.rest, [&](auto with_rest) {
      constexpr int DT = decltype(dt)::value;
      constexpr bool REST = decltype(with_rest)::value;
      if (whole_rows(a.rows, k.nseg)) {
        if (a.grad)
          launch_step<DT, REST>(k, a.rows, s);
        else if (k.nseg <= 4)
          launch_rows(k_distill<DT, REST, WHOLE, 256>, a.rows, 1, 256, lds, s, k);
        else if (wide_rows(a.rows, k.nseg))
          launch_rows(k_distill<DT, REST, WHOLE, 1024>, a.rows, 1, 1024, lds, s, k);
        else
          launch_rows(k_distill<DT, REST, WHOLE, 512>, a.rows, 1, 512, lds, s, k);
        return;
      }
      k.groups = part_groups(a.rows, k.nseg);
      k.parts = static_cast<Part*>(a.scratch);
      if (a.grad)
        k.stats = reinterpret_cast<float*>(static_cast<char*>(a.scratch) + round256(a.rows * k.nseg * sizeof(Part)));
      launch_rows(k_distill<DT, REST, PARTS, kPartThreads>, a.rows, k.groups, kPartThreads, lds, s, k);
      launch_rows(k_distill<DT, REST, JOIN, kJoinThreads>, a.rows, 1, kJoinThreads, lds, s, k);
    });
  });
  if (a.grad && !whole_rows(a.rows, k.nseg)) {
    DistillArgs b = a;
    b.stats = k.stats;
    launch_distill_grad(b, s);
  }
}

}  // namespace dtl

// ---- C entry points ------------------------------------------------------------------------

using namespace dtl;

namespace {

bool temperature_ok(float t) { return t >= kScoreMinTemperature && t <= kScoreMaxTemperature; }

DistillArgs distill_args(const dtl_logits* z, const dtl_teacher* t, float temperature) {
  DistillArgs a{};
  a.z = z->data;
  a.stride = z->stride;
  a.rows = z->rows;
  a.dtype = z->dtype;
  a.vocab = (int)z->vocab;
  a.ids = t->ids;
  a.wide = t->id_bytes == 8;
  a.teacher = t->log_probs;
  a.k = (int)t->k;
  a.rest = t->rest != 0;
  a.temperature = temperature;
  return a;
}
int check_distill(const dtl_logits* z, const dtl_teacher* t, float temperature) {
  const int st = check_logits(z);
  if (st) return st;
  if (!t || !index_bytes_ok(t->id_bytes) || !temperature_ok(temperature)) return DTL_ERR_INVALID_ARGUMENT;
  if (t->k == 0 || t->k > (size_t)kDistillMaxK) return DTL_ERR_SHAPE;
  if (z->rows && (!t->ids || !t->log_probs)) return DTL_ERR_INVALID_ARGUMENT;
  return DTL_OK;
}

}  // namespace

extern "C" {

size_t dtl_token_scores_scratch(size_t rows, size_t vocab, size_t top) {
  if (rows > kMostRows || vocab > (size_t)kScoreMaxVocab) return 0;
  return score_scratch_bytes(rows, vocab, top);
}

int dtl_token_scores(const dtl_logits* z, const void* tokens, int token_bytes, float temperature, size_t top,
                     float* log_probs, float* entropy, float* stats, int32_t* top_ids, float* top_log_probs,
                     void* scratch, size_t scratch_bytes, void* stream) {
  const int st = check_logits(z);
  if (st) return st;
  if (!temperature_ok(temperature) || (tokens && !index_bytes_ok(token_bytes))) return DTL_ERR_INVALID_ARGUMENT;
  if (top > (size_t)kScoreMaxTop || top > z->vocab) return DTL_ERR_SHAPE;
  if (z->rows == 0) return DTL_OK;
  if ((log_probs && !tokens) || (top && (!top_ids || !top_log_probs))) return DTL_ERR_INVALID_ARGUMENT;
  const size_t need = score_scratch_bytes(z->rows, z->vocab, top);
  if (scratch_bytes < need) return DTL_ERR_BUFFER_TOO_SMALL;
  if (need && (!scratch || reinterpret_cast<uintptr_t>(scratch) % 16)) return DTL_ERR_INVALID_ARGUMENT;
  ScoreArgs a{};
  a.z = z->data;
  a.stride = z->stride;
  a.rows = z->rows;
  a.dtype = z->dtype;
  a.vocab = (int)z->vocab;
  a.tokens = tokens;
  a.wide = token_bytes == 8;
  a.temperature = temperature;
  a.top = (int)top;
  a.log_probs = log_probs;
  a.entropy = entropy;
  a.stats = stats;
  a.top_ids = top_ids;
  a.top_log_probs = top_log_probs;
  a.scratch = scratch;
  launch_token_scores(a, static_cast<hipStream_t>(stream));
  return launch_status();
}

int dtl_token_scores_backward(const dtl_logits* z, const void* tokens, int token_bytes, float temperature,
                              const float* stats, const float* entropy, const float* grad_log_probs,
                              const float* grad_entropy, void* grad, size_t grad_stride, void* stream) {
  int st = check_logits(z);
  if (!st) st = check_grad(z, grad, grad_stride);
  if (st) return st;
  if (!temperature_ok(temperature) || (tokens && !index_bytes_ok(token_bytes))) return DTL_ERR_INVALID_ARGUMENT;
  if (z->rows == 0) return DTL_OK;
  if (!stats || (grad_log_probs && !tokens) || (grad_entropy && !entropy)) return DTL_ERR_INVALID_ARGUMENT;
  ScoreGradArgs a{};
  a.z = z->data;
  a.stride = z->stride;
  a.rows = z->rows;
  a.dtype = z->dtype;
  a.vocab = (int)z->vocab;
  a.tokens = tokens;
  a.wide = token_bytes == 8;
  a.temperature = temperature;
  a.stats = stats;
  a.entropy = entropy;
  a.g_log_probs = grad_log_probs;
  a.g_entropy = grad_entropy;
  a.grad = grad;
  a.grad_stride = grad_stride;
  launch_token_scores_grad(a, static_cast<hipStream_t>(stream));
  return launch_status();
}

size_t dtl_distill_scratch(size_t rows, size_t vocab) {
  if (rows > kMostRows || vocab > (size_t)kScoreMaxVocab) return 0;
  return distill_scratch_bytes(rows, vocab, true);
}

int dtl_distill(const dtl_logits* z, const dtl_teacher* teacher, float temperature, float* loss, float* stats,
                void* scratch, size_t scratch_bytes, void* stream) {
  const int st = check_distill(z, teacher, temperature);
  if (st) return st;
  if (z->rows == 0) return DTL_OK;
  if (!loss) return DTL_ERR_INVALID_ARGUMENT;
  const size_t need = distill_scratch_bytes(z->rows, z->vocab, false);
  if (scratch_bytes < need) return DTL_ERR_BUFFER_TOO_SMALL;
  if (need && (!scratch || reinterpret_cast<uintptr_t>(scratch) % 16)) return DTL_ERR_INVALID_ARGUMENT;
  DistillArgs a = distill_args(z, teacher, temperature);
  a.loss = loss;
  a.stats = stats;
  a.scratch = scratch;
  launch_distill(a, static_cast<hipStream_t>(stream));
  return launch_status();
}

int dtl_distill_backward(const dtl_logits* z, const dtl_teacher* teacher, float temperature, const float* stats,
                         const float* grad_loss, void* grad, size_t grad_stride, void* stream) {
  int st = check_distill(z, teacher, temperature);
  if (!st) st = check_grad(z, grad, grad_stride);
  if (st) return st;
  if (z->rows == 0) return DTL_OK;
  if (!stats || !grad_loss) return DTL_ERR_INVALID_ARGUMENT;
  DistillArgs a = distill_args(z, teacher, temperature);
  a.stats = const_cast<float*>(stats);
  a.weights = grad_loss;
  a.grad = grad;
  a.grad_stride = grad_stride;
  launch_distill_grad(a, static_cast<hipStream_t>(stream));
  return launch_status();
}

int dtl_distill_step(const dtl_logits* z, const dtl_teacher* teacher, float temperature, const float* weights,
                     float* loss, void* grad, size_t grad_stride, void* scratch, size_t scratch_bytes, void* stream) {
  int st = check_distill(z, teacher, temperature);
  if (!st) st = check_grad(z, grad, grad_stride);
  if (st) return st;
  if (z->rows == 0) return DTL_OK;
  if (!loss) return DTL_ERR_INVALID_ARGUMENT;
  const size_t need = distill_scratch_bytes(z->rows, z->vocab, true);
  if (scratch_bytes < need) return DTL_ERR_BUFFER_TOO_SMALL;
  if (need && (!scratch || reinterpret_cast<uintptr_t>(scratch) % 16)) return DTL_ERR_INVALID_ARGUMENT;
  DistillArgs a = distill_args(z, teacher, temperature);
  a.weights = weights;
  a.loss = loss;
  a.grad = grad;
  a.grad_stride = grad_stride;
  a.scratch = scratch;
  launch_distill(a, static_cast<hipStream_t>(stream));
  return launch_status();
}

}  // extern "C"
