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

#include "../csrc/dtl_device.h"

namespace dtl {
namespace {

constexpr int kRowThreads = 512;
constexpr int kRowWaves = kRowThreads / 64;
constexpr int kPer = kScoreSeg / 64;  // logits a lane holds of a segment
constexpr int kKeysPerThread = kScoreMaxSegs / kRowWaves;
constexpr double kLog2E = 1.4426950408889634074;
constexpr double kLn2 = 0.6931471805599453094;

// ---- logits of the three types ------------------------------------------------

// 16 bytes at an element's alignment: rows of an odd stride are only aligned
// to their elements, and gfx950 loads and stores 16 bytes at any address.
typedef uint32_t packet __attribute__((ext_vector_type(4)));
typedef packet packet4 __attribute__((aligned(4)));
typedef packet packet2 __attribute__((aligned(2)));

template <int DT>
struct Type {  // bf16 and f16
  static constexpr int kBytes = 2, kInPacket = 8, kPackets = kPer / 8;
  static constexpr uint32_t kMasked = DT == DTL_BF16 ? 0xff80ff80u : 0xfc00fc00u;
  typedef packet2 mem;
};
template <>
struct Type<DTL_F32> {
  static constexpr int kBytes = 4, kInPacket = 4, kPackets = kPer / 4;
  static constexpr uint32_t kMasked = 0xff800000u;
  typedef packet4 mem;
};
template <int DT>
struct Seg {  // a lane's logits of a segment: packets of 16 bytes, 64 lanes apart
  packet w[Type<DT>::kPackets];
};

// Where logit i of a lane lies in its segment.
template <int DT>
__device__ __forceinline__ int place(int i, int lane) {
  constexpr int n = Type<DT>::kInPacket;
  return i / n * (64 * n) + lane * n + i % n;
}

template <int DT>
__device__ __forceinline__ float value(const packet& p, int i) {
  const uint32_t w = p[DT == DTL_F32 ? i : i / 2];
  if constexpr (DT == DTL_F32) return __builtin_bit_cast(float, w);
  if constexpr (DT == DTL_BF16) return __builtin_bit_cast(float, i & 1 ? w & 0xffff0000u : w << 16);
  return (float)__builtin_bit_cast(_Float16, (uint16_t)(i & 1 ? w >> 16 : w));
}
template <int DT>
__device__ __forceinline__ float value(const Seg<DT>& s, int i) {
  return value<DT>(s.w[i / Type<DT>::kInPacket], i % Type<DT>::kInPacket);
}

template <int DT>
__device__ __forceinline__ float load_one(const char* row, int j) {
  if constexpr (DT == DTL_F32) return reinterpret_cast<const float*>(row)[j];
  const uint32_t h = reinterpret_cast<const uint16_t*>(row)[j];
  if constexpr (DT == DTL_BF16) return __builtin_bit_cast(float, h << 16);
  return (float)__builtin_bit_cast(_Float16, (uint16_t)h);
}
template <int DT>
__device__ __forceinline__ uint32_t bits_of(float v) {  // rounded to nearest, ties to even
  if constexpr (DT == DTL_F32) return __builtin_bit_cast(uint32_t, v);
  if constexpr (DT == DTL_BF16) return __builtin_bit_cast(uint16_t, (__bf16)v);
  return __builtin_bit_cast(uint16_t, (_Float16)v);
}
template <int DT>
__device__ __forceinline__ void store_one(char* row, int j, float v) {
  if constexpr (DT == DTL_F32)
    reinterpret_cast<float*>(row)[j] = v;
  else
    reinterpret_cast<uint16_t*>(row)[j] = (uint16_t)bits_of<DT>(v);
}

// The packet of logits j .. j + kInPacket, masked (-inf) past V.
template <int DT>
__device__ __forceinline__ packet load_packet(const char* row, int j, int V) {
  constexpr int n = Type<DT>::kInPacket;
  if (j + n <= V) return *reinterpret_cast<const typename Type<DT>::mem*>(row + (size_t)j * Type<DT>::kBytes);
  packet p;
#pragma unroll
  for (int q = 0; q < 4; q++) {
    uint32_t w = Type<DT>::kMasked;
    if constexpr (DT == DTL_F32) {
      if (j + q < V) w = reinterpret_cast<const uint32_t*>(row)[j + q];
    } else {
      const uint16_t* h = reinterpret_cast<const uint16_t*>(row);
      if (j + 2 * q < V) w = (w & 0xffff0000u) | h[j + 2 * q];
      if (j + 2 * q + 1 < V) w = (w & 0xffffu) | ((uint32_t)h[j + 2 * q + 1] << 16);
    }
    p[q] = w;
  }
  return p;
}

template <int DT>
__device__ __forceinline__ void load_seg(Seg<DT>& s, const char* row, int seg, int lane, int V) {
  constexpr int n = Type<DT>::kInPacket;
  const int at = seg * kScoreSeg + lane * n;
  if (seg * kScoreSeg + kScoreSeg <= V) {
#pragma unroll
    for (int q = 0; q < Type<DT>::kPackets; q++)
      s.w[q] = *reinterpret_cast<const typename Type<DT>::mem*>(row + (size_t)(at + q * 64 * n) * Type<DT>::kBytes);
  } else {
#pragma unroll
    for (int q = 0; q < Type<DT>::kPackets; q++) s.w[q] = load_packet<DT>(row, at + q * 64 * n, V);
  }
}

// Masks the lane's logits whose bit is set.
template <int DT>
__device__ __forceinline__ void mask_seg(Seg<DT>& s, uint32_t bits) {
#pragma unroll
  for (int q = 0; q < Type<DT>::kPackets; q++)
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

// ---- over the lanes of a wave ---------------------------------------------------

template <int CTRL, int ROWS>
__device__ __forceinline__ float dpp(float x, float idle) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(__builtin_bit_cast(int, idle), __builtin_bit_cast(int, x),
                                                               CTRL, ROWS, 0xf, false));
}
__device__ __forceinline__ float last_lane(float x) {
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), 63));
}
__device__ __forceinline__ float wave_sum(float x) {
  x += dpp<0x111, 0xf>(x, 0.0f);  // row_shr 1, 2, 4, 8, then lane 15 and 31 to the rows behind
  x += dpp<0x112, 0xf>(x, 0.0f);
  x += dpp<0x114, 0xf>(x, 0.0f);
  x += dpp<0x118, 0xf>(x, 0.0f);
  x += dpp<0x142, 0xa>(x, 0.0f);
  x += dpp<0x143, 0xc>(x, 0.0f);
  return last_lane(x);
}
__device__ __forceinline__ float wave_max(float x) {
  const float no = -__builtin_inff();
  x = fmaxf(x, dpp<0x111, 0xf>(x, no));
  x = fmaxf(x, dpp<0x112, 0xf>(x, no));
  x = fmaxf(x, dpp<0x114, 0xf>(x, no));
  x = fmaxf(x, dpp<0x118, 0xf>(x, no));
  x = fmaxf(x, dpp<0x142, 0xa>(x, no));
  x = fmaxf(x, dpp<0x143, 0xc>(x, no));
  return last_lane(x);
}
__device__ __forceinline__ double wave_sum(double x) {
#pragma unroll
  for (int d = 32; d; d >>= 1) x += __shfl_xor(x, d);
  return x;
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

template <int DT, bool ENT>
__device__ __forceinline__ Part seg_part(const Seg<DT>& z, float most, float c) {
  Part p{wave_max(most), 0.0f, 0.0f};
  float s[4] = {}, u[4] = {};
  const float m = p.m == -__builtin_inff() ? 0.0f : p.m;
#pragma unroll
  for (int i = 0; i < kPer; i++) {
    const float t = (value<DT>(z, i) - m) * c;
    const float e = __builtin_amdgcn_exp2f(t);
    s[i & 3] += e;
    if (ENT) u[i & 3] = __builtin_fmaf(e, fmaxf(t, kLowest), u[i & 3]);
  }
  p.s = wave_sum((s[0] + s[1]) + (s[2] + s[3]));
  if (ENT) p.u = wave_sum((u[0] + u[1]) + (u[2] + u[3]));
  return p;
}

// ---- a row, its segments' parts in LDS -------------------------------------------

struct RowStats {
  float m;      // the largest logit; -inf: every logit is masked
  double r, u;  // over the row, relative to m
  bool bad;     // a logit is NaN or +inf
};

// One wave joins the parts of a row.  The first segment that holds the maximum
// is read again for its sum without it.  `mask` (may be null): per segment and
// lane the logits that the parts left out.
template <int DT>
__device__ RowStats join_parts(const char* row, int V, int nseg, const Part* parts, const uint32_t* mask, float c,
                               int lane) {
  const float no = -__builtin_inff();
  const Part a = lane < nseg ? parts[lane] : Part{no, 0.0f, 0.0f};
  const Part b = lane + 64 < nseg ? parts[lane + 64] : Part{no, 0.0f, 0.0f};
  RowStats st;
  st.m = wave_max(fmaxf(a.m, b.m));
  const bool nan = !(a.s == a.s) || !(b.s == b.s);
  st.bad = __ballot(nan) != 0 || st.m == __builtin_inff();
  st.r = st.u = 0.0;
  if (st.bad || st.m == no) return st;
  const uint64_t in_a = __ballot(a.m == st.m), in_b = __ballot(b.m == st.m);
  const int first = in_a ? __builtin_ctzll(in_a) : 64 + __builtin_ctzll(in_b);

  Seg<DT> z;
  load_seg<DT>(z, row, first, lane, V);
  if (mask) mask_seg<DT>(z, mask[first * 64 + lane]);
  const float most = lane_max<DT>(z);
  const uint64_t have = __ballot(most == st.m);
  bool out = lane == __builtin_ctzll(have);  // this lane's first maximum stays out
  float s = 0.0f;
#pragma unroll
  for (int i = 0; i < kPer; i++) {
    const float v = value<DT>(z, i), e = __builtin_amdgcn_exp2f((v - st.m) * c);
    const bool skip = out && v == st.m;
    out = out && !skip;
    s += skip ? 0.0f : e;
  }
  double r = s, u = 0.0;
  const Part* two[2] = {&a, &b};
#pragma unroll
  for (int i = 0; i < 2; i++) {
    const Part& p = *two[i];
    if (p.m == no) continue;
    const float d = fmaxf((p.m - st.m) * c, -1000.0f);
    const double f = __builtin_amdgcn_exp2f(d);
    if (lane + 64 * i != first) r += f * p.s;
    u += f * ((double)p.u + (double)d * p.s);
  }
  st.r = wave_sum(r);
  st.u = wave_sum(u);
  return st;
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

struct TopLds {
  uint32_t counts[2][kRowWaves];
  uint32_t buckets, candidates, chosen;
  uint16_t ties[kScoreMaxSegs];
  uint16_t bucket[kScoreMaxTop + 64];
  uint64_t best[kScoreMaxTop];
};
// Candidates: every logit of K + 64 buckets at most.
constexpr size_t candidate_bytes(size_t top) { return (top + 64) * kPer * sizeof(uint64_t); }

// How many of the workgroup's flags are set, for step `step` of a loop: the two
// sets of counts let one barrier a step do.
__device__ __forceinline__ int group_count(TopLds& t, int step, int in_wave, int wave, int lane) {
  if (lane == 0) t.counts[step & 1][wave] = in_wave;
  __syncthreads();
  int n = 0;
#pragma unroll
  for (int w = 0; w < kRowWaves; w++) n += t.counts[step & 1][w];
  return n;
}

// The `top` largest logits of a row in order (value, then the lower index), by
// the whole workgroup, from keys[nseg * 64]: the order of the largest logit of
// each bucket, a lane's share of a segment.  Put the buckets in the order of
// their largest logits: the row's `top` largest lie in the first `top` buckets,
// since each of those holds one that is as large.  So:
//   1. tau, the value of bucket number `top` (bit by bit; 16 keys a thread);
//   2. the buckets above tau, and those equal to it up to the segment where
//      there are enough: the lowest indices among equals lie no further;
//   3. their logits from tau on, read again (32 a bucket);
//   4. these ranked by counting, each against each.
// All but 3 is in LDS and registers, whatever the logits hold: rows of equal
// logits take the same steps.  keys' memory is used again for the candidates.
template <int DT, typename Emit>
__device__ void select_top(const char* row, int V, int nseg, int top, uint64_t* memory, TopLds& t, Emit&& emit) {
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t* keys = reinterpret_cast<const uint32_t*>(memory);
  uint32_t key[kKeysPerThread];
#pragma unroll
  for (int i = 0; i < kKeysPerThread; i++) key[i] = i * kRowWaves + wave < nseg ? keys[i * kRowThreads + tid] : 0;

  uint32_t tau = 0;
  for (int bit = 31; bit >= 0; bit--) {
    const uint32_t trial = tau | 1u << bit;
    int in_wave = 0;
#pragma unroll
    for (int i = 0; i < kKeysPerThread; i++)
      if (i * kRowWaves < nseg) in_wave += __popcll(__ballot(key[i] >= trial));
    const int n = group_count(t, bit, in_wave, wave, lane);
    if (n >= top) tau = trial;
    if (n == top) break;
  }
  if (tau == 0) tau = 1;  // fewer buckets than `top` hold anything unmasked

  int above = 0;
#pragma unroll
  for (int i = 0; i < kKeysPerThread; i++)
    if (i * kRowWaves + wave < nseg) {
      above += __popcll(__ballot(key[i] > tau));
      const int same = __popcll(__ballot(key[i] == tau));
      if (lane == 0) t.ties[i * kRowWaves + wave] = same;
    }
  __syncthreads();  // the counts of the last step have been read
  if (lane == 0) t.counts[0][wave] = above;
  if (tid == 0) t.buckets = t.candidates = t.chosen = 0;
  __syncthreads();
  above = 0;
#pragma unroll
  for (int w = 0; w < kRowWaves; w++) above += t.counts[0][w];
  int last = 0;
  for (int have = above; last < nseg; last++) {
    have += t.ties[last];
    if (have >= top) break;
  }
#pragma unroll
  for (int i = 0; i < kKeysPerThread; i++) {
    const int seg = i * kRowWaves + wave;
    if (seg < nseg && (key[i] > tau || (key[i] == tau && seg <= last)))
      t.bucket[atomicAdd(&t.buckets, 1u)] = (uint16_t)(seg * 64 + lane);
  }
  __syncthreads();

  constexpr int np = Type<DT>::kPackets, in = Type<DT>::kInPacket;
  const int work = (int)t.buckets * np;
  for (int w = tid; w < work; w += kRowThreads) {
    const int b = t.bucket[w / np];
    const int j = (b >> 6) * kScoreSeg + (w % np) * (64 * in) + (b & 63) * in;
    const packet p = load_packet<DT>(row, j, V);
#pragma unroll
    for (int i = 0; i < in; i++) {
      const uint32_t k = order_of(value<DT>(p, i));
      if (k >= tau) memory[atomicAdd(&t.candidates, 1u)] = (uint64_t)k << 18 | (uint32_t)(kScoreMaxVocab - 1 - (j + i));
    }
  }
  __syncthreads();

  const uint64_t* list = memory;
  int n = t.candidates;
  if (n > kRowThreads) {  // many equal or neighbouring ones: the `top` best by their 50 bits first
    uint64_t floor = 0;
    for (int bit = 49; bit >= 0; bit--) {
      const uint64_t trial = floor | (uint64_t)1 << bit;
      int in_wave = 0;
      for (int i = tid - lane; i < n; i += kRowThreads) in_wave += __popcll(__ballot(i + lane < n && memory[i + lane] >= trial));
      const int got = group_count(t, bit, in_wave, wave, lane);
      if (got >= top) floor = trial;
      if (got == top) break;
    }
    for (int i = tid; i < n; i += kRowThreads)
      if (memory[i] >= floor) t.best[atomicAdd(&t.chosen, 1u)] = memory[i];
    __syncthreads();
    list = t.best;
    n = top;
  }
  if (tid < n) {
    const uint64_t mine = list[tid];
    int rank = 0;
    for (int i = 0; i < n; i++) rank += list[i] > mine;
    if (rank < top) emit(rank, kScoreMaxVocab - 1 - (int)(mine & (kScoreMaxVocab - 1)), of_order((uint32_t)(mine >> 18)));
  }
  if (tid < top && tid >= n) emit(tid, -1, -__builtin_inff());
}

// ---- reading a row ------------------------------------------------------------------

// Segments seg0 + wave, seg0 + wave + waves, ... below seg1: their parts, and
// with KEYS their buckets' largest logits.  The next segment's loads are in
// flight while one is reduced.
template <int DT, bool ENT, bool KEYS>
__device__ __forceinline__ void read_segs(const char* row, int V, int seg0, int seg1, int wave, int waves, int lane,
                                          float c, Part* parts, uint32_t* keys, const uint32_t* mask) {
  int seg = seg0 + wave;
  if (seg >= seg1) return;
  Seg<DT> z, next;
  load_seg<DT>(z, row, seg, lane, V);
  for (; seg < seg1; seg += waves) {
    if (seg + waves < seg1) load_seg<DT>(next, row, seg + waves, lane, V);
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

// Whole rows by one workgroup each, or for few rows one part of a row each
// (PARTS) and a second launch that joins them (JOIN).
enum Phase { WHOLE, PARTS, JOIN };

__device__ __forceinline__ long load_index(const void* p, int wide, size_t i) {
  return wide ? (long)reinterpret_cast<const int64_t*>(p)[i] : (long)reinterpret_cast<const int32_t*>(p)[i];
}

// ---- scores ---------------------------------------------------------------------------

struct ScoreK {
  const char* z;
  size_t row_bytes, rows;
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

template <int DT, bool TOP, int PHASE>
__global__ __launch_bounds__(kRowThreads) void k_scores(ScoreK a) {
  extern __shared__ uint64_t memory[];
  __shared__ Part lds_parts[PHASE == PARTS ? 1 : kScoreMaxSegs];
  __shared__ TopLds tl;
  __shared__ float row_m;
  __shared__ double row_log;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int waves = blockDim.x >> 6;
  const float no = -__builtin_inff();

  if constexpr (PHASE == PARTS) {
    for (size_t w = blockIdx.x; w < a.rows * a.groups; w += gridDim.x) {
      const size_t row = w / a.groups;
      const int g = (int)(w % a.groups), per = (a.nseg + a.groups - 1) / a.groups;
      const int seg1 = min(a.nseg, (g + 1) * per);
      read_segs<DT, true, TOP>(a.z + row * a.row_bytes, a.V, g * per, seg1, wave, waves, lane, a.c,
                               a.parts + row * a.nseg, TOP ? a.keys + row * a.nseg * 64 : nullptr, nullptr);
    }
    return;
  }

  uint32_t* keys = reinterpret_cast<uint32_t*>(memory);
  for (size_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const char* z = a.z + row * a.row_bytes;
    long y = -1;
    float zy = 0.0f;
    if (wave == 0 && a.tokens) {
      y = load_index(a.tokens, a.wide, row);
      if (y >= 0 && y < a.V) zy = load_one<DT>(z, (int)y);
    }
    if constexpr (PHASE == WHOLE) {
      read_segs<DT, true, TOP>(z, a.V, 0, a.nseg, wave, waves, lane, a.c, lds_parts, keys, nullptr);
    } else {
      for (int i = threadIdx.x; i < a.nseg; i += kRowThreads) lds_parts[i] = a.parts[row * a.nseg + i];
      if (TOP)
        for (int i = threadIdx.x; i < a.nseg * 64; i += kRowThreads) keys[i] = a.keys[row * a.nseg * 64 + i];
    }
    __syncthreads();
    if (wave == 0) {
      const RowStats st = join_parts<DT>(z, a.V, a.nseg, lds_parts, nullptr, a.c, lane);
      const double l = st.bad ? (double)__builtin_nanf("") : log1p(st.r);
      const float m = st.bad ? __builtin_nanf("") : st.m;
      if (lane == 0) {
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
      }
    }
    if constexpr (TOP) {
      int32_t* ids = a.top_ids + row * a.top;
      float* lps = a.top_log_probs + row * a.top;
      select_top<DT>(z, a.V, a.nseg, a.top, memory, tl, [&](int at, int id, float v) {
        const float m = row_m;
        const bool bad = !(m == m);
        ids[at] = bad ? -1 : id;
        lps[at] = bad ? m : id < 0 ? no : (float)(((double)v - m) * a.inv_t - row_log);
      });
    }
    __syncthreads();
  }
}

// dz = ( g (delta_y - p) - h p (log p + H) ) / T for the gradients g of the
// token's log probability and h of the entropy.  With p = e / (1 + r) that is
// e (A + B t) per logit, and at the token 1 - p = -expm1(log p).
struct ScoreGradK {
  const char* z;
  char* grad;
  size_t row_bytes, grad_bytes, rows;
  int V, nseg, chunks;
  const void* tokens;
  int wide;
  float c;
  double inv_t;
  const float *stats, *entropy, *g, *h;
};

// Segments a wave takes one after another; a workgroup has kGradWaves waves.
constexpr int kGradWaves = 4, kGradSegs = 2;

template <int DT, typename F>
__device__ __forceinline__ void write_seg(const Seg<DT>& z, char* out, int seg, int lane, int V, F&& f) {
  constexpr int in = Type<DT>::kInPacket;
  const bool whole = seg * kScoreSeg + kScoreSeg <= V;
#pragma unroll
  for (int q = 0; q < Type<DT>::kPackets; q++) {
    const int j = seg * kScoreSeg + (q * 64 + lane) * in;
    float v[in];
#pragma unroll
    for (int i = 0; i < in; i++) v[i] = f(value<DT>(z.w[q], i), j + i);
    packet p;
#pragma unroll
    for (int d = 0; d < 4; d++)
      p[d] = DT == DTL_F32 ? bits_of<DT>(v[d]) : bits_of<DT>(v[2 * d % in]) | bits_of<DT>(v[(2 * d + 1) % in]) << 16;
    if (whole || j + in <= V) {
      *reinterpret_cast<typename Type<DT>::mem*>(out + (size_t)j * Type<DT>::kBytes) = p;
    } else {
#pragma unroll
      for (int i = 0; i < in; i++)
        if (j + i < V) store_one<DT>(out, j + i, v[i]);
    }
  }
}

template <int DT, bool ENT>
__global__ __launch_bounds__(kGradWaves * 64) void k_scores_grad(ScoreGradK a) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const float no = -__builtin_inff();
  for (size_t w = blockIdx.x; w < a.rows * a.chunks; w += gridDim.x) {
    const size_t row = w / a.chunks;
    const int seg0 = (int)(w % a.chunks) * (kGradWaves * kGradSegs) + wave;
    const char* z = a.z + row * a.row_bytes;
    char* out = a.grad + row * a.grad_bytes;
    const long y = a.tokens ? load_index(a.tokens, a.wide, row) : -1;
    const double g = a.g && y >= 0 ? a.g[row] : 0.0f, h = ENT && a.h ? a.h[row] : 0.0f;
    const float m = a.stats[2 * row];
    const double r = a.stats[2 * row + 1], p0 = 1.0 / (1.0 + r);
    // padding, and rows whose mask leaves nothing: zeros, whatever they hold
    const bool zero = (g == 0.0 && h == 0.0) || m == no;
    const bool bad = y >= a.V, here = y >= 0 && !bad && !zero && ((int)(y >> 11) - seg0) % kGradWaves == 0;
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
#pragma unroll
    for (int i = 0; i < kGradSegs; i++) {
      const int seg = seg0 + i * kGradWaves;
      if (seg >= a.nseg) break;
      Seg<DT> s;
      if (zero) {
        write_seg<DT>(s, out, seg, lane, a.V, [](float, int) { return 0.0f; });
        continue;
      }
      load_seg<DT>(s, z, seg, lane, a.V);
      auto value_of = [&](float v) {
        const float t = (v - m) * a.c, e = __builtin_amdgcn_exp2f(t);
        return e * (ENT ? __builtin_fmaf(B, fmaxf(t, kLowest), A) : A);
      };
      if (y >> 11 == seg)
        write_seg<DT>(s, out, seg, lane, a.V, [&](float v, int j) { return j == (int)y ? at_y : value_of(v); });
      else
        write_seg<DT>(s, out, seg, lane, a.V, [&](float v, int) { return value_of(v); });
    }
  }
}
static_assert(kScoreSeg == 1 << 11, "the token's segment");

// ---- distillation ------------------------------------------------------------------------

// A row's teacher: up to 256 slots (id, log probability v).
//   renormalised: p_k = e^(v_k) / sum;  rest: p_k = e^(v_k), and what is left of
//   one is the teacher's mass outside the list.
// loss = w T^2 (sum p_k (log p_k - log q_k) + rest (log rest - log q_rest)); the
// last term only where a logit outside the list is unmasked.
// dz_j = w T (e_j share - p_j) with share = (sum p + rest) / sum of e, and for j
// outside the list e_j (share - rest / sum of e outside) instead.
// The slots' terms are formed in 64 bits: the loss is a small difference of
// large ones.
struct DistillK {
  const char* z;
  char* grad;
  size_t row_bytes, grad_bytes, rows;
  int V, nseg, groups;
  const void* ids;
  int wide, k;
  const float* teacher;
  const float* weights;
  float c, T;
  double inv_t;
  float* loss;
  float* stats;  // [rows][kDistillStats]: RowGrad
  Part* parts;
};

struct Slots {
  int32_t id[kDistillMaxK];  // -1: empty
  float v[kDistillMaxK];
};

// Loads the slots; the result is, for every thread, whether the row has a slot
// in use (1) and whether one is broken (2): an id past the vocabulary, a log
// probability that is NaN or +inf.
__device__ __forceinline__ int load_slots(Slots& s, const DistillK& a, size_t row) {
  int bits = 0;
  for (int i = threadIdx.x; i < kDistillMaxK; i += blockDim.x) {
    int id = -1;
    float v = -__builtin_inff();
    if (i < a.k) {
      const long j = load_index(a.ids, a.wide, row * a.k + i);
      v = a.teacher[row * a.k + i];
      if (j >= 0 && v != -__builtin_inff()) {
        bits |= 1;
        if (j >= a.V || !(v < __builtin_inff()))
          bits |= 2;
        else
          id = (int)j;
      }
    }
    s.id[i] = id;
    s.v[i] = v;
  }
  const int used = __syncthreads_or(bits & 1), broken = __syncthreads_or(bits & 2);
  return (used ? 1 : 0) | (broken ? 2 : 0);
}

// Which lane's which logit of a segment an id is: the bit of read_segs' mask.
template <int DT>
__device__ __forceinline__ void mask_bit(int id, int& word, uint32_t& bit) {
  constexpr int in = Type<DT>::kInPacket;
  const int seg = id / kScoreSeg, at = id % kScoreSeg;
  const int q = at / (64 * in), lane = at / in % 64;
  word = seg * 64 + lane;
  bit = 1u << (q * in + at % in);
}
template <int DT>
__device__ __forceinline__ void build_mask(uint32_t* mask, const Slots& s, int nseg) {
  for (int i = threadIdx.x; i < nseg * 64; i += blockDim.x) mask[i] = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < kDistillMaxK; i += blockDim.x)
    if (s.id[i] >= 0) {
      int word;
      uint32_t bit;
      mask_bit<DT>(s.id[i], word, bit);
      atomicOr(&mask[word], bit);
    }
  __syncthreads();
}

// What a row's gradient needs besides its logits: m, share, rest / sum outside,
// and the log of the teacher's sum as a float and what it leaves.
struct RowGrad {
  float m, share, outside, log_hi, log_lo;
};
static_assert(sizeof(RowGrad) == kDistillStats * sizeof(float), "stats");

// One wave: the row's loss (times T^2) and what its gradient needs, from the
// parts and the slots.
template <int DT, bool REST>
__device__ RowGrad join_distill(const DistillK& a, const char* z, const Part* parts, const uint32_t* mask,
                                const Slots& s, int state, int lane, float* loss) {
  const float no = -__builtin_inff(), nan = __builtin_nanf("");
  constexpr int n = kDistillMaxK / 64;
  RowGrad g{};
  *loss = 0.0f;
  if (state == 0) return g;
  RowStats st = join_parts<DT>(z, a.V, a.nseg, parts, REST ? mask : nullptr, a.c, lane);
  float zk[n];
  bool first[n];
  float most = no, most_v = no;
#pragma unroll
  for (int i = 0; i < n; i++) {
    const int k = lane + 64 * i, id = s.id[k];
    zk[i] = id >= 0 ? load_one<DT>(z, id) : no;
    if (id >= 0) most_v = fmaxf(most_v, s.v[k]);
    if (id >= 0) most = fmaxf(most, zk[i]);
    first[i] = id >= 0;
    if (REST && id >= 0)
      for (int j = 0; j < k; j++) first[i] = first[i] && s.id[j] != id;
    if (REST && id >= 0 && (!(zk[i] == zk[i]) || zk[i] == __builtin_inff())) st.bad = true;
  }
  st.bad = __ballot(st.bad) != 0;
  if (st.bad || (state & 2)) {
    *loss = nan;
    return RowGrad{nan, nan, nan, nan, nan};
  }
  // total of e relative to m, the row's largest logit; outside: without the list
  double total, left = 0.0;
  float m = st.m;
  if (REST) {
    most = wave_max(most);
    m = fmaxf(st.m, most);
    if (st.m != no) left = exp(((double)st.m - m) * a.inv_t) * (1.0 + st.r);
    double in = 0.0;
#pragma unroll
    for (int i = 0; i < n; i++)
      if (first[i] && zk[i] != no) in += exp(((double)zk[i] - m) * a.inv_t);
    total = left + wave_sum(in);
  } else {
    total = 1.0 + st.r;
  }
  if (m == no) {  // every logit masked: no q to compare with, nothing to move
    *loss = __builtin_inff();
    return RowGrad{no, 0.0f, 0.0f, 0.0f, 0.0f};
  }
  most_v = wave_max(most_v);
  double log_sum = 0.0;
  if (!REST) {
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < n; i++)
      if (s.id[lane + 64 * i] >= 0) sum += exp((double)s.v[lane + 64 * i] - most_v);
    log_sum = most_v + log(wave_sum(sum));
  }
  const double log_total = REST ? log(total) : log1p(st.r);
  double mass = 0.0, term = 0.0;
#pragma unroll
  for (int i = 0; i < n; i++)
    if (s.id[lane + 64 * i] >= 0) {
      const double lp = s.v[lane + 64 * i] - log_sum, p = exp(lp);
      mass += p;
      if (p > 0.0) term += p * (lp - (((double)zk[i] - m) * a.inv_t - log_total));
    }
  mass = wave_sum(mass);
  term = wave_sum(term);
  double rest = 0.0;
  if (REST && left > 0.0) {
    rest = fmax(0.0, 1.0 - mass);
    if (rest > 0.0) term += rest * (log(rest) - (log(left) - log_total));
  }
  *loss = (float)((double)a.T * a.T * term);
  g.m = m;
  g.share = (float)((mass + rest) / total);
  g.outside = rest > 0.0 ? (float)(rest / left) : 0.0f;
  g.log_hi = (float)log_sum;
  g.log_lo = (float)(log_sum - g.log_hi);
  return g;
}

// Gradient of segments seg0 + wave, seg0 + wave + waves, ... below seg1, for
// every j as if outside the list.
template <int DT>
__device__ __forceinline__ void grad_segs(const DistillK& a, const char* z, char* out, const RowGrad& g, float scale,
                                          int seg0, int seg1, int wave, int waves, int lane) {
  const bool zero = scale == 0.0f || g.m == -__builtin_inff();
  const float A = scale * (g.share - g.outside);
  for (int seg = seg0 + wave; seg < seg1; seg += waves) {
    Seg<DT> s;
    if (zero) {
      write_seg<DT>(s, out, seg, lane, a.V, [](float, int) { return 0.0f; });
      continue;
    }
    load_seg<DT>(s, z, seg, lane, a.V);
    write_seg<DT>(s, out, seg, lane, a.V,
                  [&](float v, int) { return __builtin_amdgcn_exp2f((v - g.m) * a.c) * A; });
  }
}

// The gradient at the list's ids from lo to hi, by one thread for each distinct
// id: `zk` is its logit, read before the gradient was written (grad may be z).
template <int DT>
__device__ __forceinline__ void grad_slot(const DistillK& a, char* out, const Slots& s, const RowGrad& g, float scale,
                                          int k, float zk) {
  const int id = s.id[k];
  double p = 0.0;
  for (int j = 0; j < a.k; j++)
    if (s.id[j] == id) {
      if (j < k) return;  // an earlier slot of the same id writes it
      p += exp(((double)s.v[j] - g.log_hi) - g.log_lo);
    }
  const float e = __builtin_amdgcn_exp2f((zk - g.m) * a.c);
  store_one<DT>(out, id, (float)((double)scale * ((double)e * g.share - p)));
}

template <int DT, bool REST, int PHASE, bool STEP>
__global__ __launch_bounds__(kRowThreads) void k_distill(DistillK a) {
  extern __shared__ uint64_t memory[];
  uint32_t* mask = reinterpret_cast<uint32_t*>(memory);  // REST, WHOLE and PARTS: [nseg * 64]
  __shared__ Part lds_parts[PHASE == PARTS ? 1 : kScoreMaxSegs];
  __shared__ Slots s;
  __shared__ RowGrad row_grad;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int waves = blockDim.x >> 6;

  if constexpr (PHASE == PARTS) {
    for (size_t w = blockIdx.x; w < a.rows * a.groups; w += gridDim.x) {
      const size_t row = w / a.groups;
      const int g = (int)(w % a.groups), per = (a.nseg + a.groups - 1) / a.groups;
      if (load_slots(s, a, row) == 0) continue;
      if (REST) build_mask<DT>(mask, s, a.nseg);
      read_segs<DT, false, false>(a.z + row * a.row_bytes, a.V, g * per, min(a.nseg, (g + 1) * per), wave, waves, lane,
                                  a.c, a.parts + row * a.nseg, nullptr, REST ? mask : nullptr);
      __syncthreads();
    }
    return;
  }

  for (size_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const char* z = a.z + row * a.row_bytes;
    const float w = a.weights ? a.weights[row] : 1.0f;
    int state = load_slots(s, a, row);
    if (w == 0.0f) state = 0;  // a row that does not count is not read
    if (state) {
      if (REST) build_mask<DT>(mask, s, a.nseg);
      if constexpr (PHASE == WHOLE) {
        read_segs<DT, false, false>(z, a.V, 0, a.nseg, wave, waves, lane, a.c, lds_parts, nullptr, REST ? mask : nullptr);
      } else {
        for (int i = threadIdx.x; i < a.nseg; i += kRowThreads) lds_parts[i] = a.parts[row * a.nseg + i];
      }
    }
    __syncthreads();
    if (wave == 0) {
      float loss;
      const RowGrad g = join_distill<DT, REST>(a, z, lds_parts, mask, s, state, lane, &loss);
      if (lane == 0) {
        row_grad = g;
        if (a.loss) a.loss[row] = state ? w * loss : 0.0f;
        if (a.stats) reinterpret_cast<RowGrad*>(a.stats)[row] = g;
      }
    }
    __syncthreads();
    if constexpr (STEP) {
      const RowGrad g = row_grad;
      const float scale = state ? w * a.T : 0.0f;
      char* out = a.grad + row * a.grad_bytes;
      const int k = threadIdx.x;
      const bool patch = k < a.k && s.id[k] >= 0 && scale != 0.0f && g.m != -__builtin_inff();
      const float zk = patch ? load_one<DT>(z, s.id[k]) : 0.0f;
      __syncthreads();
      grad_segs<DT>(a, z, out, g, scale, 0, a.nseg, wave, waves, lane);
      __syncthreads();
      if (patch) grad_slot<DT>(a, out, s, g, scale, k, zk);
      __syncthreads();
    }
  }
}

// The gradient alone, from the stats of the forward: workgroups of one chunk of
// a row each.
constexpr int kDistillChunk = 16;  // segments

template <int DT>
__global__ __launch_bounds__(kGradWaves * 64) void k_distill_grad(DistillK a) {
  __shared__ Slots s;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  for (size_t w = blockIdx.x; w < a.rows * a.groups; w += gridDim.x) {
    const size_t row = w / a.groups;
    const int seg0 = (int)(w % a.groups) * kDistillChunk, seg1 = min(a.nseg, seg0 + kDistillChunk);
    const char* z = a.z + row * a.row_bytes;
    char* out = a.grad + row * a.grad_bytes;
    const float weight = a.weights ? a.weights[row] : 1.0f;
    const int state = load_slots(s, a, row);
    const RowGrad g = reinterpret_cast<const RowGrad*>(a.stats)[row];
    const float scale = state ? weight * a.T : 0.0f;
    const int k = threadIdx.x, id = k < a.k ? s.id[k] : -1;
    const bool patch = id >= seg0 * kScoreSeg && id < seg1 * kScoreSeg && scale != 0.0f && g.m != -__builtin_inff();
    const float zk = patch ? load_one<DT>(z, id) : 0.0f;
    __syncthreads();
    grad_segs<DT>(a, z, out, g, scale, seg0, seg1, wave, kGradWaves, lane);
    __syncthreads();
    if (patch) grad_slot<DT>(a, out, s, g, scale, k, zk);
    __syncthreads();
  }
}
static_assert(kGradWaves * 64 >= kDistillMaxK && kRowThreads >= kDistillMaxK, "a thread a slot");

// ---- launches ---------------------------------------------------------------------------

// Rows from which on a row is one workgroup's: fewer would leave compute units
// idle, and go to several workgroups each with a second launch to join them.
constexpr size_t kWholeRows = 256;
constexpr int kPartThreads = 256;

int segments(size_t vocab) { return (int)((vocab + kScoreSeg - 1) / kScoreSeg); }

// Workgroups of four waves for a row in the split form: as many as its segments
// keep busy, until the chip has enough.
int part_groups(size_t rows, int nseg) {
  const size_t most = (nseg + kPartThreads / 64 - 1) / (kPartThreads / 64);
  const size_t enough = (2048 + rows - 1) / rows;
  return (int)(most < enough ? most : enough);
}

unsigned grid_of(size_t n) { return (unsigned)(n < (1u << 20) ? n : (1u << 20)); }

size_t round256(size_t n) { return (n + 255) & ~(size_t)255; }

template <typename F>
void by_type(int dtype, F&& f) {
  if (dtype == DTL_F32)
    f(std::integral_constant<int, DTL_F32>());
  else if (dtype == DTL_BF16)
    f(std::integral_constant<int, DTL_BF16>());
  else
    f(std::integral_constant<int, DTL_F16>());
}
size_t type_bytes(int dtype) { return dtype == DTL_F32 ? 4 : 2; }

}  // namespace

size_t score_scratch_bytes(size_t rows, size_t vocab, size_t top) {
  if (rows >= kWholeRows) return 0;
  const size_t nseg = segments(vocab);
  return round256(rows * nseg * sizeof(Part)) + (top ? rows * nseg * 64 * 4 : 0);
}

void launch_token_scores(const ScoreArgs& a, hipStream_t s) {
  if (a.rows == 0) return;
  ScoreK k{};
  k.z = static_cast<const char*>(a.z);
  k.row_bytes = a.stride * type_bytes(a.dtype);
  k.rows = a.rows;
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
    if (lds < (size_t)k.nseg * 256) lds = (size_t)k.nseg * 256;
  }
  by_type(a.dtype, [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    if (a.rows >= kWholeRows) {
      launch_kernel(a.top ? k_scores<DT, true, WHOLE> : k_scores<DT, false, WHOLE>, dim3(grid_of(a.rows)),
                    dim3(kRowThreads), lds, s, k);
      return;
    }
    k.groups = part_groups(a.rows, k.nseg);
    k.parts = static_cast<Part*>(a.scratch);
    k.keys = reinterpret_cast<uint32_t*>(static_cast<char*>(a.scratch) + round256(a.rows * k.nseg * sizeof(Part)));
    launch_kernel(a.top ? k_scores<DT, true, PARTS> : k_scores<DT, false, PARTS>, dim3(grid_of(a.rows * k.groups)),
                  dim3(kPartThreads), 0, s, k);
    launch_kernel(a.top ? k_scores<DT, true, JOIN> : k_scores<DT, false, JOIN>, dim3(grid_of(a.rows)),
                  dim3(kRowThreads), lds, s, k);
  });
}

void launch_token_scores_grad(const ScoreGradArgs& a, hipStream_t s) {
  if (a.rows == 0) return;
  ScoreGradK k{};
  k.z = static_cast<const char*>(a.z);
  k.grad = static_cast<char*>(a.grad);
  k.row_bytes = a.stride * type_bytes(a.dtype);
  k.grad_bytes = a.grad_stride * type_bytes(a.dtype);
  k.rows = a.rows;
  k.V = a.vocab;
  k.nseg = segments(a.vocab);
  k.chunks = (k.nseg + kGradWaves * kGradSegs - 1) / (kGradWaves * kGradSegs);
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
    launch_kernel(a.g_entropy ? k_scores_grad<DT, true> : k_scores_grad<DT, false>,
                  dim3(grid_of(a.rows * k.chunks)), dim3(kGradWaves * 64), 0, s, k);
  });
}

namespace {
DistillK distill_kernel_args(const DistillArgs& a) {
  DistillK k{};
  k.z = static_cast<const char*>(a.z);
  k.grad = static_cast<char*>(a.grad);
  k.row_bytes = a.stride * type_bytes(a.dtype);
  k.grad_bytes = a.grad_stride * type_bytes(a.dtype);
  k.rows = a.rows;
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
  return k;
}
}  // namespace

// Parts, and for a step of few rows the stats between its launches.
size_t distill_scratch_bytes(size_t rows, size_t vocab, bool step) {
  if (rows >= kWholeRows) return 0;
  return round256(rows * segments(vocab) * sizeof(Part)) + (step ? rows * sizeof(RowGrad) : 0);
}

void launch_distill_grad(const DistillArgs& a, hipStream_t s) {
  if (a.rows == 0) return;
  DistillK k = distill_kernel_args(a);
  k.groups = (k.nseg + kDistillChunk - 1) / kDistillChunk;
  by_type(a.dtype, [&](auto dt) {
    launch_kernel(k_distill_grad<decltype(dt)::value>, dim3(grid_of(a.rows * k.groups)), dim3(kGradWaves * 64), 0, s, k);
  });
}

void launch_distill(const DistillArgs& a, hipStream_t s) {
  if (a.rows == 0) return;
  DistillK k = distill_kernel_args(a);
  const size_t lds = a.rest ? (size_t)k.nseg * 256 : 0;
  by_type(a.dtype, [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    if (a.rows >= kWholeRows) {
      if (a.grad)
        launch_kernel(a.rest ? k_distill<DT, true, WHOLE, true> : k_distill<DT, false, WHOLE, true>,
                      dim3(grid_of(a.rows)), dim3(kRowThreads), lds, s, k);
      else
        launch_kernel(a.rest ? k_distill<DT, true, WHOLE, false> : k_distill<DT, false, WHOLE, false>,
                      dim3(grid_of(a.rows)), dim3(kRowThreads), lds, s, k);
      return;
    }
    k.groups = part_groups(a.rows, k.nseg);
    k.parts = static_cast<Part*>(a.scratch);
    if (a.grad)
      k.stats = reinterpret_cast<float*>(static_cast<char*>(a.scratch) + round256(a.rows * k.nseg * sizeof(Part)));
    launch_kernel(a.rest ? k_distill<DT, true, PARTS, false> : k_distill<DT, false, PARTS, false>,
                  dim3(grid_of(a.rows * k.groups)), dim3(kPartThreads), lds, s, k);
    launch_kernel(a.rest ? k_distill<DT, true, JOIN, false> : k_distill<DT, false, JOIN, false>, dim3(grid_of(a.rows)),
                  dim3(kRowThreads), lds, s, k);
  });
  if (a.grad && a.rows < kWholeRows) {
    DistillArgs b = a;
    b.stats = k.stats;
    launch_distill_grad(b, s);
  }
}

}  // namespace dtl

// ---- C entry points ------------------------------------------------------------------------

using namespace dtl;

namespace {

int launch_status() {
  switch (hipGetLastError()) {
    case hipSuccess: return DTL_OK;
    case hipErrorOutOfMemory: return DTL_ERR_OUT_OF_MEMORY;
    case hipErrorNoDevice:
    case hipErrorInvalidDevice: return DTL_ERR_NO_DEVICE;
    default: return DTL_ERR_DEVICE;
  }
}

constexpr size_t kMostRows = 1u << 24;

int check_logits(const dtl_logits* z) {
  if (!z) return DTL_ERR_INVALID_ARGUMENT;
  if (z->dtype != DTL_F32 && z->dtype != DTL_BF16 && z->dtype != DTL_F16) return DTL_ERR_INVALID_ARGUMENT;
  if (z->vocab == 0) return DTL_ERR_CDF_EMPTY;
  if (z->vocab > (size_t)kScoreMaxVocab) return DTL_ERR_CDF_TOO_MANY_SYMBOLS;
  if (z->rows > kMostRows || (z->rows > 1 && z->stride < z->vocab) || z->stride > (size_t)1 << 40) return DTL_ERR_SHAPE;
  if (z->rows == 0) return DTL_OK;
  if (!z->data || reinterpret_cast<uintptr_t>(z->data) % type_bytes(z->dtype)) return DTL_ERR_INVALID_ARGUMENT;
  return DTL_OK;
}
bool index_bytes_ok(int n) { return n == 4 || n == 8; }
bool temperature_ok(float t) { return t >= kScoreMinTemperature && t <= kScoreMaxTemperature; }
int check_grad(const dtl_logits* z, const void* grad, size_t stride) {
  if (z->rows > 1 && (stride < z->vocab || stride > (size_t)1 << 40)) return DTL_ERR_SHAPE;
  if (z->rows && (!grad || reinterpret_cast<uintptr_t>(grad) % type_bytes(z->dtype))) return DTL_ERR_INVALID_ARGUMENT;
  return DTL_OK;
}

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
