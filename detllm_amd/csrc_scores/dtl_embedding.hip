// Embedding lookup with scaling, and the table's gradient from positions sorted by
// token.
//
//   out[i] = s W[t_i];   dW[v] = s sum over t_i = v of g_i
//
// The gradient is bound by memory: the rows g are read once, the table is written
// once, zeros for nearly all of it.  Adding rows with atomics would write in an order
// of its own; here the positions are sorted by token instead (a stable radix sort of
// two 9-bit digits, so that a token's positions keep their order), and threads sum
// along fixed stretches of the sorted list.  A token's rows that cross a stretch's
// end are left as partial sums, which a last launch joins.  The zeros are written
// beside the sort, whose few workgroups wait on each other anyway.
#include "dtl_scores.h"

#include "dtl_rows.h"

namespace dtl {
namespace {

constexpr int kThreads = 256;
constexpr int kSortThreads = 1024, kSortWaves = kSortThreads / 64;
constexpr int kDigitBits = 9, kDigits = 1 << kDigitBits;
constexpr int kRounds = 8;    // most tokens a thread of the sort has
constexpr int kTiles = 128;   // most workgroups of the sort
constexpr int kPlaceBits = 13;
constexpr int kFew = 256;     // tokens that are ranked by counting
constexpr int kAlone = 4096;  // tokens that one workgroup sorts in LDS
constexpr size_t kBusy = 1 << 20;                  // threads that keep the chip busy
constexpr int kFillBytes = kSortThreads * 16 * 4;  // zeros a workgroup writes
static_assert(kScoreMaxVocab == 1 << (2 * kDigitBits), "two digits hold a token");
static_assert((size_t)kTiles * kRounds * kSortThreads == kEmbedMaxTokens, "the sort's workgroups hold every token");
static_assert(kAlone <= 1 << kPlaceBits && 2 * kDigitBits + kPlaceBits <= 32, "a token and its place fit a word");

// ---- lookup -----------------------------------------------------------------------

struct LookupK {
  const char* table;
  char* out;
  const void* tokens;
  size_t row0, n, table_bytes, out_bytes;
  int V, D, packets, wide;
  float scale;
  bool past;  // written past the caches
};

// Where a row's packet begins: the last one ends with the row, over a part of its
// neighbour, which has the same values there.  Rows shorter than a packet begin at 0.
template <int DT>
__device__ __forceinline__ int packet_begin(int col, int D) {
  constexpr int n = Type<DT>::kInPacket;
  return min(col * n, max(D - n, 0));
}

// A thread a packet of an output row.
template <int DT>
__global__ __launch_bounds__(kThreads) void k_embedding(LookupK a) {
  constexpr int n = Type<DT>::kInPacket;
  const uint32_t at = blockIdx.x * kThreads + threadIdx.x, r = at / (uint32_t)a.packets;
  const int j = packet_begin<DT>((int)(at - r * (uint32_t)a.packets), a.D);
  const size_t i = a.row0 + r;
  if (i >= a.n) return;
  const long t = load_index(a.tokens, a.wide, i);
  char* out = a.out + i * a.out_bytes;
  packet p{0, 0, 0, 0};
  float v[n];
  const bool real = t >= 0 && t < a.V;
  if (real) p = load_packet_at_once<DT>(a.table + (size_t)t * a.table_bytes, j, a.D);
  const float nan = __builtin_nanf("");
#pragma unroll
  for (int q = 0; q < n; q++) v[q] = t >= a.V ? nan : real ? value<DT>(p, q) * a.scale : 0.0f;
  if (j + n <= a.D) {
    packet w = p;
    if (t >= a.V || a.scale != 1.0f) {
#pragma unroll
      for (int q = 0; q < 4; q++)
        w[q] = DT == DTL_F32 ? bits_of<DT>(v[q % n]) : bits_of<DT>(v[2 * q % n]) | bits_of<DT>(v[(2 * q + 1) % n]) << 16;
    }
    store_packet<DT>(out + (size_t)j * Type<DT>::kBytes, w, a.past);
  } else {
#pragma unroll
    for (int q = 0; q < n; q++)
      if (j + q < a.D) store_one<DT>(out, j + q, v[q]);
  }
}

// ---- the sort ------------------------------------------------------------------------

struct SortK {
  const void* tokens;
  int wide, V;
  uint32_t n;       // tokens, those that are none among them
  uint32_t tile;    // a workgroup's
  int tiles;        // workgroups that sort; those behind them write zeros
  uint32_t* count;  // real tokens
  uint32_t* hist;   // [tiles][kDigits]
  uint32_t *key0, *place0, *key1, *place1;  // after the first and the second digit
  // zeros: rows of `fill_bytes`, of which this launch's workgroups write pieces from `piece0` on
  char* fill;
  size_t fill_rows, fill_bytes, fill_stride, piece0, pieces;
  bool past;
};

// 16 bytes a thread and step; a row's last bytes are at least an element's.
__device__ __forceinline__ void fill_piece(const SortK& a, size_t piece) {
  if (piece >= a.pieces) return;
  const size_t per_row = (a.fill_bytes + 15) / 16;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    size_t at = piece * (kFillBytes / 16) + i * kSortThreads + threadIdx.x, row = 0;
    if (a.fill_rows > 1) {
      row = at / per_row;
      at -= row * per_row;
    }
    if (row >= a.fill_rows || at >= per_row) continue;
    char* p = a.fill + row * a.fill_stride + at * 16;
    const size_t left = a.fill_bytes - at * 16;
    if (left >= 16)
      store_packet<DTL_BF16>(p, packet{0, 0, 0, 0}, a.past);
    else
      for (size_t b = 0; b < left; b += 2) *reinterpret_cast<uint16_t*>(p + b) = 0;
  }
}

struct RankLds {
  uint32_t count[kSortWaves][kDigits];
  uint32_t wave_sum[kDigits / 64];
};

// The lanes of this wave with the same digit, `on` among them.
__device__ __forceinline__ uint64_t same_digit(uint32_t digit, bool on) {
  uint64_t m = __ballot(on);
#pragma unroll
  for (int b = 0; b < kDigitBits; b++) {
    const uint64_t set = __ballot(digit >> b & 1);
    m &= digit >> b & 1 ? set : ~set;
  }
  return m;
}

// How many of the wave's earlier items have this one's digit; counts it.
__device__ __forceinline__ uint32_t rank_in_wave(RankLds& s, int wave, int lane, uint32_t digit, bool on) {
  const uint64_t m = same_digit(digit, on);
  const int first = m ? __builtin_ctzll(m) : 0;
  uint32_t before = 0;
  if (on && lane == first) before = atomicAdd(&s.count[wave][digit], (uint32_t)__builtin_popcountll(m));
  before = (uint32_t)__shfl((int)before, first);
  return before + (uint32_t)__builtin_popcountll(m & ((1ull << lane) - 1));
}

// For thread d < kDigits: the sum of `mine` over the digits before d.  All threads call it.
__device__ __forceinline__ uint32_t scan_digits(RankLds& s, uint32_t mine, uint32_t* total) {
  const int tid = threadIdx.x, wave = tid >> 6;
  const uint32_t up_to = wave_scan(tid < kDigits ? mine : 0);
  if (tid < kDigits && (tid & 63) == 63) s.wave_sum[wave] = up_to;
  __syncthreads();
  uint32_t before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kDigits / 64; w++) {
    if (w < wave) before += s.wave_sum[w];
    all += s.wave_sum[w];
  }
  *total = all;
  return before + up_to - mine;
}

// After the waves' counts: count[w][d] becomes the place of wave w's first item of
// digit d, the digits in order from `base` (a thread a digit) on.
__device__ __forceinline__ void place_waves(RankLds& s, uint32_t base) {
  const int d = threadIdx.x;
  if (d < kDigits) {
#pragma unroll
    for (int w = 0; w < kSortWaves; w++) {
      const uint32_t c = s.count[w][d];
      s.count[w][d] = base;
      base += c;
    }
  }
  __syncthreads();
}

__device__ __forceinline__ void clear_counts(RankLds& s) {
  for (int i = threadIdx.x; i < kSortWaves * kDigits; i += kSortThreads) (&s.count[0][0])[i] = 0;
  __syncthreads();
}
__device__ __forceinline__ uint32_t wave_total(const RankLds& s) {
  uint32_t sum = 0;
  if (threadIdx.x < kDigits)
    for (int w = 0; w < kSortWaves; w++) sum += s.count[w][threadIdx.x];
  return sum;
}

// Up to kAlone tokens by one workgroup, both digits in LDS; the others write zeros.
__global__ __launch_bounds__(kSortThreads) void k_sort_alone(SortK a) {
  constexpr int kTurns = kAlone / kSortThreads;
  __shared__ RankLds s;
  __shared__ uint32_t item[kAlone];
  if (blockIdx.x > 0) return fill_piece(a, a.piece0 + blockIdx.x - 1);
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const uint32_t per_wave = 64 * ((a.n + kSortThreads - 1) / kSortThreads);
  uint32_t mine[kTurns], rank[kTurns], all = a.n;
  bool real[kTurns];
#pragma unroll
  for (int r = 0; r < kTurns; r++) {
    const uint32_t at = wave * per_wave + r * 64 + lane;
    const bool in = (uint32_t)r * 64 < per_wave && at < a.n;
    const long t = in ? load_index(a.tokens, a.wide, at) : -1;
    real[r] = t >= 0 && t < a.V;
    mine[r] = (uint32_t)t << kPlaceBits | at;
  }
#pragma unroll
  for (int pass = 0; pass < 2; pass++) {
    clear_counts(s);
#pragma unroll
    for (int r = 0; r < kTurns; r++) {
      rank[r] = ~0u;
      if ((uint32_t)r * 64 >= per_wave) continue;
      if (pass == 1) {
        const uint32_t at = wave * per_wave + r * 64 + lane;
        real[r] = at < all;
        if (real[r]) mine[r] = item[at];
      }
      const uint32_t k = rank_in_wave(s, wave, lane, mine[r] >> (kPlaceBits + pass * kDigitBits) & (kDigits - 1), real[r]);
      if (real[r]) rank[r] = k;
    }
    __syncthreads();
    uint32_t total;
    const uint32_t base = scan_digits(s, wave_total(s), &total);
    place_waves(s, base);
#pragma unroll
    for (int r = 0; r < kTurns; r++) {
      if (rank[r] == ~0u) continue;
      const uint32_t at = s.count[wave][mine[r] >> (kPlaceBits + pass * kDigitBits) & (kDigits - 1)] + rank[r];
      if (pass == 0) {
        item[at] = mine[r];
      } else {
        a.key1[at] = mine[r] >> kPlaceBits;
        a.place1[at] = mine[r] & ((1u << kPlaceBits) - 1);
      }
    }
    all = total;
    __syncthreads();
  }
  if (tid == 0) *a.count = all;
}

// Up to kFew: a token's place is how many are smaller, or as large and before it.
__global__ __launch_bounds__(kSortThreads) void k_sort_few(SortK a) {
  __shared__ __attribute__((aligned(16))) uint32_t item[kFew];
  __shared__ uint32_t all;
  if (blockIdx.x > 0) return fill_piece(a, a.piece0 + blockIdx.x - 1);
  const int tid = threadIdx.x;
  uint32_t mine = ~0u;
  if (tid < kFew) {
    const long t = tid < (int)a.n ? load_index(a.tokens, a.wide, tid) : -1;
    if (t >= 0 && t < a.V) mine = (uint32_t)t << kPlaceBits | tid;
    item[tid] = mine;
  }
  if (tid == 0) all = 0;
  __syncthreads();
  if (mine != ~0u) {
    uint32_t rank = 0;
    for (int i = 0; i < kFew; i += 4) {
      const packet p = *reinterpret_cast<const packet*>(item + i);
#pragma unroll
      for (int k = 0; k < 4; k++) rank += p[k] < mine;
    }
    a.key1[rank] = mine >> kPlaceBits;
    a.place1[rank] = mine & ((1u << kPlaceBits) - 1);
    atomicAdd(&all, 1u);
  }
  __syncthreads();
  if (tid == 0) *a.count = all;
}

// Of more tokens: how often each digit stands in each tile,
template <int PASS>
__global__ __launch_bounds__(kSortThreads) void k_sort_count(SortK a) {
  __shared__ uint32_t count[kDigits];
  if ((int)blockIdx.x >= a.tiles) return fill_piece(a, a.piece0 + blockIdx.x - a.tiles);
  const int tid = threadIdx.x;
  if (tid < kDigits) count[tid] = 0;
  __syncthreads();
  const uint32_t n = PASS == 0 ? a.n : *a.count, first = blockIdx.x * a.tile;
  for (uint32_t i = tid; i < a.tile && first + i < n; i += kSortThreads) {
    const long t = PASS == 0 ? load_index(a.tokens, a.wide, first + i) : (long)a.key0[first + i];
    if (t >= 0 && t < a.V) atomicAdd(count + ((uint32_t)t >> (PASS * kDigitBits) & (kDigits - 1)), 1u);
  }
  __syncthreads();
  if (tid < kDigits) a.hist[(size_t)blockIdx.x * kDigits + tid] = count[tid];
}

// and each token to its place: behind the smaller digits, the same digit in the tiles
// before, and in this tile before it.  Every workgroup sums the counts for itself (a
// launch that placed the first digit and counted the second with atomics took 60 us for
// 500000 tokens, the two 21).
template <int PASS>
__global__ __launch_bounds__(kSortThreads) void k_sort_place(SortK a) {
  __shared__ RankLds s;
  if ((int)blockIdx.x >= a.tiles) return fill_piece(a, a.piece0 + blockIdx.x - a.tiles);
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const uint32_t n = PASS == 0 ? a.n : *a.count, first = blockIdx.x * a.tile, per_wave = a.tile / kSortWaves;
  uint32_t key[kRounds], place[kRounds], rank[kRounds];
#pragma unroll
  for (int r = 0; r < kRounds; r++) {
    const uint32_t at = first + wave * per_wave + r * 64 + lane;
    const bool in = (uint32_t)r * 64 < per_wave && at < n;
    const long t = !in ? -1 : PASS == 0 ? load_index(a.tokens, a.wide, at) : (long)a.key0[at];
    key[r] = t >= 0 && t < a.V ? (uint32_t)t : ~0u;
    place[r] = PASS == 0 ? at : in ? a.place0[at] : 0;
  }
  // every other tile's counts by each half of the threads, behind the tokens' own loads:
  // 500000 tokens 16.4 us a digit (one thread a digit before those loads 18.7), 16000 5.7
  // (5.2)
  static_assert(kSortThreads == 2 * kDigits, "two threads a digit");
  const int digit = tid & (kDigits - 1);
  uint32_t before = 0, all = 0;
#pragma unroll 8
  for (int t = tid / kDigits; t < a.tiles; t += 2) {
    const uint32_t c = a.hist[(size_t)t * kDigits + digit];
    if (t < (int)blockIdx.x) before += c;
    all += c;
  }
  if (tid >= kDigits) {
    s.count[0][digit] = before;
    s.count[1][digit] = all;
  }
  __syncthreads();
  if (tid < kDigits) {
    before += s.count[0][digit];
    all += s.count[1][digit];
  }
  __syncthreads();
  clear_counts(s);
#pragma unroll
  for (int r = 0; r < kRounds; r++) {
    rank[r] = ~0u;
    if ((uint32_t)r * 64 >= per_wave) continue;
    const bool on = key[r] != ~0u;
    const uint32_t k = rank_in_wave(s, wave, lane, key[r] >> (PASS * kDigitBits) & (kDigits - 1), on);
    if (on) rank[r] = k;
  }
  __syncthreads();
  uint32_t total;
  const uint32_t base = scan_digits(s, all, &total);
  place_waves(s, base + before);
  uint32_t *to_key = PASS == 0 ? a.key0 : a.key1, *to_place = PASS == 0 ? a.place0 : a.place1;
#pragma unroll
  for (int r = 0; r < kRounds; r++) {
    if (rank[r] == ~0u) continue;
    const uint32_t at = s.count[wave][key[r] >> (PASS * kDigitBits) & (kDigits - 1)] + rank[r];
    to_key[at] = key[r];
    to_place[at] = place[r];
  }
  if (PASS == 0 && blockIdx.x == 0 && tid == 0) *a.count = total;
}

// ---- sums along the sorted list --------------------------------------------------------

// The list is cut into stretches, one a thread and packet of columns, and those of a
// workgroup, `side` of them by `columns` packets, form a group.  A token's rows within a
// stretch are summed and written by its thread; what crosses a stretch's end is joined
// in LDS, what crosses a group's is left as a partial sum for the last launch.
struct SumK {
  const char* g;
  char* grad;
  size_t g_bytes, grad_bytes;
  const uint32_t *key, *place, *count;
  uint32_t n;  // tokens, those that are none among them
  float* partial;  // [groups][2][packets * kInPacket]: of the token that came in, of the one that goes out
  int D, packets, add;
  int columns_log2;        // packets of a workgroup
  uint32_t stretch;        // positions
  uint32_t slabs, groups;  // workgroups side by side and along the list
  float scale;
  bool past;
};

// scale * v to the table's row (or on top of it, but for the first `skip`, which are a
// neighbour's).
template <int DT, int OUT>
__device__ __forceinline__ void finish(const SumK& a, uint32_t token, int j, int skip, const float* v) {
  constexpr int n = Type<DT>::kInPacket, m = Type<OUT>::kInPacket;
  char* row = a.grad + (size_t)token * a.grad_bytes;
#pragma unroll
  for (int h = 0; h < n; h += m) {
    const int jh = j + h;
    if (jh + m <= a.D && !(a.add && skip)) {
      char* to = row + (size_t)jh * Type<OUT>::kBytes;
      float w[m];
      packet old{0, 0, 0, 0};
      if (a.add) old = *reinterpret_cast<const typename Type<OUT>::mem*>(to);
#pragma unroll
      for (int q = 0; q < m; q++) w[q] = v[h + q] * a.scale + (a.add ? value<OUT>(old, q) : 0.0f);
      packet p;
#pragma unroll
      for (int q = 0; q < 4; q++)
        p[q] = OUT == DTL_F32 ? bits_of<OUT>(w[q % m]) : bits_of<OUT>(w[2 * q % m]) | bits_of<OUT>(w[(2 * q + 1) % m]) << 16;
      store_packet<OUT>(to, p, a.past);
    } else {
#pragma unroll
      for (int q = 0; q < m; q++)
        if (h + q >= skip && jh + q < a.D)
          store_one<OUT>(row, jh + q, v[h + q] * a.scale + (a.add ? load_one<OUT>(row, jh + q) : 0.0f));
    }
  }
}

template <int n>
struct alignas(16) Sum {
  float v[n];
};

// The rows are read this once: without a place in the caches.
template <int DT>
__device__ __forceinline__ packet load_once(const char* row, int j, int D) {
  if (Type<DT>::kInPacket > D) return load_packet_at_once<DT>(row, 0, D);
  return __builtin_nontemporal_load(reinterpret_cast<const typename Type<DT>::mem*>(row + (size_t)j * Type<DT>::kBytes));
}

template <int DT, int OUT>
__global__ __launch_bounds__(kThreads) void k_embedding_sum(SumK a) {
  constexpr int n = Type<DT>::kInPacket, kAhead = 8;
  // of each stretch: the sum of the token that came in, and what there is
  __shared__ Sum<n> in[kThreads];
  __shared__ uint8_t state[kThreads];
  enum { CAME = 1, GOES = 2, ONE = 4 };
  const int tid = threadIdx.x, columns = 1 << a.columns_log2, side = kThreads >> a.columns_log2;
  const int s = tid >> a.columns_log2, c = tid & (columns - 1);
  const uint32_t group = blockIdx.x / a.slabs;
  const int col = (int)(blockIdx.x % a.slabs) * columns + c, j = packet_begin<DT>(col, a.D), skip = col * n - j;
  const uint32_t first = (group * side + s) * a.stretch;
  const bool mine = col < a.packets && first < a.n;
  // what the stretch begins with and what stands beside it, whether or not the list goes
  // so far (it is padded to whole stretches): these loads run together
  uint32_t key[kAhead] = {}, place[kAhead] = {}, before = 0, after = 0;
  auto take = [&](uint32_t p) {
#pragma unroll
    for (int i = 0; i < kAhead; i += 4) {
      const uint4 k = *reinterpret_cast<const uint4*>(a.key + p + i), l = *reinterpret_cast<const uint4*>(a.place + p + i);
      key[i] = k.x, key[i + 1] = k.y, key[i + 2] = k.z, key[i + 3] = k.w;
      place[i] = l.x, place[i + 1] = l.y, place[i + 2] = l.z, place[i + 3] = l.w;
    }
  };
  if (mine) {
    take(first);
    before = a.key[first ? first - 1 : 0];
    after = a.key[min(first + a.stretch, a.n - 1)];
  }
  const uint32_t all = *a.count, end = min(all, first + a.stretch);
  const bool here = mine && first < all;
  uint32_t now = key[0];
  bool came = here && first > 0 && before == now, one = true;
  float sum[n] = {};
  int what = came ? CAME : 0;
  for (uint32_t p = first; here && p < end; p += kAhead) {
    packet x[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; i++)
      if (p + i < end) x[i] = load_once<DT>(a.g + (size_t)place[i] * a.g_bytes, j, a.D);
    uint32_t held[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; i++) held[i] = key[i];
    if (p + kAhead < end) take(p + kAhead);
#pragma unroll
    for (int i = 0; i < kAhead; i++) {
      if (p + i >= end) break;
      if (held[i] != now) {
        if (came) {
#pragma unroll
          for (int q = 0; q < n; q++) in[tid].v[q] = sum[q];
        } else {
          finish<DT, OUT>(a, now, j, skip, sum);
        }
        came = one = false;
        now = held[i];
#pragma unroll
        for (int q = 0; q < n; q++) sum[q] = 0.0f;
      }
#pragma unroll
      for (int q = 0; q < n; q++) sum[q] += value<DT>(x[i], q);
    }
  }
  const bool goes = here && end < all && after == now;
  if (goes) what |= GOES;
  if (one) what |= ONE;
  if (here && !came && !goes) finish<DT, OUT>(a, now, j, skip, sum);
  if (came) {
#pragma unroll
    for (int q = 0; q < n; q++) in[tid].v[q] = sum[q];
  }
  state[tid] = (uint8_t)what;
  __syncthreads();
  if (!here) return;

  // from stretch t on: adds what came in, as far as the token goes; whether past the group
  auto follow = [&](int t) {
    for (; t < side; t++) {
      const int at = (t << a.columns_log2) + c;
#pragma unroll
      for (int q = 0; q < n; q++) sum[q] += in[at].v[q];
      if (!(state[at] & ONE && state[at] & GOES)) return false;
    }
    return true;
  };
  float* partial = a.partial + (size_t)group * 2 * a.packets * n + col * n;
  auto keep = [&](float* p) {
#pragma unroll
    for (int q = 0; q < n; q += 4) *reinterpret_cast<float4*>(p + q) = make_float4(sum[q], sum[q + 1], sum[q + 2], sum[q + 3]);
  };
  if (goes && !came) {  // it began here
    if (follow(s + 1))
      keep(partial + (size_t)a.packets * n);
    else
      finish<DT, OUT>(a, now, j, skip, sum);
  }
  if (s == 0 && what & CAME) {
#pragma unroll
    for (int q = 0; q < n; q++) sum[q] = 0.0f;
    follow(0);
    keep(partial);
  }
}

// The tokens that go out of a group where they began: a workgroup a group and slab, its
// sides sharing the groups that such a token goes through.
template <int DT, int OUT>
__global__ __launch_bounds__(kThreads) void k_embedding_join(SumK a) {
  constexpr int n = Type<DT>::kInPacket, kAhead = 4;
  __shared__ double part[kThreads][n];
  const int tid = threadIdx.x, columns = 1 << a.columns_log2, side = kThreads >> a.columns_log2;
  const int s = tid >> a.columns_log2, c = tid & (columns - 1);
  const uint32_t group = blockIdx.x / a.slabs, size = side * a.stretch;
  const int col = (int)(blockIdx.x % a.slabs) * columns + c;
  const uint32_t all = *a.count, first = group * size, end = first + size;
  if (end >= all) return;
  const uint32_t token = a.key[end];
  if (a.key[end - 1] != token || (first > 0 && a.key[first - 1] == token)) return;
  // the last group that it comes into
  uint32_t last = group + 1, step = 1;
  const uint32_t groups = (all - 1) / size;  // the last of all
  while (last + step <= groups && a.key[(last + step) * size] == token) last += step, step *= 2;
  for (; step; step /= 2)
    if (last + step <= groups && a.key[(last + step) * size] == token) last += step;
  const size_t one = (size_t)a.packets * n;
  double sum[n] = {};
  if (col < a.packets) {
    if (s == 0) {
      const float* p = a.partial + (size_t)group * 2 * one + one + col * n;
#pragma unroll
      for (int q = 0; q < n; q++) sum[q] = p[q];
    }
    uint32_t d = group + 1 + s;
    for (; d + (kAhead - 1) * side <= last; d += kAhead * side) {
      Sum<n> x[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; i++) x[i] = *reinterpret_cast<const Sum<n>*>(a.partial + (size_t)(d + i * side) * 2 * one + col * n);
#pragma unroll
      for (int i = 0; i < kAhead; i++)
#pragma unroll
        for (int q = 0; q < n; q++) sum[q] += x[i].v[q];
    }
    for (; d <= last; d += side) {
      const float* p = a.partial + (size_t)d * 2 * one + col * n;
#pragma unroll
      for (int q = 0; q < n; q++) sum[q] += p[q];
    }
  }
#pragma unroll
  for (int q = 0; q < n; q++) part[tid][q] = sum[q];
  __syncthreads();
  if (s || col >= a.packets) return;
  const int sides = last - group < (uint32_t)side ? (int)(last - group) : side;
  for (int t = 1; t < sides; t++)
#pragma unroll
    for (int q = 0; q < n; q++) sum[q] += part[(t << a.columns_log2) + c][q];
  float v[n];
#pragma unroll
  for (int q = 0; q < n; q++) v[q] = (float)sum[q];
  const int j = packet_begin<DT>(col, a.D);
  finish<DT, OUT>(a, token, j, col * n - j, v);
}

// ---- launches ---------------------------------------------------------------------------

// What does not fit the memory-side cache together with what it is made of is written
// past it, so that what is read beside it stays.  One pass of lookup and gradient, us,
// past / not: 65536 bf16 rows of 2048 into 32000 167 / 208, 16384 of 896 into 151936
// 80 / 86, 8192 f32 rows of 2048 into 32000 94 / 102; where it fits (2048 f32 rows of 576
// into 49152) 37 / 30.
bool past_caches(size_t bytes) { return bytes > (size_t)256 << 20; }

int packets_of(size_t width, int dtype) { return (int)((width * type_bytes(dtype) + 15) / 16); }

// How a gradient of n positions by so many packets is cut.
struct Cut {
  int columns_log2;
  uint32_t stretch, slabs, groups;
};
Cut cut_of(size_t n, size_t packets) {
  Cut c{};
  while (c.columns_log2 < 4 && (size_t)1 << c.columns_log2 < packets) c.columns_log2++;
  c.slabs = (uint32_t)((packets + ((size_t)1 << c.columns_log2) - 1) >> c.columns_log2);
  c.stretch = 8;
  while (c.stretch < 64 && n * packets / c.stretch > kBusy) c.stretch *= 2;
  const size_t size = (size_t)c.stretch * (kThreads >> c.columns_log2);
  c.groups = (uint32_t)((n + size - 1) / size);
  return c;
}

struct Layout {  // of the scratch
  uint32_t tile;
  int tiles;
  size_t list, hist, key0, place0, key1, place1, partial, bytes;
};
Layout layout_of(size_t n, size_t width) {
  Layout l{};
  // us for both digits of 74894 tokens by tiles of 1024 / 2048 24 / 24; of
  // 500000 by 4096 / 8192 41 / 54
  const size_t per = n <= 65536 ? 1024 : n <= 131072 ? 2048 : (n + kTiles - 1) / kTiles;
  l.tile = (uint32_t)((per + kSortThreads - 1) / kSortThreads * kSortThreads);
  l.tiles = (int)((n + l.tile - 1) / (l.tile ? l.tile : 1));
  l.list = (n + 1023) / 1024 * 1024 * 4;
  l.hist = 256;
  l.key0 = l.hist + (size_t)kTiles * kDigits * 4;
  l.place0 = l.key0 + l.list;
  l.key1 = l.place0 + l.list;
  l.place1 = l.key1 + l.list;
  l.partial = l.place1 + l.list;
  l.bytes = l.partial;
  for (int e : {DTL_F32, DTL_BF16}) {  // whichever the rows are
    const size_t packets = packets_of(width, e);
    const size_t need = l.partial + cut_of(n, packets).groups * 2 * packets * (e == DTL_F32 ? 4 : 8) * 4;
    if (need > l.bytes) l.bytes = need;
  }
  return l;
}

}  // namespace
}  // namespace dtl

// ---- C entry points ------------------------------------------------------------------------

using namespace dtl;

namespace {

// As for rows of logits.
bool spacing_ok(size_t rows, size_t width, size_t stride) {
  return rows <= 1 || (stride >= width && stride <= ((size_t)1 << 48) / rows);
}

bool dtype_ok(int t) { return t == DTL_F32 || t == DTL_BF16 || t == DTL_F16; }

int check_table(const dtl_table* t) {
  if (!t || !dtype_ok(t->dtype)) return DTL_ERR_INVALID_ARGUMENT;
  if (t->vocab == 0) return DTL_ERR_CDF_EMPTY;
  if (t->vocab > (size_t)kScoreMaxVocab) return DTL_ERR_CDF_TOO_MANY_SYMBOLS;
  if (t->width == 0 || t->width > kEmbedMaxWidth) return DTL_ERR_SHAPE;
  if (!spacing_ok(t->vocab, t->width, t->stride)) return DTL_ERR_SHAPE;
  if (!t->data || reinterpret_cast<uintptr_t>(t->data) % type_bytes(t->dtype)) return DTL_ERR_INVALID_ARGUMENT;
  return DTL_OK;
}
int check_rows(const void* p, int dtype, size_t n, size_t width, size_t stride) {
  if (!spacing_ok(n, width, stride)) return DTL_ERR_SHAPE;
  return n && (!p || reinterpret_cast<uintptr_t>(p) % type_bytes(dtype)) ? DTL_ERR_INVALID_ARGUMENT : DTL_OK;
}
// From a tensor's first row to the end of its last.
size_t extent(size_t n, size_t width, size_t stride, int dtype) {
  return n ? ((n - 1) * stride + width) * type_bytes(dtype) : 0;
}
bool apart(const void* a, size_t na, const void* b, size_t nb) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  return x + na <= y || y + nb <= x;
}
template <typename K>
void launch_threads(void (*kernel)(K), size_t threads, hipStream_t s, const K& k) {
  launch_kernel(kernel, dim3((unsigned)((threads + kThreads - 1) / kThreads)), dim3(kThreads), 0, s, k);
}

}  // namespace

extern "C" {

int dtl_embedding(const dtl_table* t, const void* tokens, int token_bytes, size_t n, float scale, void* out,
                  size_t out_stride, void* stream) {
  int st = check_table(t);
  if (st) return st;
  if (n > kMostRows) return DTL_ERR_SHAPE;
  if (!index_bytes_ok(token_bytes) || (n && !tokens)) return DTL_ERR_INVALID_ARGUMENT;
  st = check_rows(out, t->dtype, n, t->width, out_stride);
  if (st || n == 0) return st;
  if (!apart(out, extent(n, t->width, out_stride, t->dtype), t->data, extent(t->vocab, t->width, t->stride, t->dtype)))
    return DTL_ERR_INVALID_ARGUMENT;
  LookupK k{};
  k.table = static_cast<const char*>(t->data);
  k.out = static_cast<char*>(out);
  k.tokens = tokens;
  k.n = n;
  k.table_bytes = t->stride * type_bytes(t->dtype);
  k.out_bytes = out_stride * type_bytes(t->dtype);
  k.V = (int)t->vocab;
  k.D = (int)t->width;
  k.packets = packets_of(t->width, t->dtype);
  k.wide = token_bytes == 8;
  k.scale = scale;
  k.past = past_caches((n + (n < t->vocab ? n : t->vocab)) * t->width * type_bytes(t->dtype));
  const size_t most = ((size_t)1 << 31) / k.packets;  // rows a launch
  by_type(t->dtype, [&](auto dt) {
    for (k.row0 = 0; k.row0 < n; k.row0 += most)
      launch_threads(k_embedding<decltype(dt)::value>, (n - k.row0 < most ? n - k.row0 : most) * k.packets,
                     static_cast<hipStream_t>(stream), k);
  });
  return launch_status();
}

size_t dtl_embedding_backward_scratch(size_t n, size_t vocab, size_t width) {
  if (n > kEmbedMaxTokens || vocab > (size_t)kScoreMaxVocab || width > kEmbedMaxWidth) return 0;
  return layout_of(n, width).bytes;
}

int dtl_embedding_backward(const void* tokens, int token_bytes, size_t n, const void* grad_out, int grad_dtype,
                           size_t grad_out_stride, float scale, const dtl_table* grad, int add, void* scratch,
                           size_t scratch_bytes, void* stream) {
  int st = check_table(grad);
  if (st) return st;
  if (!dtype_ok(grad_dtype) || (grad->dtype != grad_dtype && grad->dtype != DTL_F32)) return DTL_ERR_INVALID_ARGUMENT;
  if (n > kEmbedMaxTokens) return DTL_ERR_SHAPE;
  if (!index_bytes_ok(token_bytes) || (n && !tokens)) return DTL_ERR_INVALID_ARGUMENT;
  st = check_rows(grad_out, grad_dtype, n, grad->width, grad_out_stride);
  if (st) return st;
  const Layout l = layout_of(n, grad->width);
  if (scratch_bytes < l.bytes) return DTL_ERR_BUFFER_TOO_SMALL;
  if (!scratch || reinterpret_cast<uintptr_t>(scratch) % 16) return DTL_ERR_INVALID_ARGUMENT;
  const size_t e = type_bytes(grad->dtype), all = extent(grad->vocab, grad->width, grad->stride, grad->dtype);
  if (n && !apart(grad->data, all, grad_out, extent(n, grad->width, grad_out_stride, grad_dtype)))
    return DTL_ERR_INVALID_ARGUMENT;
  if (n == 0 && add) return DTL_OK;
  hipStream_t s = static_cast<hipStream_t>(stream);
  char* mem = static_cast<char*>(scratch);

  SortK k{};
  k.tokens = tokens;
  k.wide = token_bytes == 8;
  k.V = (int)grad->vocab;
  k.n = (uint32_t)n;
  k.tile = l.tile;
  k.count = reinterpret_cast<uint32_t*>(mem);
  k.hist = reinterpret_cast<uint32_t*>(mem + l.hist);
  k.key0 = reinterpret_cast<uint32_t*>(mem + l.key0);
  k.place0 = reinterpret_cast<uint32_t*>(mem + l.place0);
  k.key1 = reinterpret_cast<uint32_t*>(mem + l.key1);
  k.place1 = reinterpret_cast<uint32_t*>(mem + l.place1);
  k.past = past_caches(grad->vocab * grad->width * e + n * grad->width * type_bytes(grad_dtype));
  if (!add) {
    const bool whole = grad->vocab == 1 || grad->stride == grad->width;
    k.fill = static_cast<char*>(grad->data);
    k.fill_rows = whole ? 1 : grad->vocab;
    k.fill_bytes = (whole ? grad->vocab : 1) * grad->width * e;
    k.fill_stride = grad->stride * e;
    k.pieces = (k.fill_rows * ((k.fill_bytes + 15) / 16) * 16 + kFillBytes - 1) / kFillBytes;
  }
  if (n <= (size_t)kAlone) {
    // us, zeros aside: 7 to 200 tokens 4 by counting, 9 by digits; 1000 5, 2118 8, 4096 11
    // by digits, 8000 19 (18 in four launches)
    launch_kernel(n <= kFew ? k_sort_few : k_sort_alone, dim3((unsigned)(1 + k.pieces)), dim3(kSortThreads), 0, s, k);
  } else {
    k.tiles = l.tiles;
    const size_t quarter = (k.pieces + 3) / 4;
    void (*const steps[])(SortK) = {k_sort_count<0>, k_sort_place<0>, k_sort_count<1>, k_sort_place<1>};
    for (auto step : steps) {
      launch_kernel(step, dim3((unsigned)(k.tiles + quarter)), dim3(kSortThreads), 0, s, k);
      k.piece0 += quarter;
    }
  }
  if (n) {
    SumK u{};
    u.g = static_cast<const char*>(grad_out);
    u.grad = static_cast<char*>(grad->data);
    u.g_bytes = grad_out_stride * type_bytes(grad_dtype);
    u.grad_bytes = grad->stride * e;
    u.key = k.key1;
    u.place = k.place1;
    u.count = k.count;
    u.n = k.n;
    u.partial = reinterpret_cast<float*>(mem + l.partial);
    u.D = (int)grad->width;
    u.packets = packets_of(grad->width, grad_dtype);
    u.add = add != 0;
    const Cut cut = cut_of(n, u.packets);
    u.columns_log2 = cut.columns_log2;
    u.stretch = cut.stretch;
    u.slabs = cut.slabs;
    u.groups = cut.groups;
    u.scale = scale;
    u.past = k.past;
    const size_t threads = (size_t)cut.groups * cut.slabs * kThreads;
    by_type(grad_dtype, [&](auto dt) {
      constexpr int DT = decltype(dt)::value;
      by_bool(grad->dtype == DTL_F32, [&](auto wide) {
        constexpr int OUT = decltype(wide)::value ? DTL_F32 : DT;
        launch_threads(k_embedding_sum<DT, OUT>, threads, s, u);
        if (cut.groups > 1) launch_threads(k_embedding_join<DT, OUT>, threads, s, u);
      });
    });
  }
  return launch_status();
}

}  // extern "C"
