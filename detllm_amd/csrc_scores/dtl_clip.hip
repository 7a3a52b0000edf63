// The norm over many tensors, and the tensors times what brings it down to a maximum.
//
//   norm = |s| sqrt(sum x^2) or |s| max |x|;   y = x s min(1, max_norm / (norm + 1e-6))
//
// Bound by memory: one read for the norm, one more and a write for the product, whose
// factor is known only when every element has been read.  A launch takes a table of
// tensors as its argument (nothing to upload, nothing that a captured graph could lose),
// each workgroup a piece of one of them.  Squares and sums are in 64 bits: a gradient of
// 1e20 has a norm, one of 1e-30 too.  The pieces' sums are joined by one workgroup in a
// fixed order: the same list gives the same bits; the same elements cut otherwise differ by
// some 2^-53 of the sum, far below the norm's rounding to 32 bits.
#include "dtl_scores.h"

#include <algorithm>
#include <new>
#include <vector>

#include "dtl_rows.h"

namespace dtl {
namespace {

constexpr int kThreads = 256, kJoinThreads = 1024;
// Elements a workgroup reads for the norm, and scales.  us for 201 bf16 tensors of 1.1e9
// elements: norm by 16384 / 32768 328 / 325, and 10 / 6.5 to join the pieces; clipping by
// 8192 / 16384 / 32768 757 / 792 / 808.
constexpr size_t kPiece = 32768, kClipPiece = 8192;
// Workgroups of a clipping in place at most: with a factor of 1 there is nothing to do, and
// 201 bf16 tensors of 133000 pieces take 347 us in all instead of the 368 of a workgroup a
// piece; with another one their pieces one after the other take 1175 instead of 1144.
constexpr uint32_t kInPlaceGroups = 16384;
constexpr size_t kCache = (size_t)256 << 20, kKept = (size_t)192 << 20;
constexpr int kNormEntries = 180, kClipEntries = 128;

struct Entry {
  const char* x;
  uint64_t bits;  // the count, above it the element's type and whether the output is f32
};
constexpr int kTypeShift = 48, kWideShift = 56;
__device__ inline uint64_t count_of(const Entry& e) { return e.bits & (((uint64_t)1 << kTypeShift) - 1); }
__device__ inline int type_of(const Entry& e) { return (int)(e.bits >> kTypeShift & 15); }
__device__ inline bool wide_of(const Entry& e) { return e.bits >> kWideShift; }

struct NormK {
  Entry entry[kNormEntries];
  uint32_t first[kNormEntries];  // each tensor's first piece of the launch
  int n;
  uint32_t slot0;      // of the launch's first piece among all
  uint32_t keep_from;  // pieces from here on are left in the caches
  double* part;
};
struct ClipK {
  Entry entry[kClipEntries];
  char* out[kClipEntries];
  uint32_t first[kClipEntries];
  int n;
  uint32_t pieces;
  bool past;  // written past the caches
  bool in_place;
  const float* factor;
};
static_assert(sizeof(NormK) <= 4096 && sizeof(ClipK) <= 4096, "fit a kernel's arguments");

// The tensor that holds a piece.
template <typename K>
__device__ __forceinline__ int find(const K& a, uint32_t piece) {
  int lo = 0, hi = a.n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (a.first[mid] <= piece)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

// A number that orders magnitudes, infinities above and NaN on top.
__device__ __forceinline__ uint32_t magnitude(float v) { return __builtin_bit_cast(uint32_t, v) & 0x7fffffffu; }

template <int DT, bool LARGEST, bool ONCE>
__device__ __forceinline__ double piece_of(const char* x, uint64_t count, uint64_t at) {
  constexpr int n = Type<DT>::kInPacket, ahead = 4;
  typedef typename Type<DT>::mem mem;
  const int tid = threadIdx.x, left = (int)(count - at < kPiece ? count - at : kPiece);
  x += at * Type<DT>::kBytes;
  double sum[ahead] = {};
  uint32_t most = 0;
  auto take = [&](int k, float v) {
    if (LARGEST)
      most = max(most, magnitude(v));
    else
      sum[k] = __builtin_fma((double)v, (double)v, sum[k]);
  };
  int j = tid * n;
  for (; j + (ahead - 1) * kThreads * n + n <= left; j += ahead * kThreads * n) {
    packet p[ahead];
#pragma unroll
    for (int k = 0; k < ahead; k++) {
      const mem* from = reinterpret_cast<const mem*>(x + (size_t)(j + k * kThreads * n) * Type<DT>::kBytes);
      p[k] = ONCE ? __builtin_nontemporal_load(from) : *from;
    }
#pragma unroll
    for (int q = 0; q < n; q++)
#pragma unroll
      for (int k = 0; k < ahead; k++) take(k, value<DT>(p[k], q));
  }
  for (; j < left; j += kThreads * n)
    for (int q = 0; q < n && j + q < left; q++) take(0, load_one<DT>(x, j + q));
  if (LARGEST) return (double)__builtin_bit_cast(float, wave_max(most));
  return wave_sum((sum[0] + sum[1]) + (sum[2] + sum[3]));
}

// Whichever is larger, NaN above all.
__device__ __forceinline__ double larger(double a, double b) { return !(a == a) || a > b ? a : b; }

template <bool LARGEST, bool ONCE>
__device__ __forceinline__ double piece_of(const Entry& t, uint64_t at) {
  switch (type_of(t)) {
    case DTL_F32: return piece_of<DTL_F32, LARGEST, ONCE>(t.x, count_of(t), at);
    case DTL_BF16: return piece_of<DTL_BF16, LARGEST, ONCE>(t.x, count_of(t), at);
    default: return piece_of<DTL_F16, LARGEST, ONCE>(t.x, count_of(t), at);
  }
}

template <bool LARGEST>
__global__ __launch_bounds__(kThreads) void k_norm(NormK a) {
  __shared__ double waves[kThreads / 64];
  const int e = find(a, blockIdx.x);
  const Entry t = a.entry[e];
  const uint64_t at = (uint64_t)(blockIdx.x - a.first[e]) * kPiece;
  const uint32_t slot = a.slot0 + blockIdx.x;
  double v = slot < a.keep_from ? piece_of<LARGEST, true>(t, at) : piece_of<LARGEST, false>(t, at);
  if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = v;
  __syncthreads();
  if (threadIdx.x) return;
  for (int w = 1; w < kThreads / 64; w++) v = LARGEST ? larger(waves[w], v) : v + waves[w];
  a.part[slot] = v;
}

struct JoinK {
  const double* part;
  uint32_t n;
  int clip;
  float scale, max_norm;
  const float* scale_at;
  float *norm, *factor;
};

template <bool LARGEST>
__global__ __launch_bounds__(kJoinThreads) void k_norm_join(JoinK a) {
  constexpr int ahead = 8;
  __shared__ double all[kJoinThreads / 64];
  const int tid = threadIdx.x;
  double v = 0.0;
  auto take = [&](double p) { v = LARGEST ? larger(p, v) : v + p; };
  uint32_t i = tid;
  for (; i + (ahead - 1) * kJoinThreads < a.n; i += ahead * kJoinThreads) {
    double p[ahead];
#pragma unroll
    for (int k = 0; k < ahead; k++) p[k] = a.part[i + k * kJoinThreads];
#pragma unroll
    for (int k = 0; k < ahead; k++) take(p[k]);
  }
  for (; i < a.n; i += kJoinThreads) take(a.part[i]);
  for (int d = 1; d < 64; d *= 2) take(__shfl_xor(v, d));
  if ((tid & 63) == 0) all[tid >> 6] = v;
  __syncthreads();
  if (tid) return;
  for (int w = 1; w < kJoinThreads / 64; w++) take(all[w]);
  const double s = a.scale_at ? *a.scale_at : a.scale, norm = __builtin_fabs(s) * (LARGEST ? v : __builtin_sqrt(v));
  *a.norm = (float)norm;
  if (!a.clip) return;
  const double c = a.max_norm / (norm + 1e-6);
  *a.factor = (float)(s * (c > 1.0 ? 1.0 : c));
}

// A lane's stores are 16 bytes and next to its neighbours', so of 16-bit elements that
// become f32 it reads 8.
template <int DT, int OUT>
__device__ __forceinline__ void scale_piece(const char* x, char* y, uint64_t count, uint64_t at, float f,
                                            bool past) {
  constexpr int n = Type<OUT>::kInPacket, ahead = 4;
  typedef uint32_t half __attribute__((ext_vector_type(2)));
  typedef half half2 __attribute__((aligned(2)));
  typedef std::conditional_t<DT == OUT, typename Type<DT>::mem, half2> mem;
  const int tid = threadIdx.x, left = (int)(count - at < kClipPiece ? count - at : kClipPiece);
  x += at * Type<DT>::kBytes;
  y += at * Type<OUT>::kBytes;
  int j = tid * n;
  for (; j + (ahead - 1) * kThreads * n + n <= left; j += ahead * kThreads * n) {
    packet p[ahead];
#pragma unroll
    for (int k = 0; k < ahead; k++) {
      const mem v = *reinterpret_cast<const mem*>(x + (size_t)(j + k * kThreads * n) * Type<DT>::kBytes);
      if constexpr (DT == OUT)
        p[k] = v;
      else
        p[k] = packet{v[0], v[1], 0, 0};
    }
#pragma unroll
    for (int k = 0; k < ahead; k++) {
      packet w;
#pragma unroll
      for (int q = 0; q < 4; q++)
        w[q] = OUT == DTL_F32 ? bits_of<OUT>(value<DT>(p[k], q) * f)
                              : bits_of<OUT>(value<DT>(p[k], 2 * q % n) * f) | bits_of<OUT>(value<DT>(p[k], (2 * q + 1) % n) * f) << 16;
      store_packet<OUT>(y + (size_t)(j + k * kThreads * n) * Type<OUT>::kBytes, w, past);
    }
  }
  for (; j < left; j += kThreads * n)
    for (int q = 0; q < n && j + q < left; q++) store_one<OUT>(y, j + q, load_one<DT>(x, j + q) * f);
}

__global__ __launch_bounds__(kThreads) void k_clip(ClipK a) {
  const float f = *a.factor;
  if (f == 1.0f && a.in_place) return;
  for (uint32_t piece = blockIdx.x; piece < a.pieces; piece += gridDim.x) {
    const int e = find(a, piece);
    const Entry t = a.entry[e];
    // what the norm read last may still be in the cache: backwards
    const uint64_t last = (count_of(t) - 1) / kClipPiece, at = (last - (piece - a.first[e])) * kClipPiece;
    char* y = a.out[e];
    switch (type_of(t)) {
      case DTL_F32: scale_piece<DTL_F32, DTL_F32>(t.x, y, count_of(t), at, f, a.past); break;
      case DTL_BF16:
        if (wide_of(t))
          scale_piece<DTL_BF16, DTL_F32>(t.x, y, count_of(t), at, f, a.past);
        else
          scale_piece<DTL_BF16, DTL_BF16>(t.x, y, count_of(t), at, f, a.past);
        break;
      default:
        if (wide_of(t))
          scale_piece<DTL_F16, DTL_F32>(t.x, y, count_of(t), at, f, a.past);
        else
          scale_piece<DTL_F16, DTL_F16>(t.x, y, count_of(t), at, f, a.past);
    }
  }
}

}  // namespace
}  // namespace dtl

// ---- C entry points ------------------------------------------------------------------------

using namespace dtl;

namespace {

constexpr size_t kMostCount = (size_t)1 << 36;  // the pieces of one tensor fit a launch
constexpr uint32_t kMostPieces = 0xffffffffu / kThreads;
static_assert(kMostCount / kClipPiece <= kMostPieces, "fewer than 2^32 threads");

size_t pieces_of(const dtl_tensor& t, size_t piece = kPiece) { return (t.count + piece - 1) / piece; }

// The tensors' pieces; 0 with *st set for a list that is refused.
size_t check_tensors(const dtl_tensor* t, size_t n, int* st) {
  size_t pieces = 0;
  *st = n > kClipMaxTensors ? DTL_ERR_SHAPE : n && !t ? DTL_ERR_INVALID_ARGUMENT : DTL_OK;
  for (size_t i = 0; i < n && !*st; i++) {
    if (t[i].dtype != DTL_F32 && t[i].dtype != DTL_BF16 && t[i].dtype != DTL_F16)
      *st = DTL_ERR_INVALID_ARGUMENT;
    else if (t[i].count > kMostCount || (pieces += pieces_of(t[i])) > (size_t)1 << 31)
      *st = DTL_ERR_SHAPE;
    else if (t[i].count && (!t[i].data || reinterpret_cast<uintptr_t>(t[i].data) % type_bytes(t[i].dtype)))
      *st = DTL_ERR_INVALID_ARGUMENT;
  }
  return *st ? 0 : pieces;
}

size_t scratch_of(size_t pieces) { return 16 + pieces * sizeof(double); }

int check_out(const dtl_tensor* t, const dtl_tensor* out, size_t n) {
  int st;
  check_tensors(out, n, &st);
  if (st) return st;
  struct Span {
    uintptr_t begin, end;
    size_t i;
  };
  try {
    std::vector<Span> spans;
    for (size_t i = 0; i < n; i++) {
      if (out[i].count != t[i].count) return DTL_ERR_SHAPE;
      if (out[i].dtype != t[i].dtype && out[i].dtype != DTL_F32) return DTL_ERR_INVALID_ARGUMENT;
      const uintptr_t at = reinterpret_cast<uintptr_t>(out[i].data);
      if (out[i].count) spans.push_back({at, at + out[i].count * type_bytes(out[i].dtype), i});
    }
    std::sort(spans.begin(), spans.end(), [](const Span& a, const Span& b) { return a.begin < b.begin; });
    for (size_t k = 1; k < spans.size(); k++)
      if (spans[k].begin < spans[k - 1].end) return DTL_ERR_INVALID_ARGUMENT;
    for (size_t i = 0; i < n; i++) {  // what is read of another tensor, or elsewhere, must not be written
      if (!t[i].count) continue;
      const uintptr_t at = reinterpret_cast<uintptr_t>(t[i].data), end = at + t[i].count * type_bytes(t[i].dtype);
      auto s = std::upper_bound(spans.begin(), spans.end(), at, [](uintptr_t a, const Span& b) { return a < b.end; });
      for (; s != spans.end() && s->begin < end; ++s)
        if (s->i != i || s->begin != at || out[i].dtype != t[i].dtype) return DTL_ERR_INVALID_ARGUMENT;
    }
  } catch (const std::bad_alloc&) {
    return DTL_ERR_OUT_OF_MEMORY;
  }
  return DTL_OK;
}

// Cuts the list, or the list backwards, into launches of at most `most` tensors that
// have elements.
template <typename K, typename Put, typename Go>
void in_launches(K& k, int most, size_t piece, bool back, const dtl_tensor* t, size_t n, Put&& put, Go&& go) {
  uint32_t pieces = 0;
  k.n = 0;
  for (size_t j = 0; j < n; j++) {
    const size_t i = back ? n - 1 - j : j;
    if (!t[i].count) continue;
    const uint32_t more = (uint32_t)pieces_of(t[i], piece);
    if (k.n == most || pieces > kMostPieces - more) {
      go(pieces);
      k.n = 0;
      pieces = 0;
    }
    k.entry[k.n] = {static_cast<const char*>(t[i].data), (uint64_t)t[i].dtype << kTypeShift | t[i].count};
    k.first[k.n] = pieces;
    put(k.n++, i);
    pieces += more;
  }
  if (k.n) go(pieces);
}

int norm_and_clip(const dtl_tensor* t, size_t n, int largest, float scale, const float* scale_at, bool clip, float max_norm,
                  const dtl_tensor* out, float* norm, void* scratch, size_t scratch_bytes, void* stream) {
  int st;
  const size_t pieces = check_tensors(t, n, &st);
  if (st) return st;
  if (!norm) return DTL_ERR_INVALID_ARGUMENT;
  if (clip) {
    if (!(max_norm >= 0.0f)) return DTL_ERR_INVALID_ARGUMENT;
    st = check_out(t, out ? out : t, n);
    if (st) return st;
  }
  if (scratch_bytes < scratch_of(pieces)) return DTL_ERR_BUFFER_TOO_SMALL;
  if (!scratch || reinterpret_cast<uintptr_t>(scratch) % 16) return DTL_ERR_INVALID_ARGUMENT;
  hipStream_t s = static_cast<hipStream_t>(stream);
  float* factor = static_cast<float*>(scratch);
  NormK k{};
  k.part = reinterpret_cast<double*>(static_cast<char*>(scratch) + 16);
  // More than the memory-side cache holds is read past it, but for what the clipping,
  // which goes backwards and writes past it, will still find there (kKept; us for norm and
  // clipping, 0 / 128 / 192 MB kept: 201 bf16 tensors of 2.2 GB 1098 / 1087 / 1086, cached
  // throughout 1125; 392 MB of f16 to f32 264 / 260 / 253, cached throughout 259).
  size_t bytes = 0;
  for (size_t i = 0; i < n; i++) bytes += t[i].count * type_bytes(t[i].dtype);
  if (bytes > kCache) {
    size_t keep = 0, left = clip ? kKept : 0;
    for (size_t i = n; i-- && left;) {
      const size_t piece = kPiece * type_bytes(t[i].dtype), fit = left / piece;
      if (pieces_of(t[i]) >= fit) {
        keep += fit;
        break;
      }
      keep += pieces_of(t[i]);
      left -= pieces_of(t[i]) * piece;
    }
    k.keep_from = (uint32_t)(pieces - keep);
  }
  in_launches(k, kNormEntries, kPiece, false, t, n, [](int, size_t) {}, [&](uint32_t count) {
    launch_kernel(largest ? k_norm<true> : k_norm<false>, dim3(count), dim3(kThreads), 0, s, k);
    k.slot0 += count;
  });
  JoinK j{k.part, (uint32_t)pieces, clip, scale, max_norm, scale_at, norm, factor};
  launch_kernel(largest ? k_norm_join<true> : k_norm_join<false>, dim3(1), dim3(kJoinThreads), 0, s, j);
  if (clip) {
    ClipK c{};
    c.factor = factor;
    c.past = bytes > kCache;
    c.in_place = out == nullptr;
    const dtl_tensor* to = out ? out : t;
    in_launches(
        c, kClipEntries, kClipPiece, true, t, n,
        [&](int e, size_t i) {
          c.out[e] = static_cast<char*>(to[i].data);
          if (to[i].dtype == DTL_F32) c.entry[e].bits |= (uint64_t)1 << kWideShift;
        },
        [&](uint32_t count) {
          c.pieces = count;
          launch_kernel(k_clip, dim3(c.in_place && count > kInPlaceGroups ? kInPlaceGroups : count), dim3(kThreads), 0, s, c);
        });
  }
  return launch_status();
}

}  // namespace

extern "C" {

size_t dtl_grad_norm_scratch(const dtl_tensor* tensors, size_t n) {
  int st;
  const size_t pieces = check_tensors(tensors, n, &st);
  return st ? 0 : scratch_of(pieces);
}

int dtl_grad_norm(const dtl_tensor* tensors, size_t n, int largest, float scale, const float* scale_at, float* norm,
                  void* scratch, size_t scratch_bytes, void* stream) {
  return norm_and_clip(tensors, n, largest, scale, scale_at, false, 0.0f, nullptr, norm, scratch, scratch_bytes, stream);
}

int dtl_clip_grads(const dtl_tensor* tensors, size_t n, int largest, float scale, const float* scale_at, float max_norm,
                   const dtl_tensor* out, float* norm, void* scratch, size_t scratch_bytes, void* stream) {
  return norm_and_clip(tensors, n, largest, scale, scale_at, true, max_norm, out, norm, scratch, scratch_bytes, stream);
}

}  // extern "C"
