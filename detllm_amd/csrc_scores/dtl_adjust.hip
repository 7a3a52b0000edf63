// Penalties for repeated tokens, biases and masks on rows of logits, and their
// gradient.
//
//   a = z;  token in the history: a = z > 0 ? z / theta : z theta;  n times behind
//   the prompt: a -= presence + frequency n;  a += bias;  not allowed: a = -inf.
//   dz = g (theta^-1 or theta where the token stood, 0 where it is not allowed).
//
// Bound by memory: one read and one write of the logits (in place, only what changes
// is read and written), an eighth of a byte of mask.  A workgroup has a segment of a
// row, whose logits go through registers in 16-byte packets.  It counts the history's
// tokens there in a table in LDS, one word a logit of the segment: a direct table needs
// no probing, and integer sums have no order.  Almost every logit is only copied or
// masked, so a lane goes through those of its packet that the table names one by one.
// Each segment's workgroup scans the whole history, from the caches.
#include "dtl_scores.h"

#include "dtl_rows.h"

namespace dtl {
namespace {

// A table word: 13 bits of the last bias's place + 1, whether the token stands in
// the prompt, and how often behind it.
constexpr uint32_t kPlaceMask = (1u << 13) - 1, kInPrompt = 1u << 13, kOnce = 1u << 14;
static_assert(kAdjustMaxBiases <= kPlaceMask && kAdjustMaxHistory < 1 << 18, "fit a table word");

enum { COPY, IN_PLACE, GRAD };

struct AdjustK {
  const char* z;
  const char* from;  // what is copied: the logits, or the gradient
  char* out;
  size_t z_bytes, from_bytes, out_bytes, row0;
  int V, nseg;
  int history_len, bias_len;  // 0 where they change nothing
  dtl_adjust by;
  bool past;  // written past the caches
};

template <int DT>
__device__ __forceinline__ uint32_t allowed_bits(const AdjustK& a, size_t row, int j, int n) {
  // of logits j .. j + n, n at most a packet's: bit i for logit j + i
  const char* p = static_cast<const char*>(a.by.allowed) + row * a.by.allowed_stride * (a.by.allowed_bits == 1 ? 4 : 1);
  if (a.by.allowed_bits == 1) return (uint32_t)(uint8_t)p[j >> 3] >> (j & 7);
  constexpr int all = Type<DT>::kInPacket;
  if (n == all) {
    typedef uint32_t word __attribute__((aligned(1)));
    uint32_t m = (reinterpret_cast<const word*>(p + j)[0] & 0x01010101u) * 0x01020408u >> 24 & 15;
    if (all == 8) m |= ((reinterpret_cast<const word*>(p + j)[1] & 0x01010101u) * 0x01020408u >> 24 & 15) << 4;
    return m;
  }
  uint32_t m = 0;
  for (int i = 0; i < n; i++) m |= (uint32_t)(p[j + i] & 1) << i;
  return m;
}

// The packet with `no` in the places whose bit is not set.
template <int DT>
__device__ __forceinline__ packet blend(packet p, uint32_t bits, uint32_t no) {
#pragma unroll
  for (int d = 0; d < 4; d++) {
    uint32_t keep;
    if constexpr (DT == DTL_F32)
      keep = (uint32_t)((int32_t)(bits << (31 - d)) >> 31);
    else
      keep = ((uint32_t)((int32_t)(bits << (31 - 2 * d)) >> 31) & 0xffffu) |
             ((uint32_t)((int32_t)(bits << (30 - 2 * d)) >> 31) & 0xffff0000u);
    p[d] = (p[d] & keep) | (no & ~keep);
  }
  return p;
}

__device__ __forceinline__ float of_row(const float* rows, float one, size_t row) { return rows ? rows[row] : one; }

// An element of a packet, and its bits put back; q differs from lane to lane.
template <int DT>
__device__ __forceinline__ uint32_t word_of(const packet& p, int q) {
  const int d = DT == DTL_F32 ? q : q / 2;
  return d == 0 ? p[0] : d == 1 ? p[1] : d == 2 ? p[2] : p[3];
}
template <int DT>
__device__ __forceinline__ float pick(const packet& p, int q) {
  const uint32_t w = word_of<DT>(p, q);
  if constexpr (DT == DTL_F32) return __builtin_bit_cast(float, w);
  const uint32_t h = q & 1 ? w >> 16 : w & 0xffffu;
  if constexpr (DT == DTL_BF16) return __builtin_bit_cast(float, h << 16);
  return (float)__builtin_bit_cast(_Float16, (uint16_t)h);
}
template <int DT>
__device__ __forceinline__ void put(packet& p, int q, float v) {
  uint32_t w = bits_of<DT>(v);
  if constexpr (DT != DTL_F32) w = q & 1 ? (word_of<DT>(p, q) & 0xffffu) | w << 16 : (word_of<DT>(p, q) & 0xffff0000u) | w;
  const int at = DT == DTL_F32 ? q : q / 2;
#pragma unroll
  for (int d = 0; d < 4; d++) p[d] = at == d ? w : p[d];
}

// Workgroups go to the eight dies in turn, each with a cache of its own: those of one
// row on one die read its history into one cache instead of eight.
__device__ __forceinline__ uint32_t by_die(uint32_t block, uint32_t blocks) {
  const uint32_t each = blocks / 8;
  return block < each * 8 ? block % 8 * each + block / 8 : block;
}

template <int DT, int MODE, bool TABLE, int SEG, int kThreads>
__global__ __launch_bounds__(kThreads) void k_adjust(AdjustK a) {
  constexpr int n = Type<DT>::kInPacket, np = SEG / (kThreads * n), kHistory = 4;
  constexpr uint32_t no = MODE == GRAD ? 0u : Type<DT>::kMasked;
  static_assert(np * kThreads * n == SEG, "whole packets");
  __shared__ __attribute__((aligned(16))) uint32_t table[TABLE ? SEG : 4];
  const int tid = threadIdx.x;
  const uint32_t block = TABLE ? by_die(blockIdx.x, gridDim.x) : blockIdx.x;
  const size_t row = a.row0 + block / a.nseg;
  const int base = (int)(block % a.nseg) * SEG, end = min(a.V, base + SEG);
  const char* from = a.from + row * a.from_bytes;
  char* out = a.out + row * a.out_bytes;

  // the first ids of the lists, then the segment: their loads run together
  long ids[kHistory], bias_id = -1;
  const size_t hrow = row * a.by.history_stride, brow = row * a.by.bias_stride;
  if (TABLE) {
#pragma unroll
    for (int i = 0; i < kHistory; i++) {
      const int at = tid + i * kThreads;
      ids[i] = at < a.history_len ? load_index(a.by.history, a.by.history_bytes == 8, hrow + at) : -1;
    }
    if (tid < a.bias_len) bias_id = load_index(a.by.bias_ids, a.by.bias_bytes == 8, brow + tid);
  }
  const bool masked = a.by.allowed != nullptr;
  packet p[np];
  uint32_t bits[np];
#pragma unroll
  for (int i = 0; i < np; i++) {
    const int j = base + (i * kThreads + tid) * n;
    bits[i] = ~0u;
    if (j < end) {
      if (masked) bits[i] = allowed_bits<DT>(a, row, j, min(n, end - j));
      if (MODE != IN_PLACE) p[i] = load_packet_at_once<DT>(from, j, end);
    }
  }

  float theta = 1.0f, presence = 0.0f, frequency = 0.0f;
  if (TABLE) {
    theta = of_row(a.by.repetitions, a.by.repetition, row);
    presence = of_row(a.by.presences, a.by.presence, row);
    frequency = of_row(a.by.frequencies, a.by.frequency, row);
    const int prompt = a.by.prompt ? a.by.prompt[row] : 0;
    for (int i = tid * 4; i < SEG; i += kThreads * 4) *reinterpret_cast<packet*>(table + i) = packet{0, 0, 0, 0};
    __syncthreads();
    if (a.bias_len) {
      auto place = [&](long id, int k) {
        const uint64_t j = (uint64_t)id - (uint64_t)base;
        if (j < (uint64_t)(end - base)) atomicMax(table + j, (uint32_t)k + 1);
      };
      place(bias_id, tid);
      for (int k = tid + kThreads; k < a.bias_len; k += kThreads)
        place(load_index(a.by.bias_ids, a.by.bias_bytes == 8, brow + k), k);
      __syncthreads();
    }
    if (a.history_len) {
      auto count = [&](long id, int at) {
        const uint64_t j = (uint64_t)id - (uint64_t)base;
        if (j >= (uint64_t)(end - base)) return;
        if (at < prompt)
          atomicOr(table + j, kInPrompt);
        else
          atomicAdd(table + j, kOnce);
      };
#pragma unroll
      for (int i = 0; i < kHistory; i++) count(ids[i], tid + i * kThreads);
      auto rest = [&](const auto* list) {
        int at = tid + kHistory * kThreads;
        for (; at + 7 * kThreads < a.history_len; at += 8 * kThreads) {
          long more[8];
#pragma unroll
          for (int i = 0; i < 8; i++) more[i] = list[hrow + at + i * kThreads];
#pragma unroll
          for (int i = 0; i < 8; i++) count(more[i], at + i * kThreads);
        }
        for (; at < a.history_len; at += kThreads) count(list[hrow + at], at);
      };
      if (a.by.history_bytes == 8)
        rest(static_cast<const int64_t*>(a.by.history));
      else
        rest(static_cast<const int32_t*>(a.by.history));
      __syncthreads();
    }
  }

  // which of a packet's logits were touched and stay allowed
  uint32_t hits[np];
  packet sign[MODE == GRAD ? np : 1];
#pragma unroll
  for (int i = 0; i < np; i++) {
    hits[i] = 0;
    if (!TABLE) continue;
    const int at = (i * kThreads + tid) * n;
#pragma unroll
    for (int q = 0; q < n; q += 4) {
      const packet w = *reinterpret_cast<const packet*>(table + at + q);
#pragma unroll
      for (int k = 0; k < 4; k++) hits[i] |= w[k] ? 1u << (q + k) : 0u;
    }
    hits[i] &= bits[i];
    if (MODE == GRAD && hits[i]) sign[i] = load_packet_at_once<DT>(a.z + row * a.z_bytes, base + at, end);
  }

#pragma unroll
  for (int i = 0; i < np; i++) {
    const int at = (i * kThreads + tid) * n, j = base + at;
    if (j >= end) continue;
    const int here = min(n, end - j);
    const uint32_t all = (1u << here) - 1, on = bits[i] & all;
    if (MODE == IN_PLACE) {
      if (on == all && !hits[i]) continue;
      // few to write: without reading their neighbours (256 rows of 151936 bf16, half of
      // them with 3 % masked: 16.3 us, 20.8 with a read of every packet, 17.8 with none)
      if (!hits[i] && here == n && __builtin_popcount(all & ~on) <= n / 2) {
        for (uint32_t off = all & ~on; off; off &= off - 1) store_one<DT>(out, j + __builtin_ctz(off), -__builtin_inff());
        continue;
      }
      p[i] = on ? load_packet_at_once<DT>(from, j, end) : packet{no, no, no, no};
    }
    packet w = blend<DT>(p[i], bits[i], no);
    for (uint32_t h = hits[i]; h; h &= h - 1) {
      const int q = __builtin_ctz(h);
      const uint32_t word = table[at + q], times = word / kOnce;
      const float x = pick<DT>(w, q);
      if (MODE == GRAD) {
        put<DT>(w, q, pick<DT>(sign[i], q) > 0.0f ? x / theta : x * theta);
        continue;
      }
      float v = x;
      if (word > kPlaceMask) v = x > 0.0f ? x / theta : x * theta;
      if (times) v -= presence + frequency * (float)times;
      if (word & kPlaceMask) v += a.by.biases[brow + (word & kPlaceMask) - 1];
      put<DT>(w, q, v);
    }
    if (here == n) {
      store_packet<DT>(out + (size_t)j * Type<DT>::kBytes, w, a.past);
    } else {
#pragma unroll
      for (int q = 0; q < n; q++)
        if (q < here) {
          if constexpr (DT == DTL_F32)
            reinterpret_cast<uint32_t*>(out)[j + q] = w[q];
          else
            reinterpret_cast<uint16_t*>(out)[j + q] = (uint16_t)(w[q / 2] >> (q & 1 ? 16 : 0));
        }
    }
  }
}

template <int DT, int MODE, bool TABLE, int SEG, int THREADS>
void launch_as(AdjustK& k, size_t rows, hipStream_t s) {
  k.nseg = (k.V + SEG - 1) / SEG;
  launch_rows(k_adjust<DT, MODE, TABLE, SEG, THREADS>, rows, k.nseg, THREADS, 0, s, k);
}

// A row's segments by its length and the history's.  us of 2048 logits by four waves /
// 8192 by eight / 16384 by sixteen: 16384 rows of 1000 bf16 25 / 52 / 101, 8192 of 2500
// 37 / 42 / 65; histories of 200, 16 rows of 32000 3.9 / 4.6 / 5.4; of 2048, 64 rows of
// 151936 15.2 / 11.6 / 12.7; of 8192, 512 such rows 207 / 108 / 103; of 32768, 64 of them
// 80 / 33 / 27, 8 of them 17.3 / 11.5 / 12.1.  Segments of 8192 by four / eight / sixteen
// waves: 2048 rows of 151936 f32 478 / 436 / 470; 4096 of bf16 418 / 417 / 573, their
// gradients 527 / 464 / 633.
template <int DT, int MODE>
void launch_mode(AdjustK& k, size_t rows, bool table, hipStream_t s) {
  if (k.V <= 4096 || (rows * k.V < (1u << 21) && k.history_len <= 1024))
    by_bool(table, [&](auto t) { launch_as<DT, MODE, decltype(t)::value, 2048, 256>(k, rows, s); });
  else if (k.history_len > 4096)  // of which there is a table
    launch_as<DT, MODE, true, 16384, 1024>(k, rows, s);
  else
    by_bool(table, [&](auto t) { launch_as<DT, MODE, decltype(t)::value, 8192, 512>(k, rows, s); });
}

}  // namespace

int check_adjust(const dtl_adjust* by, size_t rows, size_t vocab) {
  if (!by) return DTL_ERR_INVALID_ARGUMENT;
  if (rows && by->history_len && !by->history) return DTL_ERR_INVALID_ARGUMENT;
  if (rows && by->bias_len && (!by->bias_ids || !by->biases)) return DTL_ERR_INVALID_ARGUMENT;
  if (by->history_len) {
    if (!index_bytes_ok(by->history_bytes)) return DTL_ERR_INVALID_ARGUMENT;
    if (by->history_len > (size_t)kAdjustMaxHistory || by->history_stride > ((size_t)1 << 40)) return DTL_ERR_SHAPE;
    if (!by->repetitions && !(by->repetition > 0.0f && by->repetition < __builtin_inff())) return DTL_ERR_INVALID_ARGUMENT;
    if (!by->presences && !(by->presence - by->presence == 0.0f)) return DTL_ERR_INVALID_ARGUMENT;
    if (!by->frequencies && !(by->frequency - by->frequency == 0.0f)) return DTL_ERR_INVALID_ARGUMENT;
  }
  if (by->bias_len) {
    if (!index_bytes_ok(by->bias_bytes)) return DTL_ERR_INVALID_ARGUMENT;
    if (by->bias_len > (size_t)kAdjustMaxBiases || by->bias_stride > ((size_t)1 << 40)) return DTL_ERR_SHAPE;
  }
  if (by->allowed) {
    if (by->allowed_bits != 1 && by->allowed_bits != 8) return DTL_ERR_INVALID_ARGUMENT;
    const size_t row = by->allowed_bits == 1 ? (vocab + 31) / 32 : vocab;
    if (rows > 1 && by->allowed_stride && by->allowed_stride < row) return DTL_ERR_SHAPE;
    if (by->allowed_stride > ((size_t)1 << 40)) return DTL_ERR_SHAPE;
    if (by->allowed_bits == 1 && reinterpret_cast<uintptr_t>(by->allowed) % 4) return DTL_ERR_INVALID_ARGUMENT;
  }
  return DTL_OK;
}

void launch_adjust(const AdjustArgs& a, hipStream_t s) {
  if (a.rows == 0) return;
  const size_t e = type_bytes(a.dtype);
  AdjustK k{};
  k.z = static_cast<const char*>(a.z);
  k.from = static_cast<const char*>(a.grad ? a.grad : a.z);
  k.out = static_cast<char*>(a.out);
  k.z_bytes = a.stride * e;
  k.from_bytes = (a.grad ? a.grad_stride : a.stride) * e;
  k.out_bytes = a.out_stride * e;
  k.V = a.vocab;
  k.by = a.by;
  k.past = write_past(a.rows, k.out_bytes);
  const bool repeats = a.by.repetitions || a.by.repetition != 1.0f;
  const bool counts = a.by.presences || a.by.frequencies || a.by.presence != 0.0f || a.by.frequency != 0.0f;
  if (a.by.history && (repeats || (counts && !a.grad))) k.history_len = (int)a.by.history_len;
  if (a.by.bias_ids && !a.grad) k.bias_len = (int)a.by.bias_len;
  const bool table = k.history_len || k.bias_len, same = k.from == k.out;
  if (same && !table && !a.by.allowed) return;
  by_type(a.dtype, [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    if (a.grad)
      launch_mode<DT, GRAD>(k, a.rows, table, s);
    else if (same)
      launch_mode<DT, IN_PLACE>(k, a.rows, table, s);
    else
      launch_mode<DT, COPY>(k, a.rows, table, s);
  });
}

}  // namespace dtl

// ---- C entry points ------------------------------------------------------------------------

using namespace dtl;

namespace {
AdjustArgs adjust_args(const dtl_logits* z, const dtl_adjust* by, void* out, size_t out_stride) {
  AdjustArgs a{};
  a.z = z->data;
  a.stride = z->stride;
  a.rows = z->rows;
  a.dtype = z->dtype;
  a.vocab = (int)z->vocab;
  a.by = *by;
  a.out = out;
  a.out_stride = out_stride;
  return a;
}
}  // namespace

extern "C" {

int dtl_adjust_logits(const dtl_logits* z, const dtl_adjust* by, void* out, size_t out_stride, void* stream) {
  int st = check_logits(z);
  if (!st) st = check_adjust(by, z->rows, z->vocab);
  if (!st) st = check_grad(z, out, out_stride);
  if (st || z->rows == 0) return st;
  launch_adjust(adjust_args(z, by, out, out_stride), static_cast<hipStream_t>(stream));
  return launch_status();
}

int dtl_adjust_logits_backward(const dtl_logits* z, const dtl_adjust* by, const void* grad_out, size_t grad_out_stride,
                               void* grad, size_t grad_stride, void* stream) {
  int st = check_logits(z);
  if (!st) st = check_adjust(by, z->rows, z->vocab);
  if (st) return st;
  dtl_logits g = *z;
  g.data = grad_out;
  g.stride = grad_out_stride;
  st = check_logits(&g);
  if (!st) st = check_grad(&g, grad, grad_stride);
  if (!st) st = check_grad(z, grad, grad_stride);
  if (st || z->rows == 0) return st;
  // a logit's sign is read after its gradient is written
  if (grad == z->data) return DTL_ERR_INVALID_ARGUMENT;
  AdjustArgs a = adjust_args(z, by, grad, grad_stride);
  a.grad = grad_out;
  a.grad_stride = grad_out_stride;
  launch_adjust(a, static_cast<hipStream_t>(stream));
  return launch_status();
}

}  // extern "C"
