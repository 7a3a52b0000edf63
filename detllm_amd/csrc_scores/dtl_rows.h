// What the operators on rows in device memory share: elements of the three
// types, sums over a wave, launches, and the checks of their entry points.
#pragma once

#include <type_traits>

#include "../csrc/dtl_device.h"
#include "dtl_scores.h"

namespace dtl {

// ---- logits of the three types ------------------------------------------------

// 16 bytes at an element's alignment: rows of an odd stride are only aligned
// to their elements, and gfx950 loads and stores 16 bytes at any address.
typedef uint32_t packet __attribute__((ext_vector_type(4)));
typedef packet packet4 __attribute__((aligned(4)));
typedef packet packet2 __attribute__((aligned(2)));

template <int DT>
struct Type {  // bf16 and f16
  static constexpr int kBytes = 2, kInPacket = 8;
  static constexpr uint32_t kMasked = DT == DTL_BF16 ? 0xff80ff80u : 0xfc00fc00u;
  typedef packet2 mem;
};
template <>
struct Type<DTL_F32> {
  static constexpr int kBytes = 4, kInPacket = 4;
  static constexpr uint32_t kMasked = 0xff800000u;
  typedef packet4 mem;
};
template <int DT>
__device__ __forceinline__ float value(const packet& p, int i) {
  const uint32_t w = p[DT == DTL_F32 ? i : i / 2];
  if constexpr (DT == DTL_F32) return __builtin_bit_cast(float, w);
  if constexpr (DT == DTL_BF16) return __builtin_bit_cast(float, i & 1 ? w & 0xffff0000u : w << 16);
  return (float)__builtin_bit_cast(_Float16, (uint16_t)(i & 1 ? w >> 16 : w));
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

// The same by loads that do not wait for each other: every element's, the last one's in
// place of those past V.  V > j.
template <int DT>
__device__ __forceinline__ packet load_packet_at_once(const char* row, int j, int V) {
  constexpr int n = Type<DT>::kInPacket;
  if (j + n <= V) return *reinterpret_cast<const typename Type<DT>::mem*>(row + (size_t)j * Type<DT>::kBytes);
  packet p;
  uint32_t e[n];
#pragma unroll
  for (int q = 0; q < n; q++) {
    const int at = min(j + q, V - 1);
    if constexpr (DT == DTL_F32)
      e[q] = reinterpret_cast<const uint32_t*>(row)[at];
    else
      e[q] = reinterpret_cast<const uint16_t*>(row)[at];
  }
#pragma unroll
  for (int q = 0; q < n; q++)
    if (j + q >= V) e[q] = Type<DT>::kMasked & (DT == DTL_F32 ? ~0u : 0xffffu);
#pragma unroll
  for (int q = 0; q < 4; q++) p[q] = DT == DTL_F32 ? e[q % n] : e[2 * q % n] | e[(2 * q + 1) % n] << 16;
  return p;
}

// Past the caches or not.  The two stores are kept apart: the compiler would make one
// of them, without the hint.
template <int DT>
__device__ __forceinline__ void store_packet(char* at, const packet& p, bool past) {
  typename Type<DT>::mem* to = reinterpret_cast<typename Type<DT>::mem*>(at);
  if (past) {
    asm volatile("");
    __builtin_nontemporal_store(p, to);
    asm volatile("");
  } else {
    *to = p;
  }
}

__device__ __forceinline__ long load_index(const void* p, int wide, size_t i) {
  return wide ? (long)reinterpret_cast<const int64_t*>(p)[i] : (long)reinterpret_cast<const int32_t*>(p)[i];
}

// Before a workgroup writes again over what its other waves wrote: every store is
// done, not only issued (a barrier by itself leaves stores of other waves in flight).
__device__ __forceinline__ void wait_for_stores() {
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
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
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t dpp(uint32_t x, uint32_t idle) {
  return __builtin_amdgcn_update_dpp((int)idle, (int)x, CTRL, ROWS, 0xf, false);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ double dpp(double x) {
  const uint64_t b = __builtin_bit_cast(uint64_t, x);
  const uint32_t lo = dpp<CTRL, ROWS>((uint32_t)b, 0u), hi = dpp<CTRL, ROWS>((uint32_t)(b >> 32), 0u);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ double wave_sum(double x) {
  x += dpp<0x111, 0xf>(x);
  x += dpp<0x112, 0xf>(x);
  x += dpp<0x114, 0xf>(x);
  x += dpp<0x118, 0xf>(x);
  x += dpp<0x142, 0xa>(x);
  x += dpp<0x143, 0xc>(x);
  const uint64_t b = __builtin_bit_cast(uint64_t, x);
  const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)b, 63), hi = __builtin_amdgcn_readlane((int)(b >> 32), 63);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
// Inclusive sums over the lanes up to each.
__device__ __forceinline__ uint32_t wave_scan(uint32_t x) {
  x += dpp<0x111, 0xf>(x, 0u);
  x += dpp<0x112, 0xf>(x, 0u);
  x += dpp<0x114, 0xf>(x, 0u);
  x += dpp<0x118, 0xf>(x, 0u);
  x += dpp<0x142, 0xa>(x, 0u);
  x += dpp<0x143, 0xc>(x, 0u);
  return x;
}
__device__ __forceinline__ uint32_t wave_max(uint32_t x) {
  x = max(x, dpp<0x111, 0xf>(x, 0u));
  x = max(x, dpp<0x112, 0xf>(x, 0u));
  x = max(x, dpp<0x114, 0xf>(x, 0u));
  x = max(x, dpp<0x118, 0xf>(x, 0u));
  x = max(x, dpp<0x142, 0xa>(x, 0u));
  x = max(x, dpp<0x143, 0xc>(x, 0u));
  return __builtin_amdgcn_readlane((int)x, 63);
}

// ---- launches ---------------------------------------------------------------------------

// A launch of `per_row` workgroups a row; of many rows several, of as many as keep the
// launch's threads below 2^32.
constexpr size_t kRowsPerLaunch = 1u << 18;
template <typename K>
void launch_rows(void (*kernel)(K), size_t rows, int per_row, int threads, size_t lds, hipStream_t s, K k) {
  const size_t fit = 0xffffffffu / ((size_t)per_row * threads), most = fit < kRowsPerLaunch ? fit : kRowsPerLaunch;
  for (k.row0 = 0; k.row0 < rows; k.row0 += most) {
    const size_t n = rows - k.row0 < most ? rows - k.row0 : most;
    launch_kernel(kernel, dim3((unsigned)(n * per_row)), dim3(threads), lds, s, k);
  }
}

inline size_t round256(size_t n) { return (n + 255) & ~(size_t)255; }

template <typename F>
void by_bool(bool b, F&& f) {
  if (b)
    f(std::true_type());
  else
    f(std::false_type());
}
template <typename F>
void by_type(int dtype, F&& f) {
  if (dtype == DTL_F32)
    f(std::integral_constant<int, DTL_F32>());
  else if (dtype == DTL_BF16)
    f(std::integral_constant<int, DTL_BF16>());
  else
    f(std::integral_constant<int, DTL_F16>());
}
inline size_t type_bytes(int dtype) { return dtype == DTL_F32 ? 4 : 2; }

// Gradients larger than the memory-side cache are written past it: 423 instead of
// 450 us for 4096 rows of 151936 bf16, 408 instead of 426 for 2048 of f32.
inline bool write_past(size_t rows, size_t row_bytes) { return rows * row_bytes > (size_t)256 << 20; }

// ---- entry points --------------------------------------------------------------------------

inline int launch_status() {
  switch (hipGetLastError()) {
    case hipSuccess: return DTL_OK;
    case hipErrorOutOfMemory: return DTL_ERR_OUT_OF_MEMORY;
    case hipErrorNoDevice:
    case hipErrorInvalidDevice: return DTL_ERR_NO_DEVICE;
    default: return DTL_ERR_DEVICE;
  }
}

constexpr size_t kMostRows = 1u << 24;

// One row has no stride; others do not overlap, and their bytes can be counted.
inline bool stride_ok(const dtl_logits* z, size_t stride) {
  return z->rows <= 1 || (stride >= z->vocab && stride <= ((size_t)1 << 48) / z->rows);
}

inline int check_logits(const dtl_logits* z) {
  if (!z) return DTL_ERR_INVALID_ARGUMENT;
  if (z->dtype != DTL_F32 && z->dtype != DTL_BF16 && z->dtype != DTL_F16) return DTL_ERR_INVALID_ARGUMENT;
  if (z->vocab == 0) return DTL_ERR_CDF_EMPTY;
  if (z->vocab > (size_t)kScoreMaxVocab) return DTL_ERR_CDF_TOO_MANY_SYMBOLS;
  if (z->rows > kMostRows || !stride_ok(z, z->stride)) return DTL_ERR_SHAPE;
  if (z->rows == 0) return DTL_OK;
  if (!z->data || reinterpret_cast<uintptr_t>(z->data) % type_bytes(z->dtype)) return DTL_ERR_INVALID_ARGUMENT;
  return DTL_OK;
}
inline bool index_bytes_ok(int n) { return n == 4 || n == 8; }

// Whether a row of the gradient lies over a part of the logits' rows other than
// itself: logits would be overwritten that another wave has yet to read.  Rows may
// interleave (two halves of one matrix, say).
inline bool overlap(const dtl_logits* z, const void* grad, size_t grad_stride) {
  const size_t n = type_bytes(z->dtype), row = z->vocab * n, zs = z->stride * n, gs = grad_stride * n, last = z->rows - 1;
  const uintptr_t a = reinterpret_cast<uintptr_t>(z->data), g = reinterpret_cast<uintptr_t>(grad);
  if (last == 0) return a != g && a < g + row && g < a + row;
  if (a == g && zs == gs) return false;
  if (a >= g + last * gs + row || g >= a + last * zs + row) return false;
  for (size_t i = 0; i <= last; i++) {  // against the last of the gradient's rows that begins before this one's end
    const uintptr_t at = a + i * zs;
    if (at + row <= g) continue;
    const size_t j = (at + row - 1 - g) / gs;
    if (at < g + (j < last ? j : last) * gs + row) return true;
  }
  return false;
}

inline int check_grad(const dtl_logits* z, const void* grad, size_t stride) {
  if (!stride_ok(z, stride)) return DTL_ERR_SHAPE;
  if (z->rows == 0) return DTL_OK;
  if (!grad || reinterpret_cast<uintptr_t>(grad) % type_bytes(z->dtype)) return DTL_ERR_INVALID_ARGUMENT;
  return overlap(z, grad, stride) ? DTL_ERR_INVALID_ARGUMENT : DTL_OK;
}

}  // namespace dtl
