// 16-bit scalars, their matrix instructions and the small pieces the low-rank and checkpoint kernels share.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace eigamd {

using f32x4 = float __attribute__((ext_vector_type(4)));
using i16x4 = short __attribute__((ext_vector_type(4)));

#define EIGAMD_LDS(T, p) ((__attribute__((address_space(3))) T*)(p))
#define EIGAMD_GLOBAL(p) ((const __attribute__((address_space(1))) void*)(p))

// Eight consecutive elements along the reduction are what a lane hands to one 16 x 16 x 32 product: lane l holds row (or
// column) l % 16 and positions 8 (l / 16) .. + 7 of the reduction.  The result holds column l % 16, rows 4 (l / 16) .. + 3.
struct Bf16 {
  using elem = __bf16;
  using x8 = __bf16 __attribute__((ext_vector_type(8)));
  using x4 = __bf16 __attribute__((ext_vector_type(4)));
  static constexpr int bytes = 2;
  static __device__ __forceinline__ f32x4 mma(x8 a, x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
  static __device__ __forceinline__ x4 read_transposed(const void* p) { return __builtin_bit_cast(x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16(EIGAMD_LDS(i16x4, p))); }
};
struct F16 {
  using elem = _Float16;
  using x8 = _Float16 __attribute__((ext_vector_type(8)));
  using x4 = _Float16 __attribute__((ext_vector_type(4)));
  static constexpr int bytes = 2;
  static __device__ __forceinline__ f32x4 mma(x8 a, x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
  static __device__ __forceinline__ x4 read_transposed(const void* p) { return __builtin_bit_cast(x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16(EIGAMD_LDS(i16x4, p))); }
};
// Single precision has no 32-deep product; the eight values of a lane go through eight 4-deep ones, which reduce over the
// same 32 positions (in another order, the same one for both operands).
struct Fp32 {
  using elem = float;
  using x8 = float __attribute__((ext_vector_type(8)));
  static constexpr int bytes = 4;
  static __device__ __forceinline__ f32x4 mma(x8 a, x8 b, f32x4 c) {
#pragma unroll
    for (int i = 0; i < 8; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], c, 0, 0, 0);
    return c;
  }
};

// A float as a sum of three bf16 values, each the leading 8 bits of what is left: they hold all 24 bits of any finite v.  They are cut,
// not rounded (rounding up could leave the range).  An infinity leaves NaN, and pieces may be zero, which an infinity on the other side
// makes NaN: who multiplies them looks for NaN and takes v itself then.
__device__ __forceinline__ float upper_half(float v) { return __int_as_float(__float_as_int(v) & 0xffff0000); }
__device__ __forceinline__ void split_bf16(float v, __bf16 (&piece)[3]) {
  const float first = upper_half(v), left = v - first, second = upper_half(left);
  piece[0] = (__bf16)first;
  piece[1] = (__bf16)second;
  piece[2] = (__bf16)(left - second);
}

// Power of two that brings the largest of |v| into [2^14, 2^15) (below it for what is smaller than 2^-112), and its inverse; 1 where that
// is not finite.
struct Norm {
  float down, up;
};
__device__ __forceinline__ Norm norm_of(float largest) {
  int e = (__float_as_int(largest) >> 23) & 255;
  if (e == 255) return {1.0f, 1.0f};
  e = e < 15 ? 15 : e;
  return {__int_as_float((268 - e) << 23), __int_as_float((e - 14) << 23)};
}

// A v below 2^15 as three f16 values in the same way, 11 bits each, the second and third of 2^UP times what the first leaves (UP at most
// 10, as that is below 2^5).  They hold all of v from smallest_f16<UP>() on, where its last bit is a whole multiple of f16's smallest
// number, 2^-24, over 2^UP.
template <int UP> __device__ __forceinline__ void split_f16(float v, _Float16 (&piece)[3]) {
  piece[0] = (_Float16)__builtin_amdgcn_cvt_pkrtz(v, 0.0f)[0];
  const float left = (v - (float)piece[0]) * (float)(1 << UP);
  piece[1] = (_Float16)__builtin_amdgcn_cvt_pkrtz(left, 0.0f)[0];
  piece[2] = (_Float16)(left - (float)piece[1]);
}
template <int UP> constexpr float smallest_f16() { return 0.5f / (float)(1 << UP); }

// Of 8 values: is one of them, other than zero, below `least` in magnitude?  (As whole numbers magnitudes keep their order, and zero, less
// one, is above all of them.)
template <typename V> __device__ __forceinline__ bool some_below(const V& v, float least) {
  unsigned low = ~0u;
#pragma unroll
  for (int t = 0; t < 8; ++t) {
    const unsigned b = (__float_as_uint(v[t]) & 0x7fffffff) - 1;
    low = low < b ? low : b;
  }
  return low < __float_as_uint(least) - 1;
}
template <typename V> __device__ __forceinline__ float largest_of(const V& v) {
  float top = 0.0f;
#pragma unroll
  for (int t = 0; t < 8; ++t) top = fmaxf(top, __builtin_fabsf(v[t]));
  return top;
}

// 2^(e - 127) for an exponent byte.  255 gives infinity: a block that held infinities or NaN is stored as zeros with
// exponent 255 and comes back as 0 * inf = NaN.
__device__ __forceinline__ float exponent_scale(unsigned e) { return __int_as_float((int)(e << 23)); }

// The 8 values q * scale of one chunk: |q| <= 127 has 7 bits, so they are exact in every type (the packing keeps the exponent in
// the type's range).
template <typename T> __device__ __forceinline__ typename T::x8 unpack_8(uint64_t q, float scale) {
  typename T::x8 v;
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = (typename T::elem)((float)(int8_t)(q >> (8 * i)) * scale);
  return v;
}

template <typename E, typename V> __device__ __forceinline__ V load_8(const E* p) {
  V v;
  __builtin_memcpy(&v, p, 8 * sizeof(E));
  return v;
}
// n <= 8 elements from p (any alignment), the rest zero.
template <typename E, typename V> __device__ __forceinline__ V load_up_to_8(const E* p, int n) {
  if (n >= 8) return load_8<E, V>(p);
  V v;
  {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < n ? p[i] : (E)0.0f;
  }
  return v;
}

// The first n of 8 elements `stride` apart, the rest zero (p itself has to be readable even for n <= 0).  No load is conditional:
// conditional ones would be waited for one by one.
template <typename E, typename V> __device__ __forceinline__ V load_first(const E* p, int64_t stride, int n) {
  V v;
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = p[(i < n ? i : 0) * stride];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = i < n ? v[i] : (E)0.0f;
  return v;
}

// Between the LDS accesses of a wave's lanes that meet each other's data: the hardware keeps a wave's accesses in order, and this makes
// the compiler do so too (it reasons about one lane, whose own addresses may well differ).  No instruction.
__device__ __forceinline__ void wave_order() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// n <= 8 whole numbers of 8 bits from p (any alignment), the rest zero.
__device__ __forceinline__ uint64_t load_bytes(const int8_t* p, int n) {
  uint64_t v = 0;
  if (n >= 8) {
    __builtin_memcpy(&v, p, 8);
  } else {
    for (int i = 0; i < 8; ++i)
      if (i < n) v |= (uint64_t)(uint8_t)p[i] << (8 * i);
  }
  return v;
}

// Which piece of which adapter workgroup-slot t stands for, when every adapter's run of the sorted batch is cut into pieces of
// `size` tokens.  Adapter j's pieces take the slots from starts[j] / size + j on: the base of j + 1 is never below the base of
// j plus j's pieces, so slots are unique without a prefix sum, and there are at most n / size + adapters + 1 of them.
// One wave finds j by counting bases <= t, four loads under way together.  Returns false for a slot that no piece has.
struct Piece {
  int adapter, index, begin, end, run_begin, run_end;      // index: of the run's pieces
};
__device__ __forceinline__ bool find_piece(const int* starts, int segments, int size, int t, Piece& out) {
  const int lane = threadIdx.x & 63;
  int below = 0;
  for (int j0 = 0; j0 < segments; j0 += 256) {
    int start[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) start[u] = starts[j0 + u * 64 + lane < segments ? j0 + u * 64 + lane : segments];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int j = j0 + u * 64 + lane;
      below += __popcll(__ballot(j < segments && start[u] / size + j <= t));
    }
  }
  const int j = below - 1;   // base of adapter 0 is 0
  out.adapter = j;
  out.run_begin = starts[j];
  out.run_end = starts[j + 1];
  out.index = t - (out.run_begin / size + j);
  out.begin = out.run_begin + out.index * size;
  out.end = out.begin + size < out.run_end ? out.begin + size : out.run_end;
  return out.begin < out.run_end;
}

// The same where there are more adapters than tokens: slot t is the t-th place of the sorted batch where an adapter's tokens or a
// multiple of SIZE begins; no more than n / SIZE + n slots, and n tokens to look at instead of all adapters (17 tokens x 2048 x 2048,
// 4096 adapters of rank 64 577 -> 12 us).  (index, run_begin and run_end are not looked for.)
template <int SIZE> __device__ __forceinline__ bool find_piece_by_tokens(const int* seg, int n, int t, Piece& out) {
  static_assert(64 % SIZE == 0, "a piece ends inside the 64 tokens it begins in");
  const int lane = threadIdx.x & 63;
  for (int i0 = 0; i0 < n; i0 += 256) {
    int own[4], before[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int i = i0 + u * 64 + lane < n ? i0 + u * 64 + lane : n - 1;
      own[u] = seg[i];
      before[u] = seg[i > 0 ? i - 1 : 0];
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int i = i0 + u * 64 + lane;
      const bool first = i < n && (i % SIZE == 0 || own[u] != before[u]);
      const unsigned long long places = __ballot(first);
      if (t < __popcll(places)) {
        const int at = __builtin_ctzll(__ballot(first && __popcll(places & ((1ull << lane) - 1)) == t));
        const unsigned long long behind = places & ~((2ull << at) - 1);
        out.adapter = __builtin_amdgcn_readlane(own[u], at);
        out.begin = i0 + u * 64 + at;
        out.end = i0 + u * 64 + (behind ? __builtin_ctzll(behind) : 64);
        out.end = out.end < n ? out.end : n;
        return true;
      }
      t -= __popcll(places);
    }
  }
  return false;
}

}  // namespace eigamd
