// Activations held in 8 bits for the backward pass, and the weight gradient that reads them.
//
// 32 consecutive features of a token share a power-of-two scale 2^e, e the smallest with max|x| <= 127 2^e: q = round(x / 2^e)
// to whole numbers, ties to even.  A power of two costs up to one of the eight bits against a free scale and makes the rest
// exact: the division, and q 2^e as a bf16, f16 or float (7 bits of significand), so a product with the checkpoint rounds
// nothing that a product with the unpacked matrix would not.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "gemm_launch.hpp"
#include "half_gemm.hpp"
#include "lowrank.hpp"

namespace eigamd {

namespace {

// Limits of a type: smallest exponent of a scale (f16: its subnormals are whole multiples of 2^-24), and the exponent of its
// largest values, above which 127 2^e would leave the type and q stops at 63.
template <typename T> struct Range { static constexpr int low = -126, top = 127; static constexpr unsigned infinity = 0x7f80; };
template <> struct Range<F16> { static constexpr int low = -24, top = 15; static constexpr unsigned infinity = 0x7c00; };
template <> struct Range<Fp32> { static constexpr int low = -126, top = 127; static constexpr unsigned infinity = 0x7f800000; };

// Largest magnitude of 8 values, as the type's bits without the sign: their order is that of the magnitudes, and everything that
// is not finite is at or above infinity's.
template <typename T> __device__ __forceinline__ unsigned largest_bits(typename T::x8 v) {
  if constexpr (T::bytes == 2) {
    using u16x2 = uint16_t __attribute__((ext_vector_type(2)));
    using u16x8 = uint16_t __attribute__((ext_vector_type(8)));
    const u16x8 b = __builtin_bit_cast(u16x8, v) & (uint16_t)0x7fff;
    u16x2 m = __builtin_elementwise_max(__builtin_elementwise_max(b.s01, b.s23), __builtin_elementwise_max(b.s45, b.s67));
    return m.x > m.y ? m.x : m.y;
  } else {
    unsigned m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const unsigned b = __float_as_uint(v[i]) & 0x7fffffff;
      m = m > b ? m : b;
    }
    return m;
  }
}
template <typename T> __device__ __forceinline__ float value_of_bits(unsigned b) {
  if constexpr (T::bytes == 4) return __uint_as_float(b);
  else return (float)__builtin_bit_cast(typename T::elem, (uint16_t)b);
}

struct PackArgs {
  int k, chunks;          // features; chunks of 8 features a token takes (whole blocks of 32)
  int64_t total;          // chunks in all
  const void* x; int64_t ldx;
  int8_t* q; int64_t ldq;
  uint8_t* e; int64_t lde;
  void* out;
};

// Chunk `first` + this thread of the whole matrix; first is the workgroup's, so the 64-bit division is done once.
__device__ __forceinline__ bool chunk_of(const PackArgs& g, int64_t first, int64_t& token, int& c) {
  const int64_t t0 = first / g.chunks;
  const unsigned in = (unsigned)(first - t0 * g.chunks) + threadIdx.x;
  token = t0 + in / (unsigned)g.chunks;
  c = (int)(in % (unsigned)g.chunks);
  return first + threadIdx.x < g.total;
}

// A thread takes 8 features, four neighbours a block (`chunks` is a multiple of 4, so a block never leaves its wave), and U such
// chunks with all their loads under way at once: 4 from 2^20 chunks on, 1 below, where every chunk is wanted at once.
template <typename T, int U> __global__ __launch_bounds__(256) void ckpt8_pack_kernel(PackArgs g) {
  using E = typename T::elem;
  using x8 = typename T::x8;
  int64_t token[U];
  int c[U], n[U];
  x8 v[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    n[u] = chunk_of(g, ((int64_t)blockIdx.x * U + u) * 256, token[u], c[u]) ? g.k - c[u] * 8 : 0;
    v[u] = load_up_to_8<E, x8>(static_cast<const E*>(g.x) + token[u] * g.ldx + c[u] * 8, n[u]);
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    unsigned top = largest_bits<T>(v[u]);
    unsigned other = __shfl_xor(top, 1);
    top = top > other ? top : other;
    other = __shfl_xor(top, 2);
    top = top > other ? top : other;
    const bool flag = top >= Range<T>::infinity;
    const int bits = __float_as_int(value_of_bits<T>(top));
    int e = (bits >> 23) - 127 - ((bits & 0x7fffff) > 0x7e0000 ? 5 : 6);     // 127 = 1.984375 * 2^6
    e = e < Range<T>::low ? Range<T>::low : e;
    const float inverse = __int_as_float((127 - e) << 23);
    // x / 2^e + 1.5 * 2^23 in one rounding: its low byte is the nearest whole number, ties to even, in two's complement
    unsigned r[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = __float_as_uint(__builtin_fmaf((float)v[u][i], inverse, 12582912.0f));
    if (e > Range<T>::top - 6) {      // 64 * 2^e is no finite number of the type
#pragma unroll
      for (int i = 0; i < 8; ++i) r[i] = __float_as_uint(fminf(fmaxf(__uint_as_float(r[i]), 12582912.0f - 63.0f), 12582912.0f + 63.0f));
    }
    // bytes 0 of four words into one
    auto pack = [](unsigned a, unsigned b, unsigned cc, unsigned d) {
      return __builtin_amdgcn_perm(__builtin_amdgcn_perm(d, cc, 0x0c0c0400u), __builtin_amdgcn_perm(b, a, 0x0c0c0400u), 0x05040100u);
    };
    const uint64_t q = flag ? 0ull : (uint64_t)pack(r[4], r[5], r[6], r[7]) << 32 | pack(r[0], r[1], r[2], r[3]);
    int8_t* to = g.q + token[u] * g.ldq + c[u] * 8;
    if (n[u] >= 8) {
      __builtin_memcpy(to, &q, 8);
    } else {
      for (int i = 0; i < 8; ++i)
        if (i < n[u]) to[i] = (int8_t)(q >> (8 * i));
    }
    if (n[u] > 0 && c[u] % 4 == 0) g.e[token[u] * g.lde + c[u] / 4] = (uint8_t)(flag ? 255 : e + 127);
  }
}

template <typename T, int U> __global__ __launch_bounds__(256) void ckpt8_unpack_kernel(PackArgs g) {
  using E = typename T::elem;
  using x8 = typename T::x8;
  int64_t token[U];
  int c[U], n[U];
  uint64_t q[U];
  unsigned e[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    n[u] = chunk_of(g, ((int64_t)blockIdx.x * U + u) * 256, token[u], c[u]) ? g.k - c[u] * 8 : 0;
    q[u] = load_bytes(g.q + token[u] * g.ldq + c[u] * 8, n[u]);
    e[u] = n[u] > 0 ? g.e[token[u] * g.lde + c[u] / 4] : 0u;
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const x8 v = unpack_8<T>(q[u], exponent_scale(e[u]));
    E* to = static_cast<E*>(g.out) + token[u] * g.ldx + c[u] * 8;
    if (n[u] >= 8) {
      __builtin_memcpy(to, &v, sizeof v);
    } else {
      for (int i = 0; i < 8; ++i)
        if (i < n[u]) to[i] = v[i];
    }
  }
}

template <typename T> void launch_pack(const PackArgs& g, hipStream_t s) {
  if (g.total >= 1 << 20) hipLaunchKernelGGL((ckpt8_pack_kernel<T, 4>), dim3((unsigned)((g.total + 1023) / 1024)), dim3(256), 0, s, g);
  else hipLaunchKernelGGL((ckpt8_pack_kernel<T, 1>), dim3((unsigned)((g.total + 255) / 256)), dim3(256), 0, s, g);
}
template <typename T> void launch_unpack(const PackArgs& g, hipStream_t s) {
  if (g.total >= 1 << 20) hipLaunchKernelGGL((ckpt8_unpack_kernel<T, 4>), dim3((unsigned)((g.total + 1023) / 1024)), dim3(256), 0, s, g);
  else hipLaunchKernelGGL((ckpt8_unpack_kernel<T, 1>), dim3((unsigned)((g.total + 255) / 256)), dim3(256), 0, s, g);
}

PackArgs pack_args(int64_t k, int64_t n) {
  PackArgs g = {};
  g.k = (int)k;
  g.chunks = (int)((k + 31) / 32 * 4);
  g.total = n * g.chunks;
  return g;
}

template <typename T, int OUT, int B, int WM, int WN, int D> hipError_t launch_tiles(const HalfGemm& g, hipStream_t s) {
  const dim3 grid((unsigned)(((g.m + B - 1) / B) * (((int64_t)g.n + B - 1) / B)), g.splits);
  hipLaunchKernelGGL((half_gemm_kernel<T, MC, MC, OUT, B, B, WM, WN, D>), grid, dim3(WM * WN * 64), 0, s, g);
  return hipGetLastError();
}
template <typename T, int OUT> hipError_t launch_out(const HalfGemm& g, int tile, hipStream_t s) {
  return tile == TILE_256   ? launch_tiles<T, OUT, 256, 2, 4, 2>(g, s)
         : tile == TILE_128 ? launch_tiles<T, OUT, 128, 2, 2, 2>(g, s)
                            : launch_tiles<T, OUT, 128, 2, 4, 4>(g, s);
}
int64_t sums_bytes(int64_t m, int64_t n, int64_t k) {
  const int splits = plan_tiles(k, m, n).splits;
  return splits > 1 ? (splits * m * k * 4 + 255) / 256 * 256 : 0;
}

}  // namespace

hipError_t ckpt8_pack_device(int kind, int64_t k, int64_t n, const void* x, int64_t ldx, int8_t* q, int64_t ldq, uint8_t* e,
                             int64_t lde, hipStream_t s) {
  PackArgs g = pack_args(k, n);
  g.x = x; g.ldx = ldx; g.q = q; g.ldq = ldq; g.e = e; g.lde = lde;
  if (kind == BF16) launch_pack<Bf16>(g, s);
  else if (kind == F16K) launch_pack<F16>(g, s);
  else launch_pack<Fp32>(g, s);
  return hipGetLastError();
}

hipError_t ckpt8_unpack_device(int kind, int64_t k, int64_t n, const int8_t* q, int64_t ldq, const uint8_t* e, int64_t lde,
                               void* x, int64_t ldx, hipStream_t s) {
  PackArgs g = pack_args(k, n);
  g.out = x; g.ldx = ldx; g.q = const_cast<int8_t*>(q); g.ldq = ldq; g.e = const_cast<uint8_t*>(e); g.lde = lde;
  if (kind == BF16) launch_unpack<Bf16>(g, s);
  else if (kind == F16K) launch_unpack<F16>(g, s);
  else launch_unpack<Fp32>(g, s);
  return hipGetLastError();
}

int64_t ckpt8_grad_work_bytes(int kind, int64_t m, int64_t n, int64_t k, const void* dy, int64_t lddy) {
  if (m <= 0 || n <= 0 || k <= 0) return 0;
  if (kind == F32) return (k * n * 4 + 255) / 256 * 256 + std::min<int64_t>(16 * m * k * 4, (int64_t)256 << 20);
  return sums_bytes(m, n, k) + padded_bytes(k, n) + (whole_chunks(dy, lddy, m) ? 0 : padded_bytes(m, n));
}

hipError_t ckpt8_grad_device(const Ckpt8GradArgs& c, hipStream_t s) {
  if (c.kind == F32) {
    // unpacked once, then the library's own product
    float* x = static_cast<float*>(c.work);
    hipError_t e = c.n > 0 ? ckpt8_unpack_device(F32, c.k, c.n, c.q, c.ldq, c.e, c.lde, x, c.k, s) : hipSuccess;
    if (e != hipSuccess) return e;
    GemmCall q;
    q.kind = F32;
    q.m = c.trans ? c.k : c.m; q.n = c.trans ? c.m : c.k; q.k = c.n;
    q.opa = OP_N; q.opb = OP_T;
    q.alpha[0] = 1.0; q.alpha[1] = 0.0; q.beta[0] = c.beta; q.beta[1] = 0.0;
    q.A = c.trans ? x : c.dy; q.lda = c.trans ? c.k : c.lddy;
    q.B = c.trans ? c.dy : x; q.ldb = c.trans ? c.lddy : c.k;
    q.C = c.dw; q.ldc = c.lddw;
    const int64_t used = (c.k * c.n * 4 + 255) / 256 * 256;
    q.partials = c.work ? static_cast<char*>(c.work) + used : static_cast<void*>(c.dw);
    q.partials_bytes = c.work && c.work_bytes > used ? (size_t)(c.work_bytes - used) : 0;
    return launch_gemm_f32(q, s);
  }
  // The checkpoint is unpacked into scratch memory once, and the product reads that.  Unpacking inside the product (every tile's
  // chunks through registers) kept its loads from going to LDS directly and cost more than the extra pass: 16384 tokens x 4096 x
  // 4096 took 520 us so, 465 now, 34 of them unpacking.
  char* work = static_cast<char*>(c.work);
  const int64_t sums = sums_bytes(c.m, c.n, c.k);
  HalfGemm g;
  g.m = (int)c.k; g.n = (int)c.m; g.k = (int)c.n;
  g.a = work + sums; g.lda = padded(c.k);
  g.b = c.dy; g.ldb = c.lddy;
  g.c = c.dw; g.ldc = c.lddw;
  g.beta = c.beta;
  g.partial = reinterpret_cast<float*>(work);
  const TilePlan plan = plan_tiles(c.k, c.m, c.n);
  g.splits = plan.splits;
  g.k_piece = (int)plan.k_piece;
  hipError_t e;
  if (c.n > 0) {
    if ((e = ckpt8_unpack_device(c.kind, c.k, c.n, c.q, c.ldq, c.e, c.lde, work + sums, g.lda, s)) != hipSuccess) return e;
    if (!whole_chunks(c.dy, c.lddy, c.m)) {
      const PadCopy copy = pad_copy(c.dy, c.lddy, c.m, c.n, work + sums + padded_bytes(c.k, c.n));
      g.b = copy.to;
      g.ldb = padded(c.m);
      if ((e = launch_pad_copy(copy, {}, s)) != hipSuccess) return e;
    }
  }
  if (c.kind == BF16) e = c.trans ? launch_out<Bf16, OUT_F32>(g, plan.tile, s) : launch_out<Bf16, OUT_F32_SWAPPED>(g, plan.tile, s);
  else e = c.trans ? launch_out<F16, OUT_F32>(g, plan.tile, s) : launch_out<F16, OUT_F32_SWAPPED>(g, plan.tile, s);
  if (e != hipSuccess || g.splits == 1) return e;
  return launch_half_join(g.partial, g.splits, (int)(c.trans ? c.k : c.m), c.m * c.k, c.beta, c.dw, c.lddw, (const int*)nullptr, s);
}

}  // namespace eigamd
