// Tiled product of 16-bit matrices with 32-bit sums, on the matrix units: C (M x N, column-major) from op(A) (M x K) and
// B (K x N), the core of the adapter product (lora.hip) and of the weight gradient from a checkpoint (ckpt8.hip).
//
// A workgroup owns a BM x BN tile of C; every 64-deep slice of the two operands goes through LDS, one slice ahead of the
// products.  Both orientations of an operand keep their order in memory in LDS:
//   KC  the reduction is contiguous: a row of the slice is 128 bytes, read as 16-byte fragments;
//   MC  the rows (columns of B) are contiguous: fragments come from the transposing LDS read, 4 elements at a time.
// LDS is filled in order of address (the direct loads can do nothing else), so bank conflicts are avoided by permuting
// which 16-byte chunk of a line goes where: the lanes that read together then touch all 64 banks once.
#pragma once
#include "half.hpp"

namespace eigamd {

enum { KC = 0, MC = 1 };                       // orientation
enum { DIRECT = 0, STAGED = 1, QUANT = 2 };    // global -> LDS by hardware / through registers, any alignment / from 8 bits

struct HalfGemm {
  int m, n, k;
  const void* a;
  int64_t lda;
  const void* b;
  int64_t ldb;
  void* c;
  int64_t ldc;
  const int* order = nullptr;   // column j of B and C is column order[j] of the stored matrices
  // exponents of an 8-bit operand, one per 32 features (its contiguous direction)
  const uint8_t* exponents = nullptr;
  int64_t lde = 0;
  // adapters: column j belongs to seg[j] (`none`: no adapter)
  const int* seg = nullptr;
  int none = 0, rank = 0;
  const void* up = nullptr;
  int64_t up_row = 0, up_rank = 0, up_stride = 0;   // strides of up_j(row, r) and of j, in elements
  const float* p = nullptr;
  int64_t ldp = 0;
  const float* scale = nullptr;
  float beta = 0.0f;
  // split reduction: piece z of `splits` covers k_piece positions and leaves its sums at partial + z * m * n
  int splits = 1, k_piece = 0;
  float* partial = nullptr;
};

// 64 zero bytes that out-of-range chunks are loaded from.
static __device__ __align__(64) unsigned char zero_page[64];

// One operand's slice of R rows x 64 positions, loaded by NT threads in chunks of 8 elements; NT * N chunks in all.
template <typename T, int LAY, int SRC, int R, int NT> struct SliceLoader {
  static_assert(LAY == KC || R >= 128, "the permutation of a line needs 16 chunks");
  static constexpr int N = R * 8 / NT;
  static constexpr int bytes = R * 128;
  using E = typename T::elem;
  using x8 = typename T::x8;
  const char* ptr[N];      // this thread's chunks at position k0 = 0
  int pos[N];              // KC: first position of the chunk inside the slice; MC: its line
  int len[N];              // MC: elements of the chunk inside the matrix (0..8); KC: 8 inside, 0 outside
  int64_t step;            // bytes from one slice to the next
  const uint8_t* exps[N];
  int64_t estep;
  x8 reg[N];
  uint64_t qreg[N];
  unsigned ereg[N];

  static __device__ __forceinline__ int swizzle(int line) {
    // KC: rows 0..7 of an 8-lane phase; MC: lines {0..3, 8..11} (+4, +16) of a half wave, 32 bytes each
    return LAY == KC ? (line & 7) : (((line & 3) | ((line >> 1) & 4)) << 1);
  }

  __device__ __forceinline__ void init(const void* base, int64_t ld, int row0, int rows, int k0, const int* order, const uint8_t* e, int64_t lde) {
    constexpr int es = SRC == QUANT ? 1 : 2;
    step = (LAY == KC ? 64 : 64 * ld) * es;
    estep = 64 * lde;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int ch = threadIdx.x + i * NT;
      if constexpr (LAY == KC) {
        const int line = ch / 8, c = (ch % 8) ^ swizzle(line);
        int row = row0 + line;
        len[i] = row < rows ? 8 : 0;
        row = row < rows ? row : rows - 1;
        const int64_t at = order ? order[row] : row;
        pos[i] = c * 8;
        ptr[i] = static_cast<const char*>(base) + (at * ld + k0 + c * 8) * es;
      } else {
        const int line = ch / (R / 8), c = (ch % (R / 8)) ^ swizzle(line);
        const int row = row0 + c * 8;
        len[i] = rows - row < 0 ? 0 : (rows - row < 8 ? rows - row : 8);
        pos[i] = line;
        ptr[i] = static_cast<const char*>(base) + ((int64_t)(k0 + line) * ld + row) * es;
        if constexpr (SRC == QUANT) exps[i] = e + (int64_t)(k0 + line) * lde + row / 32;
      }
    }
  }

  // Chunks of the slice `s` slices further on, of which `left` positions are inside the reduction.
  __device__ __forceinline__ void load(char* lds, int s, int left) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const char* q = ptr[i] + (int64_t)s * step;
      const int n = LAY == KC ? (len[i] ? left - pos[i] : 0) : (pos[i] < left ? len[i] : 0);
      if constexpr (SRC == DIRECT) {
        // whole chunks only (the launcher checks extents); outside: zeros
        const char* from = n > 0 ? q : reinterpret_cast<const char*>(zero_page);
        const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
        char* to = lds + (i * NT + wave * 64) * 16;
        __builtin_amdgcn_global_load_lds(EIGAMD_GLOBAL(from), EIGAMD_LDS(void, to), 16, 0, 0);
      } else if constexpr (SRC == STAGED) {
        reg[i] = load_up_to_8<E, x8>(reinterpret_cast<const E*>(q), n);
      } else {
        uint64_t v = 0;
        if (n >= 8) {
          __builtin_memcpy(&v, q, 8);
        } else {
          for (int t = 0; t < 8; ++t)
            if (t < n) v |= (uint64_t)(uint8_t)q[t] << (8 * t);
        }
        qreg[i] = v;
        ereg[i] = n > 0 ? exps[i][(int64_t)s * estep] : 0u;
      }
    }
  }

  // Second half of a load through registers.
  __device__ __forceinline__ void store(char* lds) {
    if constexpr (SRC == DIRECT) return;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      x8 v;
      if constexpr (SRC == STAGED) {
        v = reg[i];
      } else {
        // |q| <= 127 has 7 bits, so q * 2^e is exact in either type (the exponent is kept in the type's range by the packing)
        const float sc = exponent_scale(ereg[i]);
#pragma unroll
        for (int t = 0; t < 8; ++t) v[t] = (E)((float)(int8_t)(qreg[i] >> (8 * t)) * sc);
      }
      *reinterpret_cast<x8*>(lds + (threadIdx.x + i * NT) * 16) = v;
    }
  }

  // Fragment of rows row .. row + 15 and positions kk .. kk + 31 of a slice in LDS.
  static __device__ __forceinline__ x8 fragment(const char* lds, int row, int kk) {
    const int l = threadIdx.x & 63;
    if constexpr (LAY == KC) {
      const int line = row + (l & 15), c = (kk / 8 + l / 16) ^ swizzle(line);
      return *reinterpret_cast<const x8*>(lds + line * 128 + c * 16);
    } else {
      union { x8 v; typename T::x4 h[2]; } f;
      const int line = kk + (l / 16) * 8 + (l & 15) / 4;
      const int at = row / 8 + (l & 3) / 2;          // 16-byte chunk
#pragma unroll
      for (int h = 0; h < 2; ++h)
        f.h[h] = T::read_transposed(lds + (line + 4 * h) * (R * 2) + ((at ^ swizzle(line + 4 * h)) * 16) + (l & 1) * 8);
      return f.v;
    }
  }
};

// Adds s_j up_j P to a wave's sums: column by column of the batch, only where the column belongs to j (an infinity or NaN in
// one adapter's factor must not reach another request's column, so the products are selected, not multiplied by zero).
// P has 32 bits and goes through the matrix unit as two 16-bit pieces per value, normalised per token and 32 ranks: 16 bits
// of it (bf16) or 22 (f16) take part, more than the result's type keeps.
template <typename T, int NI, int NJ>
__device__ __forceinline__ void add_adapters(const HalfGemm& g, int row0, int col0, f32x4 (&acc)[NI][NJ]) {
  using E = typename T::elem;
  using x8 = typename T::x8;
  const int l = threadIdx.x & 63;
  const int col = col0 + l;
  const int mine = l < NJ * 16 && col < g.n ? g.seg[col] : g.none;
  unsigned long long left = __ballot(mine != g.none);
  int64_t token[NJ];
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    const int c = col0 + j * 16 + (l & 15);
    token[j] = c < g.n ? g.order[c] : 0;
  }
  while (left) {
    const int first = __builtin_ctzll(left);
    const int who = __builtin_amdgcn_readlane(mine, first);
    const unsigned long long mask = __ballot(mine == who);
    left &= ~mask;
    const E* up = static_cast<const E*>(g.up) + (int64_t)who * g.up_stride;
    const float s = g.scale[who];
    for (int r0 = 0; r0 < g.rank; r0 += 32) {
      const int r = r0 + (l / 16) * 8, rn = g.rank - r;
      x8 hi[NJ], lo[NJ];
      float back[NJ];
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        if (!((mask >> (j * 16)) & 0xffff)) continue;
        using f32x8 = float __attribute__((ext_vector_type(8)));
        const f32x8 v = load_up_to_8<float, f32x8>(g.p + token[j] * g.ldp + r, rn);
        float top = 0.0f;
#pragma unroll
        for (int t = 0; t < 8; ++t) top = fmaxf(top, __builtin_fabsf(v[t]));
        if constexpr (T::bytes == 4) {
          back[j] = s;
#pragma unroll
          for (int t = 0; t < 8; ++t) hi[j][t] = v[t];
        } else {
          top = fmaxf(top, __shfl_xor(top, 16));
          top = fmaxf(top, __shfl_xor(top, 32));
          const Norm nm = norm_of(top);
          back[j] = nm.up * s;
#pragma unroll
          for (int t = 0; t < 8; ++t) {
            E piece[2];
            split<T, 2>(v[t] * nm.down, piece);
            hi[j][t] = piece[0];
            lo[j][t] = piece[1];
          }
        }
      }
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        int row = row0 + i * 16 + (l & 15);
        asm("" : "+v"(row));   // addresses are made here, not kept for every row block across the loops
        x8 u;
        const E* at = up + (int64_t)row * g.up_row + (int64_t)r * g.up_rank;
        const int n = row < g.m ? rn : 0;
        if (g.up_rank == 1) {
          u = load_up_to_8<E, x8>(at, n);
        } else {
#pragma unroll
          for (int t = 0; t < 8; ++t) u[t] = t < n ? at[(int64_t)t * g.up_rank] : (E)0.0f;
        }
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
          if (!((mask >> (j * 16)) & 0xffff)) continue;
          f32x4 d = {0.0f, 0.0f, 0.0f, 0.0f};
          if constexpr (T::bytes == 2) d = T::mma(u, lo[j], d);
          d = T::mma(u, hi[j], d);
          const bool on = (mask >> (j * 16 + (l & 15))) & 1;
#pragma unroll
          for (int t = 0; t < 4; ++t) acc[i][j][t] += on ? d[t] * back[j] : 0.0f;
        }
        __builtin_amdgcn_sched_barrier(0);   // one row block's factors in registers at a time
      }
    }
  }
}

// Tiles are dealt to the 8 XCDs in contiguous runs (consecutive workgroups go round the XCDs), and a run walks groups of
// GROUP tile rows column by column, so that what an XCD holds at a time is a near-square patch of C.
template <int GROUP> __device__ __forceinline__ void tile_of(int id, int tiles_m, int tiles_n, int& tm, int& tn) {
  const int total = tiles_m * tiles_n, per = total / 8, extra = total % 8;
  const int x = id % 8, at = id / 8;
  id = x * per + (x < extra ? x : extra) + at;
  const int group = id / (GROUP * tiles_n), first = group * GROUP;
  const int rows = tiles_m - first < GROUP ? tiles_m - first : GROUP;
  const int in = id - group * GROUP * tiles_n;
  tm = first + in % rows;
  tn = in / rows;
}

enum { OUT_HALF = 0, OUT_F32 = 1, OUT_F32_SWAPPED = 2 };

// OUT_HALF: C in the operands' type, columns scattered by `order`, adapters added.
// OUT_F32: C = beta C + A B in 32 bits.  OUT_F32_SWAPPED: the same with C stored transposed (N x M column-major).
template <typename T, int LA, int SA, int LB, int SB, int OUT, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(WM * WN * 64) void half_gemm_kernel(HalfGemm g) {
  constexpr int NT = WM * WN * 64, TM = BM / WM, TN = BN / WN, NI = TM / 16, NJ = TN / 16;
  using LoadA = SliceLoader<T, LA, SA, BM, NT>;
  using LoadB = SliceLoader<T, LB, SB, BN, NT>;
  constexpr int slice = LoadA::bytes + LoadB::bytes;
  __shared__ __align__(1024) char lds[2 * slice];
  const int tiles_m = (g.m + BM - 1) / BM, tiles_n = (g.n + BN - 1) / BN;
  int tm, tn;
  tile_of<4>(blockIdx.x, tiles_m, tiles_n, tm, tn);
  const int k_begin = blockIdx.y * g.k_piece;
  const int k_count = g.k - k_begin < g.k_piece ? g.k - k_begin : g.k_piece;
  const int slices = (k_count + 63) / 64;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), l = threadIdx.x & 63;
  const int wr = (w % WM) * TM, wc = (w / WM) * TN;

  LoadA la;
  LoadB lb;
  la.init(g.a, g.lda, tm * BM, g.m, k_begin, nullptr, g.exponents, g.lde);
  lb.init(g.b, g.ldb, tn * BN, g.n, k_begin, g.order, g.exponents, g.lde);
  f32x4 acc[NI][NJ] = {};
  if (slices > 0) {
    la.load(lds, 0, k_count);
    lb.load(lds + LoadA::bytes, 0, k_count);
  }
  if constexpr (OUT == OUT_HALF) {
    if (g.rank > 0 && blockIdx.y == 0) add_adapters<T, NI, NJ>(g, tm * BM + wr, tn * BN + wc, acc);
  }
  if (slices > 0) {
    la.store(lds);
    lb.store(lds + LoadA::bytes);
  }
  __syncthreads();
  for (int s = 0; s < slices; ++s) {
    char* here = lds + (s & 1) * slice;
    char* next = lds + ((s & 1) ^ 1) * slice;
    const bool more = s + 1 < slices;
    if (more) {
      la.load(next, s + 1, k_count - (s + 1) * 64);
      lb.load(next + LoadA::bytes, s + 1, k_count - (s + 1) * 64);
    }
#pragma unroll
    for (int kk = 0; kk < 64; kk += 32) {
      typename T::x8 fa[NI], fb[NJ];
#pragma unroll
      for (int i = 0; i < NI; ++i) fa[i] = LoadA::fragment(here, wr + i * 16, kk);
#pragma unroll
      for (int j = 0; j < NJ; ++j) fb[j] = LoadB::fragment(here + LoadA::bytes, wc + j * 16, kk);
#pragma unroll
      for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int j = 0; j < NJ; ++j)
          acc[i][j] = OUT == OUT_F32_SWAPPED ? T::mma(fb[j], fa[i], acc[i][j]) : T::mma(fa[i], fb[j], acc[i][j]);
    }
    if (more) {
      la.store(next);
      lb.store(next + LoadA::bytes);
    }
    __syncthreads();
  }

  const int row0 = tm * BM + wr, col0 = tn * BN + wc;
  if (g.splits > 1) {
    // sums of this piece, in C's own order; joined by a second kernel in the order of the pieces
    float* out = g.partial + (int64_t)blockIdx.y * g.m * g.n;
    const int64_t ld = OUT == OUT_F32_SWAPPED ? g.n : g.m;
    const int rows = OUT == OUT_F32_SWAPPED ? g.n : g.m, cols = OUT == OUT_F32_SWAPPED ? g.m : g.n;
    const bool wide = ld % 4 == 0;
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        const int r = (OUT == OUT_F32_SWAPPED ? col0 + j * 16 : row0 + i * 16) + (l / 16) * 4;
        const int c = (OUT == OUT_F32_SWAPPED ? row0 + i * 16 : col0 + j * 16) + (l & 15);
        if (c >= cols) continue;
        float* at = out + (int64_t)c * ld + r;
        if (wide && r < rows) *reinterpret_cast<f32x4*>(at) = acc[i][j];
        else
          for (int t = 0; t < 4; ++t)
            if (r + t < rows) at[t] = acc[i][j][t];
      }
    return;
  }
  if constexpr (OUT == OUT_HALF) {
    // through LDS (the slices are done with; every wave stays in its own part): whole lines of C per store
    using E = typename T::elem;
    constexpr int line = TM * 2 + 16;
    static_assert(16 * line * WM * WN <= 2 * slice, "the epilogue's part of LDS");
    char* mine = lds + w * 16 * line;
    E* C = static_cast<E*>(g.c);
    const bool wide = (reinterpret_cast<uintptr_t>(C) & 15) == 0 && g.ldc % 8 == 0;
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        typename T::x4 v;
#pragma unroll
        for (int t = 0; t < 4; ++t) v[t] = (E)acc[i][j][t];
        *reinterpret_cast<typename T::x4*>(mine + (l & 15) * line + (i * 16 + (l / 16) * 4) * 2) = v;
      }
      __builtin_amdgcn_wave_barrier();
      constexpr int per = TM / 8;                    // 16-byte chunks of a column
#pragma unroll
      for (int q = 0; q < 16 * per / 64; ++q) {
        const int ch = q * 64 + l, cj = ch / per, r = row0 + (ch % per) * 8, c = col0 + j * 16 + cj;
        const typename T::x8 v = *reinterpret_cast<const typename T::x8*>(mine + cj * line + (ch % per) * 16);
        if (c >= g.n) continue;
        E* at = C + (int64_t)(g.order ? g.order[c] : c) * g.ldc + r;
        if (wide && r + 8 <= g.m) *reinterpret_cast<typename T::x8*>(at) = v;
        else
          for (int t = 0; t < 8; ++t)
            if (r + t < g.m) at[t] = v[t];
      }
      __builtin_amdgcn_wave_barrier();
    }
  } else {
    float* C = static_cast<float*>(g.c);
    const int rows = OUT == OUT_F32_SWAPPED ? g.n : g.m, cols = OUT == OUT_F32_SWAPPED ? g.m : g.n;
    const bool wide = (reinterpret_cast<uintptr_t>(C) & 15) == 0 && g.ldc % 4 == 0;
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        const int r = (OUT == OUT_F32_SWAPPED ? col0 + j * 16 : row0 + i * 16) + (l / 16) * 4;
        const int c = (OUT == OUT_F32_SWAPPED ? row0 + i * 16 : col0 + j * 16) + (l & 15);
        if (c >= cols) continue;
        float* at = C + (int64_t)c * g.ldc + r;
        f32x4 v = acc[i][j];
        if (wide && r + 4 <= rows) {
          if (g.beta != 0.0f) v += g.beta * *reinterpret_cast<const f32x4*>(at);
          *reinterpret_cast<f32x4*>(at) = v;
        } else {
          for (int t = 0; t < 4; ++t)
            if (r + t < rows) at[t] = v[t] + (g.beta != 0.0f ? g.beta * at[t] : 0.0f);
        }
      }
  }
}

}  // namespace eigamd
