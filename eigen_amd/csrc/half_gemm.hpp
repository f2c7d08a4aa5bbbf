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
#include <type_traits>

#include "half.hpp"

namespace eigamd {

enum { KC = 0, MC = 1 };                       // orientation

struct HalfGemm {
  int m, n, k;
  const void* a;
  int64_t lda;
  const void* b;
  int64_t ldb;
  void* c;
  int64_t ldc;
  const int* order = nullptr;   // column j of B and C is column order[j] of the stored matrices
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

// Global memory to LDS without passing through registers: lane l's 16 bytes land at `to` + 16 l (`to` the same in every lane).
// In assembly, because the compiler would wait for every such load before the next read of any LDS; it is waited for, with
// everything else, in slice_barrier().  M0 holds the LDS address.  The second form takes a base that is the same in every lane.
__device__ __forceinline__ void load_to_lds(const char* from, char* to) {
  const unsigned at = __builtin_amdgcn_readfirstlane((unsigned)(uintptr_t)EIGAMD_LDS(char, to));
  asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"{m0}"(at), "v"(from) : "memory");
}
__device__ __forceinline__ void load_to_lds(const char* base, unsigned off, char* to) {
  const unsigned at = __builtin_amdgcn_readfirstlane((unsigned)(uintptr_t)EIGAMD_LDS(char, to));
  asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"{m0}"(at), "v"(off), "s"(base) : "memory");
}
// This wave's LDS accesses and all but its newest KEEP loads are done, then those of the workgroup.
template <int KEEP> __device__ __forceinline__ void slice_barrier() {
  static_assert(KEEP < 64, "six bits of vmcnt");
  asm volatile("" ::: "memory");
  // vmcnt(KEEP) lgkmcnt(0), in a form the compiler's own counting sees
  __builtin_amdgcn_s_waitcnt(0x70 | (KEEP & 15) | (KEEP >> 4) << 14);
  asm volatile("s_barrier" ::: "memory");
}

// One operand's slice of R rows x 64 positions, loaded by NT threads in chunks of 8 elements; NT * N chunks in all.  Slices are
// taken one after the other.
// Rows past the end are not cleared: whatever stands there meets only rows of C that are not stored.  Positions past the end of
// the reduction are zero in both operands.
// GATHER: row i is row order[i] of the matrix, and every chunk has an address of its own; otherwise they are 32-bit offsets from
// a base that is the same in all lanes (256 rows or 64 lines of at most kMaxLine elements each: below 2^31 bytes).
template <typename T, int LAY, int R, int NT, bool GATHER> struct SliceLoader {
  static_assert(LAY == KC || (R >= 128 && !GATHER), "the permutation of a line needs 16 chunks");
  static constexpr int N = R * 8 / NT;
  static constexpr int bytes = R * 128;
  static constexpr int NOFF = GATHER ? 1 : LAY == KC ? N : 1, NPTR = GATHER ? N : 1;
  static constexpr int lines = NT / (R / 8);     // MC: lines from one chunk of a thread to the next
  using x8 = typename T::x8;
  const char* base;        // first position of the next slice
  int64_t step;            // bytes from one slice to the next
  int64_t across;          // MC: bytes from one chunk of a thread to the next
  unsigned off[NOFF];
  const char* ptr[NPTR];
  int left;                // positions from the next slice's first to the end of the reduction

  static __device__ __forceinline__ int swizzle(int line) {
    // KC: rows 0..7 of an 8-lane phase; MC: lines {0..3, 8..11} (+4, +16) of a half wave, 32 bytes each
    return LAY == KC ? (line & 7) : (((line & 3) | ((line >> 1) & 4)) << 1);
  }
  // position inside the slice of chunk i: KC its first (the same for all i), MC its line
  static __device__ __forceinline__ int position(int i) {
    const int t = threadIdx.x;
    return LAY == KC ? ((t % 8) ^ swizzle(t / 8)) * 8 : t / (R / 8) + i * lines;
  }

  __device__ __forceinline__ void init(const void* origin, int64_t ld, int row0, int rows, int k0, int count, const int* order) {
    step = (LAY == KC ? 64 : 64 * ld) * 2;
    left = count;
    base = static_cast<const char*>(origin);
    if constexpr (LAY == KC) {
      base += ((GATHER ? 0 : row0 * ld) + k0) * 2;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int line = threadIdx.x / 8 + i * (NT / 8);
        const int in = row0 + line < rows ? line : rows - 1 - row0;
        if constexpr (GATHER) ptr[i] = base + ((int64_t)order[row0 + in] * ld + position(0)) * 2;
        else off[i] = (unsigned)((in * ld + position(0)) * 2);
      }
    } else {
      const int line = position(0), c = (threadIdx.x % (R / 8)) ^ swizzle(line);
      base += (k0 * ld + row0) * 2;
      across = lines * ld * 2;
      off[0] = (unsigned)((line * ld + (row0 + c * 8 < rows ? c * 8 : 0)) * 2);
    }
  }
  __device__ __forceinline__ const char* at(int i) const {
    if constexpr (GATHER) return ptr[i];
    else return LAY == KC ? base + off[i] : base + i * across + off[0];
  }
  // Chunk i of a slice that is whole; next() behind the last one.
  __device__ __forceinline__ void send(char* lds, int i) {
    char* to = lds + __builtin_amdgcn_readfirstlane(threadIdx.x / 64) * 1024 + i * NT * 16;
    if constexpr (GATHER) load_to_lds(ptr[i], to);
    else if constexpr (LAY == KC) load_to_lds(base, off[i], to);
    else load_to_lds(base + i * across, off[0], to);
  }
  __device__ __forceinline__ void next() {
    left -= 64;
    base += step;
    if constexpr (GATHER) {
#pragma unroll
      for (int i = 0; i < N; ++i) ptr[i] += step;
    }
  }
  // The next slice, if there is one.
  __device__ __forceinline__ void commit(char* lds) {
    if (left <= 0) return;
    if (left >= 64) {
#pragma unroll
      for (int i = 0; i < N; ++i) send(lds, i);
    } else {
      // Whole chunks (the launcher sees to that; one that the reduction ends in has zeros behind its end); those outside: zeros.
      char* to = lds + __builtin_amdgcn_readfirstlane(threadIdx.x / 64) * 1024;
#pragma unroll
      for (int i = 0; i < N; ++i)
        load_to_lds((LAY == KC ? position(0) : position(i)) < left ? at(i) : reinterpret_cast<const char*>(zero_page), to + i * NT * 16);
    }
    next();
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

// A bit for each of the 16 columns that a wave's lanes hold: one of the column's four lanes says so.
__device__ __forceinline__ unsigned long long by_column(bool say) {
  unsigned long long b = __ballot(say);
  b |= b >> 32;
  b |= b >> 16;
  return b & 0xffff;
}

// Adds s_j up_j P to a wave's sums: column by column of the batch, only where the column belongs to j (an infinity or NaN in
// one adapter's factor must not reach another request's column, so the products are selected, not multiplied by zero).
// P goes through the matrix unit as three 16-bit pieces per value, which hold all of its 32 bits.  f16 has not P's range: there it is
// normalised per token and 32 ranks, and the second and third piece are 2^10 times as large and summed up apart.  Columns with a P below
// about 2^-26 of that largest are left to adapters_in_single (`again`, a bit a column).
// Per 32 ranks, P's fragments do not depend on the adapter; of the adapters' factors the next one's are under way while one is
// multiplied.
template <typename T, int NI, int NJ>
__device__ __forceinline__ void adapters_in_pieces(const HalfGemm& g, int row0, int col0, f32x4 (&acc)[NI][NJ], unsigned long long& again) {
  using E = typename T::elem;
  using x8 = typename T::x8;
  using f32x8 = float __attribute__((ext_vector_type(8)));
  constexpr int NP = T::bytes == 4 ? 1 : 3, UP = 10;
  constexpr bool APART = __is_same(T, F16);
  const int l = threadIdx.x & 63;
  const int col = col0 + l;
  const int mine = l < NJ * 16 && col < g.n ? g.seg[col] : g.none;
  const unsigned long long live = __ballot(mine != g.none);
  if (!live) return;
  int token[NJ];
  float scale[NJ];
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    const int c = col0 + j * 16 + (l & 15);
    token[j] = c < g.n ? g.order[c] : 0;
    const int who = __shfl(mine, j * 16 + (l & 15));
    scale[j] = who != g.none ? g.scale[who] : 0.0f;
  }
  for (int r0 = 0; r0 < g.rank; r0 += 32) {
    // rows past the end repeat the last one (they are not stored); ranks past the end are zero in both operands
    const int r = r0 + (l / 16) * 8 < g.rank ? r0 + (l / 16) * 8 : 0, rn = g.rank - r0 - (l / 16) * 8;
    const bool chunks = g.rank % 8 == 0;
    auto factor = [&](int who, int i) {
      int row = row0 + i * 16 + (l & 15);
      asm("" : "+v"(row));   // addresses are made here, not kept for every row block across the loops
      row = row < g.m ? row : g.m - 1;
      const E* at = static_cast<const E*>(g.up) + (int64_t)who * g.up_stride + (int64_t)row * g.up_row + (int64_t)r * g.up_rank;
      if (!chunks || g.up_rank != 1) return load_first<E, x8>(at, g.up_rank, rn);
      x8 u = load_8<E, x8>(at);
#pragma unroll
      for (int t = 0; t < 8; ++t) u[t] = rn > 0 ? u[t] : (E)0.0f;
      return u;
    };
    x8 part[NP][NJ];
    float back[NJ];
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      const float* at = g.p + (int64_t)token[j] * g.ldp + r;
      f32x8 v = chunks ? load_8<float, f32x8>(at) : load_first<float, f32x8>(at, 1, rn);
#pragma unroll
      for (int t = 0; t < 8; ++t) v[t] = rn > 0 ? v[t] : 0.0f;
      back[j] = scale[j];
      if constexpr (APART) {
        // (one that is infinite leaves nothing finite in its column)
        float top = largest_of(v);
        top = fmaxf(top, __shfl_xor(top, 16));
        top = fmaxf(top, __shfl_xor(top, 32));
        const Norm nm = norm_of(top);
        back[j] *= nm.up;
        again |= by_column(some_below(v, smallest_f16<UP>() * nm.up)) << (j * 16);
#pragma unroll
        for (int t = 0; t < 8; ++t) v[t] *= nm.down;
      }
#pragma unroll
      for (int t = 0; t < 8; ++t) {
        if constexpr (NP == 1) {
          part[0][j][t] = v[t];
        } else {
          E piece[NP];
          if constexpr (APART) split_f16<UP>(v[t], piece);
          else split_bf16(v[t], piece);
#pragma unroll
          for (int z = 0; z < NP; ++z) part[z][j][t] = piece[z];
        }
      }
    }
    // Four row blocks' factors under way together, two in the large tile, which has no registers for more; those of the next adapter while
    // this one's are multiplied, if they are all.
    constexpr int GI = NI < 4 ? NI : NI == 4 ? 4 : 2;
    constexpr bool AHEAD = NI == GI;
    unsigned long long left = live;
    int who = __builtin_amdgcn_readlane(mine, __builtin_ctzll(left));
    x8 u[GI];
    if constexpr (AHEAD) {
#pragma unroll
      for (int i = 0; i < GI; ++i) u[i] = factor(who, i);
    }
    while (true) {
      const unsigned long long mask = __ballot(mine == who);
      left &= ~mask;
      const bool more = left != 0;
      const int next = more ? __builtin_amdgcn_readlane(mine, __builtin_ctzll(left)) : who;
#pragma unroll
      for (int i0 = 0; i0 < NI; i0 += GI) {
        if constexpr (!AHEAD) {
#pragma unroll
          for (int i = 0; i < GI; ++i) u[i] = factor(who, i0 + i);
        }
#pragma unroll
        for (int i = 0; i < GI; ++i) {
#pragma unroll
          for (int j = 0; j < NJ; ++j) {
            if (!((mask >> (j * 16)) & 0xffff)) continue;
            f32x4 d = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int z = NP - 1; z >= 0; --z) {
              if (APART && z == 0) d *= 1.0f / (float)(1 << UP);
              d = T::mma(u[i], part[z][j], d);
            }
            const bool on = (mask >> (j * 16 + (l & 15))) & 1;
#pragma unroll
            for (int t = 0; t < 4; ++t) acc[i0 + i][j][t] += on ? d[t] * back[j] : 0.0f;
          }
          if (AHEAD && more) u[i] = factor(next, i);
        }
      }
      if (!more) break;
      who = next;
    }
  }
}

// The same in single precision for some of the columns, one block after the other: few registers beside the sums (and no addresses kept
// for the blocks).
template <typename T, int NI, int NJ>
__device__ __forceinline__ void adapters_in_single(const HalfGemm& g, int row0, int col0, unsigned long long columns, f32x4 (&acc)[NI][NJ]) {
  using E = typename T::elem;
  const int l = threadIdx.x & 63;
  const int mine = l < NJ * 16 && col0 + l < g.n ? g.seg[col0 + l] : g.none;
  unsigned long long left = __ballot(mine != g.none) & columns;
  while (left) {
    const int who = __builtin_amdgcn_readlane(mine, __builtin_ctzll(left));
    const unsigned long long mask = __ballot(mine == who) & columns;
    left &= ~mask;
    const float scale = g.scale[who];
    const E* factor = static_cast<const E*>(g.up) + (int64_t)who * g.up_stride;
    for (int r0 = 0; r0 < g.rank; r0 += 32) {
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
#pragma unroll
        for (int i = 0; i < NI; ++i) {
          int lane = l;
          asm volatile("" : "+v"(lane));
          const int r = r0 + (lane / 16) * 8 < g.rank ? r0 + (lane / 16) * 8 : 0, rn = g.rank - r0 - (lane / 16) * 8;
          const int c = col0 + j * 16 + (lane & 15), row = row0 + i * 16 + (lane & 15);
          const Fp32::x8 p = load_first<float, Fp32::x8>(g.p + (int64_t)g.order[c < g.n ? c : g.n - 1] * g.ldp + r, 1, rn);
          const typename T::x8 u = load_first<E, typename T::x8>(factor + (int64_t)(row < g.m ? row : g.m - 1) * g.up_row + (int64_t)r * g.up_rank, g.up_rank, rn);
          const f32x4 d = Fp32::mma(__builtin_convertvector(u, Fp32::x8), p, f32x4{0.0f, 0.0f, 0.0f, 0.0f});
          const bool on = (mask >> (j * 16 + (lane & 15))) & 1;
#pragma unroll
          for (int t = 0; t < 4; ++t) acc[i][j][t] += on ? d[t] * scale : 0.0f;
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    }
  }
}

// Into sums that are still zero.  A product of an infinity and a piece that is zero is a NaN, where the value's own product is an
// infinity: columns where a NaN has come up are done again in single precision, like those that the pieces do not hold (and only they:
// what a request gets does not depend on what stands beside it).
template <typename T, int NI, int NJ>
__device__ __forceinline__ void add_adapters(const HalfGemm& g, int row0, int col0, f32x4 (&acc)[NI][NJ]) {
  unsigned long long again = 0;
  adapters_in_pieces<T>(g, row0, col0, acc, again);
  if constexpr (T::bytes == 2) {
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      f32x4 all = acc[0][j];
#pragma unroll
      for (int i = 1; i < NI; ++i) all += acc[i][j];
      const float sum = (all[0] + all[1]) + (all[2] + all[3]);
      again |= by_column(sum != sum) << (j * 16);
    }
    if (__builtin_expect(again != 0, 0)) {
#pragma unroll
      for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int i = 0; i < NI; ++i)
#pragma unroll
          for (int t = 0; t < 4; ++t) acc[i][j][t] = (again >> (j * 16 + (threadIdx.x & 15))) & 1 ? 0.0f : acc[i][j][t];
      adapters_in_single<T>(g, row0, col0, again, acc);
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
template <typename T, int LA, int LB, int OUT, int BM, int BN, int WM, int WN, int D>
__global__ __launch_bounds__(WM * WN * 64, 2) void half_gemm_kernel(HalfGemm g) {
  constexpr int NT = WM * WN * 64, TM = BM / WM, TN = BN / WN, NI = TM / 16, NJ = TN / 16;
  using LoadA = SliceLoader<T, LA, BM, NT, false>;
  using LoadB = SliceLoader<T, LB, BN, NT, OUT == OUT_HALF>;
  constexpr int slice = LoadA::bytes + LoadB::bytes;
  __shared__ __align__(1024) char lds[D * slice];
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
  la.init(g.a, g.lda, tm * BM, g.m, k_begin, k_count, nullptr);
  lb.init(g.b, g.ldb, tn * BN, g.n, k_begin, k_count, g.order);
  f32x4 acc[NI][NJ] = {};
  // D slices in LDS.  Each half of a slice (32 positions) is multiplied in P steps of 16 rows each x 4 (all rows of this wave, or the
  // upper and the lower half); while one step's products run, the fragments of the next are read.  A slice's buffer is free once
  // its last fragments are in registers: from the barrier in front of slice s's last step on, slice s + D is on its way there;
  // slice s + 1 has to have arrived at that barrier, those behind it may still be under way.
#pragma unroll 1
  for (int z = 0; z < D; ++z) {
    la.commit(lds + z * slice);
    lb.commit(lds + z * slice + LoadA::bytes);
  }
  if constexpr (OUT == OUT_HALF) {
    if (g.rank > 0 && blockIdx.y == 0) add_adapters<T, NI, NJ>(g, tm * BM + wr, tn * BN + wc, acc);
  }
  slice_barrier<0>();
  constexpr int P = NI > 4 ? 2 : 1, NH = NI / P, RA = LA == KC ? 1 : 2, RB = LB == KC ? 1 : 2;
  typename T::x8 fa[2][NH], fb[2][NJ];
  // fragments of step q of the slice at `from`
  auto read = [&](const char* from, int q) {
    const int half = q / P, part = q % P;
#pragma unroll
    for (int i = 0; i < NH; ++i) fa[q & 1][i] = LoadA::fragment(from, wr + (part * NH + i) * 16, half * 32);
    if (part == 0) {
#pragma unroll
      for (int j = 0; j < NJ; ++j) fb[half][j] = LoadB::fragment(from + LoadA::bytes, wc + j * 16, half * 32);
    }
  };
  auto multiply = [&](int q) {
    const int half = q / P, part = q % P;
#pragma unroll
    for (int i = 0; i < NH; ++i)
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        f32x4& c = acc[part * NH + i][j];
        c = OUT == OUT_F32_SWAPPED ? T::mma(fb[half][j], fa[q & 1][i], c) : T::mma(fa[q & 1][i], fb[half][j], c);
      }
  };
  // The compiler would put each read right in front of the product that needs it; here every read of the next step is followed
  // by products of this one.
  constexpr int products = NH * NJ;
  auto interleave = [&](auto count) {
    constexpr int reads = decltype(count)::value, per = products >= 2 * reads ? products / reads / 2 : products >= reads ? 1 : 0;
#pragma unroll
    for (int q = 0; q < reads; ++q) {
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x008, per, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x008, products - reads * per, 0);
    __builtin_amdgcn_sched_barrier(0);
  };
  using ReadsA = std::integral_constant<int, NH * RA>;
  using ReadsAB = std::integral_constant<int, NH * RA + NJ * RB>;
  read(lds, 0);
  constexpr int keep = (D - 2) * (LoadA::N + LoadB::N);
  char* here = lds;
  int s = 0;
  // As long as slice s + D is whole its loads need no looking at: they go out between the products of the last step, one of
  // each operand behind every group.
  for (; la.left >= 64; ++s) {
    char* other = here + slice == lds + D * slice ? lds : here + slice;
#pragma unroll
    for (int q = 0; q + 1 < 2 * P; ++q) {
      read(here, q + 1);
      multiply(q);
      if ((q + 1) % P == 0) interleave(ReadsAB{});
      else interleave(ReadsA{});
    }
    slice_barrier<keep>();
    constexpr int G = LoadA::N > LoadB::N ? LoadA::N : LoadB::N;
#pragma unroll
    for (int q = 0; q < G; ++q) {
      if (q < LoadA::N) la.send(here, q);
      if (q < LoadB::N) lb.send(here + LoadA::bytes, q);
#pragma unroll
      for (int i = 0; i < NH; ++i)
        if (i * G / NH == q) fa[0][i] = LoadA::fragment(other, wr + i * 16, 0);
#pragma unroll
      for (int j = 0; j < NJ; ++j)
        if (j * G / NJ == q) fb[0][j] = LoadB::fragment(other + LoadA::bytes, wc + j * 16, 0);
#pragma unroll
      for (int i = 0; i < NH; ++i)
#pragma unroll
        for (int j = 0; j < NJ; ++j)
          if ((i * NJ + j) * G / products == q) {
            f32x4& c = acc[(P - 1) * NH + i][j];
            c = OUT == OUT_F32_SWAPPED ? T::mma(fb[1][j], fa[1][i], c) : T::mma(fa[1][i], fb[1][j], c);
          }
      __builtin_amdgcn_sched_barrier(0);
    }
    la.next();
    lb.next();
    here = other;
  }
  for (; s < slices; ++s) {
    char* other = here + slice == lds + D * slice ? lds : here + slice;
#pragma unroll
    for (int q = 0; q + 1 < 2 * P; ++q) {
      read(here, q + 1);
      multiply(q);
      if ((q + 1) % P == 0) interleave(ReadsAB{});
      else interleave(ReadsA{});
    }
    if (D == 2 || s + D > slices) slice_barrier<0>();
    else slice_barrier<keep>();
    la.commit(here);
    lb.commit(here + LoadA::bytes);
    read(other, 0);     // (behind the last slice: what was there before, not used)
    multiply(2 * P - 1);
    interleave(ReadsAB{});
    here = other;
  }
  slice_barrier<0>();

  // Out through LDS (the slices are done with; every wave stays in its own part), 16 of this wave's columns of C at a time, so that
  // neighbouring lanes store neighbouring rows, alignment or not.  Swapped: the tile's columns are C's rows.
  constexpr bool SWAPPED = OUT == OUT_F32_SWAPPED;
  constexpr int CR = SWAPPED ? TN : TM, CN = (SWAPPED ? TM : TN) / 16;
  const int c_row0 = SWAPPED ? tn * BN + wc : tm * BM + wr, c_col0 = SWAPPED ? tm * BM + wr : tn * BN + wc;
  const int c_rows = SWAPPED ? g.n : g.m, c_cols = SWAPPED ? g.m : g.n;
  auto block = [&](int r, int c) -> const f32x4& { return SWAPPED ? acc[c][r] : acc[r][c]; };
  if (OUT == OUT_HALF && g.splits == 1) {
    using E = typename T::elem;
    using x4 = typename T::x4;
    using x8 = typename T::x8;
    constexpr int line = CR * 2 + 16;
    static_assert(16 * line * WM * WN <= D * slice, "the epilogue's part of LDS");
    char* mine = lds + w * 16 * line;
    E* C = static_cast<E*>(g.c);
    const bool wide = (reinterpret_cast<uintptr_t>(C) & 15) == 0 && g.ldc % 8 == 0;
#pragma unroll
    for (int j = 0; j < CN; ++j) {
#pragma unroll
      for (int i = 0; i < CR / 16; ++i) {
        const f32x4& a = block(i, j);
        x4 v;
#pragma unroll
        for (int t = 0; t < 4; ++t) v[t] = (E)a[t];
        *reinterpret_cast<x4*>(mine + (l & 15) * line + (i * 16 + (l / 16) * 4) * 2) = v;
      }
      wave_order();
      if (wide) {
        constexpr int per = CR / 8;                    // 16-byte chunks of a column
#pragma unroll
        for (int q = 0; q < 16 * per / 64; ++q) {
          const int ch = q * 64 + l, c = c_col0 + j * 16 + ch / per, r = c_row0 + ch % per * 8;
          const x8 v = *reinterpret_cast<const x8*>(mine + ch / per * line + ch % per * 16);
          if (c >= c_cols) continue;
          E* at = C + (int64_t)(g.order ? g.order[c] : c) * g.ldc + r;
          if (r + 8 <= c_rows) *reinterpret_cast<x8*>(at) = v;
          else
            for (int t = 0; t < 8; ++t)
              if (r + t < c_rows) at[t] = v[t];
        }
      } else {
        for (int q = l; q < 16 * CR; q += 64) {
          const int c = c_col0 + j * 16 + q / CR, r = c_row0 + q % CR;
          const E v = *reinterpret_cast<const E*>(mine + q / CR * line + q % CR * 2);
          if (c < c_cols && r < c_rows) C[(int64_t)(g.order ? g.order[c] : c) * g.ldc + r] = v;
        }
      }
      wave_order();
    }
    return;
  }
  // 32 bits: the result, or this piece's sums in C's own order (joined by a second kernel in the order of the pieces); a lane's four
  // rows are 16 bytes of a column, four lanes 64, which go out as they are.
  const bool sums = g.splits > 1;
  float* C = sums ? g.partial + (int64_t)blockIdx.y * g.m * g.n : static_cast<float*>(g.c);
  const int64_t ldc = sums ? c_rows : g.ldc;
  const float beta = sums ? 0.0f : g.beta;
  if ((reinterpret_cast<uintptr_t>(C) & 15) == 0 && ldc % 4 == 0) {
#pragma unroll
    for (int j = 0; j < CN; ++j)
#pragma unroll
      for (int i = 0; i < CR / 16; ++i) {
        const int r = c_row0 + i * 16 + (l / 16) * 4, c = c_col0 + j * 16 + (l & 15);
        if (c >= c_cols) continue;
        float* at = C + (int64_t)c * ldc + r;
        f32x4 v = block(i, j);
        if (r + 4 <= c_rows) {
          if (beta != 0.0f) v += beta * *reinterpret_cast<const f32x4*>(at);
          *reinterpret_cast<f32x4*>(at) = v;
        } else {
          for (int t = 0; t < 4; ++t)
            if (r + t < c_rows) at[t] = v[t] + (beta != 0.0f ? beta * at[t] : 0.0f);
        }
      }
    return;
  }
  // Otherwise through LDS again.  What C held is loaded a step ahead of the stores; behind them every step waits for memory (589
  // tokens x 2840 x 3774: 68 us, now 42).
  constexpr int line = CR * 4 + 16;
  static_assert(16 * line * WM * WN <= D * slice, "the epilogue's part of LDS");
  char* mine = lds + w * 16 * line;
  constexpr int B = 8, NB = 16 * CR / 64 / B;      // values a lane takes in one step, steps of 16 columns
  static_assert(16 * CR / 64 % B == 0, "whole steps");
  float next[B] = {};
  auto place = [&](int step, int t) -> float* {
    const int q = (step % NB * B + t) * 64 + l, c = c_col0 + step / NB * 16 + q / CR, r = c_row0 + q % CR;
    return c < c_cols && r < c_rows ? C + (int64_t)c * ldc + r : nullptr;
  };
  auto fetch = [&](int step) {
#pragma unroll
    for (int t = 0; t < B; ++t) {
      const float* at = place(step, t);
      next[t] = *(at ? at : reinterpret_cast<const float*>(zero_page));
    }
  };
  if (beta != 0.0f) fetch(0);
#pragma unroll
  for (int j = 0; j < CN; ++j) {
#pragma unroll
    for (int i = 0; i < CR / 16; ++i) *reinterpret_cast<f32x4*>(mine + (l & 15) * line + (i * 16 + (l / 16) * 4) * 4) = block(i, j);
    wave_order();
#pragma unroll 1
    for (int b = 0; b < NB; ++b) {
      const int step = j * NB + b;
      float v[B];
#pragma unroll
      for (int t = 0; t < B; ++t) {
        const int q = (b * B + t) * 64 + l;
        v[t] = *reinterpret_cast<const float*>(mine + q / CR * line + q % CR * 4);
        v[t] += beta != 0.0f ? beta * next[t] : 0.0f;
      }
      if (beta != 0.0f && step + 1 < CN * NB) fetch(step + 1);
#pragma unroll
      for (int t = 0; t < B; ++t) {
        float* at = place(step, t);
        if (at) *at = v[t];
      }
    }
    wave_order();
  }
}

// The direct loads take whole, aligned 16-byte chunks at 32-bit offsets.  A matrix that has others (an odd leading dimension or one past
// kMaxLine, an extent that is no multiple of 8) is copied into scratch memory first, columns padded with zeros: reading it in place through registers took
// 378 us for 4096 tokens x 4095 x 4093, copies and product take 190 (4096 x 4096: 126).
constexpr int64_t kMaxLine = (int64_t)1 << 22;
inline bool whole_chunks(const void* p, int64_t ld, int64_t rows) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && ld % 8 == 0 && ld <= kMaxLine && rows % 8 == 0;
}
inline int64_t padded(int64_t rows) { return (rows + 7) / 8 * 8; }
inline int64_t padded_bytes(int64_t rows, int64_t cols) { return (padded(rows) * cols * 2 + 255) / 256 * 256; }
struct PadCopy {
  const uint16_t* from;
  int64_t ld;
  int rows;
  int64_t chunks;        // of 8 elements, in all; 0: nothing to copy
  uint16_t* to;
};
inline PadCopy pad_copy(const void* from, int64_t ld, int64_t rows, int64_t cols, void* to) {
  return {static_cast<const uint16_t*>(from), ld, (int)rows, padded(rows) / 8 * cols, static_cast<uint16_t*>(to)};
}
static __global__ __launch_bounds__(256) void pad_copy_kernel(PadCopy a, PadCopy b) {
  using u16x8 = uint16_t __attribute__((ext_vector_type(8)));
  for (int64_t q = (int64_t)blockIdx.x * 256 + threadIdx.x; q < a.chunks + b.chunks; q += (int64_t)gridDim.x * 256) {
    const PadCopy& m = q < a.chunks ? a : b;
    const int64_t ch = q < a.chunks ? q : q - a.chunks;
    const int per = (m.rows + 7) / 8;
    const int64_t col = ch / per;
    const int row = (int)(ch - col * per) * 8;
    const uint16_t* from = m.from + col * m.ld + row;
    u16x8 v;
    if (row + 8 <= m.rows) {
      __builtin_memcpy(&v, from, 16);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = row + i < m.rows ? from[i] : 0;
    }
    *reinterpret_cast<u16x8*>(m.to + ch * 8) = v;
  }
}
inline hipError_t launch_pad_copy(const PadCopy& a, const PadCopy& b, hipStream_t s) {
  const int64_t blocks = (a.chunks + b.chunks + 255) / 256;
  if (blocks == 0) return hipSuccess;
  hipLaunchKernelGGL(pad_copy_kernel, dim3((unsigned)(blocks < 16384 ? blocks : 16384)), dim3(256), 0, s, a, b);
  return hipGetLastError();
}

// Sums of a split reduction in the order of the pieces, four rows a thread: C = beta C + sum (C in the operands' type: beta is 0).
// `rows` is C's contiguous extent, `order` its columns' (nullptr: as they are).
template <typename E> __global__ __launch_bounds__(256) void half_join_kernel(const float* __restrict__ partial, int splits, int rows, int64_t total,
                                                                           float beta, E* __restrict__ c, int64_t ldc, const int* __restrict__ order) {
  const bool wide = rows % 4 == 0;
  const int per = wide ? 4 : 1;
  for (int64_t q = ((int64_t)blockIdx.x * 256 + threadIdx.x) * per; q < total; q += (int64_t)gridDim.x * 256 * per) {
    f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
    if (wide) {
      int z = 0;
      for (; z + 4 <= splits; z += 4) {
        f32x4 v[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) v[t] = *reinterpret_cast<const f32x4*>(partial + (int64_t)(z + t) * total + q);
#pragma unroll
        for (int t = 0; t < 4; ++t) sum += v[t];
      }
      for (; z < splits; ++z) sum += *reinterpret_cast<const f32x4*>(partial + (int64_t)z * total + q);
    } else {
      for (int z = 0; z < splits; ++z) sum[0] += partial[(int64_t)z * total + q];
    }
    const int64_t col = q / rows;
    E* at = c + (order ? order[col] : col) * ldc + (q - col * rows);
#pragma unroll
    for (int t = 0; t < 4; ++t)
      if (t < per) at[t] = (E)(sum[t] + (beta != 0.0f ? beta * (float)at[t] : 0.0f));
  }
}
template <typename E>
inline hipError_t launch_half_join(const float* partial, int splits, int rows, int64_t total, float beta, E* c, int64_t ldc, const int* order, hipStream_t s) {
  const int64_t blocks = rows % 4 == 0 ? (total + 1023) / 1024 : (total + 255) / 256;
  hipLaunchKernelGGL(half_join_kernel<E>, dim3((unsigned)(blocks < 8192 ? blocks : 8192)), dim3(256), 0, s, partial, splits, rows, total, beta, c, ldc, order);
  return hipGetLastError();
}

// Which tile, and how many pieces of the reduction.  Times of a 64-deep slice, measured with bf16 at 4096 rows and up to 4096
// columns: 1.5 us with 256 x 256 tiles; 0.86 with 128 x 128 tiles two to a compute unit, 0.72 where each has its unit to itself;
// 0.55 in the form for that (eight waves, four slices in LDS).  A round of tiles over the 256 units takes its slices and 11, 8 or
// 5 us beside them; splitting the reduction costs another launch and the traffic of the sums.
enum { TILE_256, TILE_128, TILE_128_ALONE };
struct TilePlan {
  int tile, splits;
  int64_t k_piece;
  double us;
};
inline TilePlan plan_tiles(int64_t m, int64_t n, int64_t k) {
  const int64_t t128 = ((m + 127) / 128) * ((n + 127) / 128), t256 = ((m + 255) / 256) * ((n + 255) / 256);
  TilePlan plan = {TILE_128_ALONE, 1, 64, 0.0};
  double best = 1e30;
  for (int64_t s = 1; s <= 32 && (s == 1 || (k / s >= 128 && s * t256 <= 512)); ++s) {
    const int64_t piece = k > 0 ? ((k + s - 1) / s + 63) / 64 * 64 : 64;
    const double slices = (double)(piece / 64), join = s > 1 ? 2.5 + (double)s * (double)m * (double)n * 8.0 / 4.0e6 : 0.0;
    const int64_t full = s * t128 / 512, rest = s * t128 % 512;
    const double rounds256 = (double)((s * t256 + 255) / 256);
    const double cost[3] = {
        rounds256 * (1.5 * slices + 11.0),
        (double)full * (0.86 * slices + 8.0) + (rest == 0 ? 0.0 : rest <= 256 ? 0.72 * slices + 8.0 : 0.86 * slices + 8.0),
        s * t128 <= 256 ? 0.55 * slices + 5.0 : 1e30,
    };
    for (int t = 0; t < 3; ++t)
      if (cost[t] + join < (s > 1 ? 0.92 : 0.999) * best) {      // a further piece has to win clearly
        best = cost[t] + join;
        plan = {t, (int)(k > 0 ? (k + piece - 1) / piece : 1), piece, best};
      }
  }
  return plan;
}

}  // namespace eigamd
