// Low-rank adapters of many requests beside a shared projection:
//   P(:,i) = op(A_j) x_i,   Y(:,i) = op(W) x_i + s_j op(B_j) P(:,i),   j the adapter of token i,
// and the gradients of the factors,
//   G_j = s_j sum over j's tokens of u_i p_i^T   (dB: u = dY, p = P; dA: u = X, p = op(B_j)^T dY).
// dX is the first operator again with the factors transposed and their roles exchanged.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "gemm_launch.hpp"
#include "half_gemm.hpp"
#include "lora_project.hpp"
#include "lowrank.hpp"

namespace eigamd {

// lora_few.hip
bool lora_few_half(int64_t m, int64_t n, int64_t k);
bool lora_few_f32(bool w_trans, int64_t m, int64_t n, int64_t k);
int64_t lora_few_work_bytes(int64_t m, int64_t n, int64_t k);
hipError_t lora_few_device(int kind, bool w_trans, const HalfGemm& g, const ProjectArgs& q, hipStream_t s);

namespace {

// ---------------------------------------------------------------------------------------------------------------- plan
// One workgroup per adapter (and one for the tokens without): its waves count, each in its part of the batch, the tokens in front
// of the adapter's run and the adapter's own, and then list those in their order, by ballots -- no atomics, no prefix sum over
// adapters, the same list every time.  Eight loads of a wave are under way together, else every 64 tokens would wait for memory (8192
// tokens, 48 adapters 4.6 us).
__global__ __launch_bounds__(512) void lora_plan_kernel(const int* __restrict__ ids, int n, int adapters, int* __restrict__ order,
                                                        int* __restrict__ seg, int* __restrict__ starts) {
  __shared__ int before[8], own[8];
  const int j = blockIdx.x, w = threadIdx.x / 64, l = threadIdx.x & 63;
  const int share = (n + 511) / 512 * 64, begin = w * share, end = begin + share < n ? begin + share : n;
  auto load = [&](int i0, int (&id)[8]) {
#pragma unroll
    for (int t = 0; t < 8; ++t) id[t] = ids[i0 + t * 64 + l < end ? i0 + t * 64 + l : i0];
#pragma unroll
    for (int t = 0; t < 8; ++t) {
      if ((unsigned)id[t] >= (unsigned)adapters) id[t] = adapters;
      if (i0 + t * 64 + l >= end) id[t] = adapters + 1;      // behind everything
    }
  };
  int less = 0, same = 0;
  for (int i0 = begin; i0 < end; i0 += 512) {
    int id[8];
    load(i0, id);
#pragma unroll
    for (int t = 0; t < 8; ++t) {
      less += __popcll(__ballot(id[t] < j));
      same += __popcll(__ballot(id[t] == j));
    }
  }
  if (l == 0) {
    before[w] = less;
    own[w] = same;
  }
  __syncthreads();
  int start = 0, at = 0;
  for (int z = 0; z < 8; ++z) {
    start += before[z];
    at += z < w ? own[z] : 0;
  }
  if (threadIdx.x == 0) {
    starts[j] = start;
    if (j == adapters) starts[adapters + 1] = n;
  }
  at += start;
  for (int i0 = begin; i0 < end; i0 += 512) {
    int id[8];
    load(i0, id);
#pragma unroll
    for (int t = 0; t < 8; ++t) {
      const unsigned long long mine = __ballot(id[t] == j);
      if (id[t] == j) {
        const int to = at + __popcll(mine & ((1ull << l) - 1));
        order[to] = i0 + t * 64 + l;
        seg[to] = j;
      }
      at += __popcll(mine);
    }
  }
}

// The workgroups of a piece, 16 RT ranks each, run side by side on one XCD (consecutive ones go round the XCDs), where X is then
// read from memory once.
template <typename T, int RT, int FORM> __global__ __launch_bounds__(kProjWaves * 64) void lora_project_kernel(ProjectArgs g) {
  __shared__ __align__(1024) char lds[project_lds(RT, T::bytes)];
  const int across = (g.rank + 16 * RT - 1) / (16 * RT), at = blockIdx.x / 8;
  project_piece<T, RT, FORM>(g, at / across * 8 + blockIdx.x % 8, at % across * 16 * RT, lds);
}
template <typename T, int RT> hipError_t launch_project_rank(const ProjectArgs& g, hipStream_t s) {
  const dim3 grid((unsigned)((project_slots(g) + 7) / 8 * 8 * ((g.rank + 16 * RT - 1) / (16 * RT)))), block(kProjWaves * 64);
  switch (project_form<T>(g)) {
    case A_K: hipLaunchKernelGGL((lora_project_kernel<T, RT, A_K>), grid, block, 0, s, g); break;
    case A_R:
      if constexpr (T::bytes == 2) hipLaunchKernelGGL((lora_project_kernel<T, RT, A_R>), grid, block, 0, s, g);
      break;
    default: hipLaunchKernelGGL((lora_project_kernel<T, RT, A_ANY>), grid, block, 0, s, g);
  }
  return hipGetLastError();
}
// 16, 32 or 64 ranks a workgroup: they take about 9.5, 13 and 15 us with 4032 positions, as long as there are at most 256 of them, and
// in proportion to their number beyond (rank 64, 3589 tokens: 16.2, 13.4, 15.5 us; 8192 tokens: 22.8, 23.9, 16.3; 142: 9.4, 12.8,
// 14.2).
template <typename T> hipError_t launch_project(const ProjectArgs& g, hipStream_t s) {
  // (an adapter's last piece is there or not)
  const double pieces = g.n / kProjTokens + (g.n <= g.none ? (double)g.n : (g.none + 1) * 0.5);
  auto cost = [&](int rt, double us) { return std::max(1.0, pieces * ((g.rank + 16 * rt - 1) / (16 * rt)) / 256.0) * us; };
  const double one = cost(1, 9.5), two = cost(2, 13.0), four = cost(4, 15.0);
  if (one <= two && one <= four) return launch_project_rank<T, 1>(g, s);
  return two <= four ? launch_project_rank<T, 2>(g, s) : launch_project_rank<T, 4>(g, s);
}

// Y += s_j op(B_j) P in single precision, behind the plain product: a wave takes 16 rows of 16 columns, so that there are many of
// them, each with few adapters (64 x 64 a wave left most units idle: 777 tokens x 1024 took 24 us, now 7).
__global__ __launch_bounds__(256) void lora_add_f32_kernel(HalfGemm g) {
  const int w = threadIdx.x / 64, l = threadIdx.x & 63;
  const int row0 = blockIdx.y * 64 + w * 16, col0 = blockIdx.x * 16;
  if (row0 >= g.m) return;
  f32x4 acc[1][1] = {};
  add_adapters<Fp32, 1, 1>(g, row0, col0, acc);
  const int c = col0 + (l & 15), r = row0 + (l / 16) * 4;
  if (c >= g.n || g.seg[c] == g.none) return;
  float* y = static_cast<float*>(g.c) + (int64_t)g.order[c] * g.ldc;
  for (int t = 0; t < 4; ++t)
    if (r + t < g.m) y[r + t] += acc[0][0][t];
}

template <typename T, int LA, int B, int WM, int WN, int D> hipError_t launch_tiles(const HalfGemm& g, hipStream_t s) {
  const dim3 grid((unsigned)(((g.m + B - 1) / B) * (((int64_t)g.n + B - 1) / B)), g.splits);
  hipLaunchKernelGGL((half_gemm_kernel<T, LA, KC, OUT_HALF, B, B, WM, WN, D>), grid, dim3(WM * WN * 64), 0, s, g);
  return hipGetLastError();
}
template <typename T, int LA> hipError_t launch_form(const HalfGemm& g, int tile, hipStream_t s) {
  return tile == TILE_256   ? launch_tiles<T, LA, 256, 2, 4, 2>(g, s)
         : tile == TILE_128 ? launch_tiles<T, LA, 128, 2, 2, 2>(g, s)
                            : launch_tiles<T, LA, 128, 2, 4, 4>(g, s);
}

// What a call keeps in its scratch memory: sums of a split reduction, then copies of W and of X with whole chunks (launch_half).
struct HalfWork {
  int64_t sums, w_copy, x_copy;
};
HalfWork half_work(bool w_trans, int64_t m, int64_t n, int64_t k, const void* w, int64_t ldw, const void* x, int64_t ldx) {
  HalfWork need = {0, 0, 0};
  const bool w_whole = whole_chunks(w, ldw, w_trans ? k : m);
  if (lora_few_half(m, n, k)) {
    need.sums = lora_few_work_bytes(m, n, k);      // (read where they are, whatever their alignment; chunks of 8 rows have to exist)
    if (!w_trans && m < 8) need.w_copy = padded_bytes(m, k);
  } else {
    const int splits = plan_tiles(m, n, k).splits;
    if (splits > 1) need.sums = (int64_t)splits * m * n * 4;
    if (!w_whole) need.w_copy = w_trans ? padded_bytes(k, m) : padded_bytes(m, k);
    if (!whole_chunks(x, ldx, k)) need.x_copy = padded_bytes(k, n);
  }
  need.sums = (need.sums + 255) / 256 * 256;
  return need;
}

HalfGemm gemm_args(const LoraArgs& c) {
  HalfGemm g;
  g.m = (int)c.m; g.n = (int)c.n; g.k = (int)c.k;
  g.a = c.w; g.lda = c.ldw;
  g.b = c.x; g.ldb = c.ldx;
  g.c = c.y; g.ldc = c.ldy;
  g.order = c.plan.order;
  g.seg = c.plan.seg;
  g.none = c.plan.adapters;
  g.rank = c.plan.adapters > 0 ? (int)c.rank : 0;
  g.up = c.b;
  g.up_row = c.b_trans ? c.ldb : 1;
  g.up_rank = c.b_trans ? 1 : c.ldb;
  g.up_stride = c.stride_b;
  g.p = c.p; g.ldp = c.ldp;
  g.scale = c.scale;
  return g;
}
// The few-token form in single precision; where W is not transposed, chunks of 4 rows have to exist.
bool few_f32(bool w_trans, int64_t m, int64_t n, int64_t k) { return (w_trans || m >= 4) && lora_few_f32(w_trans, m, n, k); }

template <typename T> hipError_t launch_half(const LoraArgs& c, const ProjectArgs& q, hipStream_t s) {
  HalfGemm g = gemm_args(c);
  const HalfWork need = half_work(c.w_trans, c.m, c.n, c.k, c.w, c.ldw, c.x, c.ldx);
  char* work = static_cast<char*>(c.work);
  g.partial = reinterpret_cast<float*>(work);
  PadCopy w_copy = {}, x_copy = {};
  if (need.w_copy) {
    w_copy = pad_copy(c.w, c.ldw, c.w_trans ? c.k : c.m, c.w_trans ? c.m : c.k, work + need.sums);
    g.a = w_copy.to;
    g.lda = padded(c.w_trans ? c.k : c.m);
  }
  if (need.x_copy) {
    x_copy = pad_copy(c.x, c.ldx, c.k, c.n, work + need.sums + need.w_copy);
    g.b = x_copy.to;
    g.ldb = padded(c.k);
  }
  hipError_t e = launch_pad_copy(w_copy, x_copy, s);
  if (e != hipSuccess) return e;
  if (lora_few_half(c.m, c.n, c.k)) return lora_few_device(c.kind, c.w_trans, g, q, s);
  if (q.p && (e = launch_project<T>(q, s)) != hipSuccess) return e;
  const TilePlan plan = plan_tiles(c.m, c.n, c.k);
  g.splits = plan.splits;
  g.k_piece = (int)plan.k_piece;
  e = c.w_trans ? launch_form<T, KC>(g, plan.tile, s) : launch_form<T, MC>(g, plan.tile, s);
  if (e != hipSuccess || g.splits == 1) return e;
  return launch_half_join(g.partial, g.splits, g.m, c.m * c.n, 0.0f, static_cast<typename T::elem*>(g.c), g.ldc, g.order, s);
}

// ------------------------------------------------------------------------------------------------ gradients of the factors
constexpr int kGradRows = 256;
enum { DIRECT, STAGED, QUANT };    // u: global -> LDS by hardware / through registers, any alignment / from 8 bits

struct GradArgs {
  int rows, rank, n, none, chunk, slots;
  bool trans, halves;
  const void* u; int64_t ldu;
  const uint8_t* exponents; int64_t lde;
  const float* p; int64_t ldp;
  const float* scale;
  const int* order;
  const int* starts;
  float beta;
  float* g; int64_t ldg, stride_g;
  float* partial;
};

// Tokens per workgroup: about 512 workgroups in all, between 128 and 1024 tokens each (1000 tokens x 1024, one
// adapter of rank 8: 9.6 us, with 256 or more 14.2).
int grad_chunk(int64_t rows, int64_t n) {
  const int64_t across = (rows + kGradRows - 1) / kGradRows;
  const int64_t pieces = std::max<int64_t>(512 / across, 1);
  const int64_t c = ((n + pieces - 1) / pieces + 31) / 32 * 32;
  return (int)std::min<int64_t>(std::max<int64_t>(c, 128), 1024);
}

// 32 tokens x 256 rows of u in LDS: lines of tokens, chunks permuted as in SliceLoader (MC).  Single precision lies unpermuted
// and is read one element a lane.
template <typename T, int SRC> struct GradTile {
  using E = typename T::elem;
  using x8 = typename T::x8;
  static constexpr int bytes = 32 * kGradRows * T::bytes;
  x8 reg[4];
  uint64_t qreg[4];
  unsigned ereg[4];
  static __device__ __forceinline__ int swizzle(int line) { return T::bytes == 4 ? 0 : ((line & 3) | ((line >> 1) & 4)) << 1; }
  // token of line i: tok[i], -1 past the end
  __device__ __forceinline__ void load(char* lds, const GradArgs& g, const int* tok, int row0) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int ch = threadIdx.x + i * 256, line = ch / 32, c = (ch % 32) ^ swizzle(line), row = row0 + c * 8;
      const int t = tok[line], n = t < 0 ? 0 : g.rows - row;
      if constexpr (SRC == DIRECT) {
        const char* q = static_cast<const char*>(g.u) + ((int64_t)t * g.ldu + row) * 2;
        const char* from = n > 0 ? q : reinterpret_cast<const char*>(zero_page);
        const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
        __builtin_amdgcn_global_load_lds(EIGAMD_GLOBAL(from), EIGAMD_LDS(void, lds + (i * 256 + wave * 64) * 16), 16, 0, 0);
      } else if constexpr (SRC == STAGED) {
        reg[i] = load_up_to_8<E, x8>(static_cast<const E*>(g.u) + (int64_t)t * g.ldu + row, n);
      } else {
        qreg[i] = load_bytes(static_cast<const int8_t*>(g.u) + (int64_t)t * g.ldu + row, n);
        ereg[i] = n > 0 ? g.exponents[(int64_t)t * g.lde + row / 32] : 0u;
      }
    }
  }
  __device__ __forceinline__ void store(char* lds) {
    if constexpr (SRC == DIRECT) return;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (SRC == QUANT) reg[i] = unpack_8<T>(qreg[i], exponent_scale(ereg[i]));
      *reinterpret_cast<x8*>(lds + (threadIdx.x + i * 256) * 8 * T::bytes) = reg[i];
    }
  }
  static __device__ __forceinline__ x8 fragment(const char* lds, int row) {
    const int l = threadIdx.x & 63;
    if constexpr (T::bytes == 4) {
      x8 v;
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = *reinterpret_cast<const float*>(lds + (((l / 16) * 8 + e) * kGradRows + row + (l & 15)) * 4);
      return v;
    } else {
      union { x8 v; typename T::x4 h[2]; } f;
      const int line = (l / 16) * 8 + (l & 15) / 4, at = row / 8 + (l & 3) / 2;
#pragma unroll
      for (int h = 0; h < 2; ++h)
        f.h[h] = T::read_transposed(lds + (line + 4 * h) * (kGradRows * 2) + ((at ^ swizzle(line + 4 * h)) * 16) + (l & 1) * 8);
      return f.v;
    }
  }
};

// G_j over one piece of j's tokens: 256 rows x 16 RT ranks per workgroup, 32 tokens a turn.  p keeps all of its 32 bits, as three 16-bit
// pieces; the sums are the matrix unit's 32 bits.  A run that is one piece goes straight to G_j.
// f16 has neither p's range nor room for three pieces of what is far below the largest: a turn's p is normalised rank by rank, and a wave
// that holds a p below about 2^-16 of its rank's largest (one turn in fifty of normally distributed p) takes that turn's products in single
// precision, six times the work.
// The product of an infinity and a piece of p that is zero is a NaN, where that with p is an infinity: where a NaN has come up, a wave's
// sums are made again in single precision, from memory as it is.
// (Three waves a SIMD: left to itself the compiler takes two registers too many for rank 64 from a checkpoint, 45 -> 48 us.)
template <typename T, int SRC, int RT, bool TRANS> __global__ __launch_bounds__(256, __is_same(T, Bf16) ? 3 : 1) void lora_grad_kernel(GradArgs g) {
  using E = typename T::elem;
  using x8 = typename T::x8;
  constexpr int NP = T::bytes == 4 ? 1 : 3;
  if ((int)blockIdx.y >= g.slots) {
    // an adapter without tokens gets beta G_j
    const int j = blockIdx.y - g.slots;
    if (g.starts[j] != g.starts[j + 1]) return;
    const int high = g.rows - blockIdx.x * kGradRows < kGradRows ? g.rows - blockIdx.x * kGradRows : kGradRows;
    const int wide = g.rank - blockIdx.z * 64 < 64 ? g.rank - blockIdx.z * 64 : 64, fast = TRANS ? wide : high;
    float* at = g.g + (int64_t)j * g.stride_g + (int64_t)blockIdx.x * kGradRows * (TRANS ? g.ldg : 1) + (int64_t)blockIdx.z * 64 * (TRANS ? 1 : g.ldg);
    for (int q = threadIdx.x; q < high * wide; q += 256) {
      float* to = at + (int64_t)(q / fast) * g.ldg + q % fast;
      *to = g.beta != 0.0f ? g.beta * *to : 0.0f;
    }
    return;
  }
  Piece piece;
  if (!find_piece(g.starts, g.none + 1, g.chunk, blockIdx.y, piece) || piece.adapter == g.none) return;
  using Tile = GradTile<T, SRC>;
  __shared__ __align__(1024) char lds[2 * Tile::bytes];
  __shared__ int tok[1024 + 32];
  const int count = piece.end - piece.begin, turns = (count + 31) / 32;
  const int w = threadIdx.x / 64, l = threadIdx.x & 63;
  const int row0 = blockIdx.x * kGradRows, r0 = blockIdx.z * 64;
  for (int i = threadIdx.x; i < turns * 32; i += 256) tok[i] = i < count ? g.order[piece.begin + i] : -1;
  __syncthreads();
  Tile tile;
  // RT waves beside each other take 16 ranks each (every wave then makes the pieces of its own p only), 4 / RT one behind the
  // other 64 RT rows each
  constexpr int NI = 4 * RT;
  const int wr = (w / RT) * 64 * RT, r = r0 + (w % RT) * 16 + (l & 15);
  f32x4 acc[NI] = {};
  // p of a turn, loaded a turn early like u
  float pv[8], pn[8];
  auto load_p = [&](float(&v)[8], int s) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int token = tok[s * 32 + (l / 16) * 8 + e];
      v[e] = token >= 0 && r < g.rank ? g.p[(int64_t)token * g.ldp + r] : 0.0f;
    }
  };
  load_p(pv, 0);
  tile.load(lds, g, tok, row0);
  tile.store(lds);
  __syncthreads();
  for (int s = 0; s < turns; ++s) {
    char* here = lds + (s & 1) * Tile::bytes;
    char* next = lds + ((s & 1) ^ 1) * Tile::bytes;
    if (s + 1 < turns) {
      load_p(pn, s + 1);
      tile.load(next, g, tok + (s + 1) * 32, row0);
    }
    x8 fp[NP];
    auto product = [&](x8 fu, f32x4 sum) {
#pragma unroll
      for (int z = NP - 1; z >= 0; --z) sum = TRANS ? T::mma(fp[z], fu, sum) : T::mma(fu, fp[z], sum);
      return sum;
    };
    if constexpr (__is_same(T, F16)) {
      float top = largest_of(pv);      // (one that is infinite leaves nothing finite in its rank)
      top = fmaxf(top, __shfl_xor(top, 16));      // (lanes l, l + 16, ... hold the same rank)
      top = fmaxf(top, __shfl_xor(top, 32));
      const Norm nm = norm_of(top);
      float v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        v[e] = pv[e] * nm.down;
        E q[NP];
        split_f16<0>(v[e], q);
#pragma unroll
        for (int z = 0; z < NP; ++z) fp[z][e] = q[z];
      }
      const bool small = some_below(v, smallest_f16<0>());
      if (__builtin_expect(__any(small), 0)) {
        Fp32::x8 p;
#pragma unroll
        for (int e = 0; e < 8; ++e) p[e] = pv[e];
#pragma unroll
        for (int i = 0; i < NI; ++i) {
          const Fp32::x8 u = __builtin_convertvector(Tile::fragment(here, wr + i * 16), Fp32::x8);
          acc[i] = TRANS ? Fp32::mma(p, u, acc[i]) : Fp32::mma(u, p, acc[i]);
        }
      } else {
        f32x4 up;      // of the ranks of a lane's four results
#pragma unroll
        for (int t = 0; t < 4; ++t) up[t] = TRANS ? __shfl(nm.up, (l / 16) * 4 + t) : nm.up;
#pragma unroll
        for (int i = 0; i < NI; ++i) acc[i] += up * product(Tile::fragment(here, wr + i * 16), f32x4{0.0f, 0.0f, 0.0f, 0.0f});
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if constexpr (NP == 1) {
          fp[0][e] = pv[e];
        } else {
          E q[NP];
          split_bf16(pv[e], q);
#pragma unroll
          for (int z = 0; z < NP; ++z) fp[z][e] = q[z];
        }
      }
#pragma unroll
      for (int i = 0; i < NI; ++i) acc[i] = product(Tile::fragment(here, wr + i * 16), acc[i]);
    }
    if (s + 1 < turns) tile.store(next);
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 8; ++e) pv[e] = pn[e];
  }
  if constexpr (T::bytes == 2) {
    f32x4 all = acc[0];
#pragma unroll
    for (int i = 1; i < NI; ++i) all += acc[i];
    const float sum = (all[0] + all[1]) + (all[2] + all[3]);
    if (__builtin_expect(__any(sum != sum), 0)) {
      auto value = [&](int token, int row) {
        if (token < 0 || row >= g.rows) return 0.0f;
        if constexpr (SRC == QUANT) return static_cast<const int8_t*>(g.u)[token * g.ldu + row] * exponent_scale(g.exponents[token * g.lde + row / 32]);
        else return (float)static_cast<const E*>(g.u)[token * g.ldu + row];
      };
#pragma unroll
      for (int i = 0; i < NI; ++i) acc[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 1
      for (int s = 0; s < turns; ++s) {
        load_p(pv, s);
        Fp32::x8 p, u;
#pragma unroll
        for (int e = 0; e < 8; ++e) p[e] = pv[e];
#pragma unroll
        for (int i = 0; i < NI; ++i) {
#pragma unroll
          for (int e = 0; e < 8; ++e) u[e] = value(tok[s * 32 + (l / 16) * 8 + e], row0 + wr + i * 16 + (l & 15));
          acc[i] = TRANS ? Fp32::mma(p, u, acc[i]) : Fp32::mma(u, p, acc[i]);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    }
  }
  const bool whole = piece.run_end - piece.run_begin <= g.chunk;
  const float sj = whole ? g.scale[piece.adapter] : 1.0f;
  const int slot = g.halves ? 2 * piece.run_begin / g.chunk + piece.index : (int)blockIdx.y;      // (lora_grad_join_kernel)
  float* out = whole ? g.g + (int64_t)piece.adapter * g.stride_g : g.partial + (int64_t)slot * g.rows * g.rank;
  const int64_t ld = whole ? g.ldg : (TRANS ? g.rank : g.rows);
  const float beta = whole ? g.beta : 0.0f;
  const int limit = TRANS ? g.rank : g.rows;
  const bool wide = (reinterpret_cast<uintptr_t>(out) & 15) == 0 && ld % 4 == 0;
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const int rank0 = r0 + (w % RT) * 16, top = row0 + wr + i * 16;
    const int fast = (TRANS ? rank0 : top) + (l / 16) * 4, slow = (TRANS ? top : rank0) + (l & 15);
    if (slow >= (TRANS ? g.rows : g.rank)) continue;
    float* at = out + (int64_t)slow * ld + fast;
    f32x4 v = acc[i] * sj;
    if (wide && fast + 4 <= limit) {
      // (one by one, four times as many addresses for the memory pipeline: 40 tokens x 1024, rank 64 16 us, now 7.7)
      if (beta != 0.0f) v += beta * *reinterpret_cast<const f32x4*>(at);
      *reinterpret_cast<f32x4*>(at) = v;
    } else {
      for (int e = 0; e < 4; ++e)
        if (fast + e < limit) at[e] = v[e] + (beta != 0.0f ? beta * at[e] : 0.0f);
    }
  }
}

// G_j = beta G_j + s_j (sum of j's pieces, in the order of the batch).
// Where the sums of a run's first piece stand, of those that a run of several pieces leaves to the join.  begin / chunk + j keeps them apart
// (find_piece), with room for every adapter; so does 2 begin / chunk (`halves`), as a run of more than `chunk` tokens has no more pieces
// than half chunks, with room for the tokens: whichever is less.
__global__ __launch_bounds__(256) void lora_grad_join_kernel(GradArgs g) {
  const int j = blockIdx.y, begin = g.starts[j], count = g.starts[j + 1] - begin;
  if (count <= g.chunk) return;
  const int pieces = (count + g.chunk - 1) / g.chunk, slot = (g.halves ? 2 * begin : begin) / g.chunk + (g.halves ? 0 : j);
  const int64_t size = (int64_t)g.rows * g.rank;
  const int fast = g.trans ? g.rank : g.rows;
  for (int64_t q = (int64_t)blockIdx.x * 256 + threadIdx.x; q < size; q += (int64_t)gridDim.x * 256) {
    float sum = 0.0f;
    int z = 0;
    for (; z + 8 <= pieces; z += 8) {      // eight loads at a time under way, added in order
      float v[8];
#pragma unroll
      for (int t = 0; t < 8; ++t) v[t] = g.partial[(int64_t)(slot + z + t) * size + q];
#pragma unroll
      for (int t = 0; t < 8; ++t) sum += v[t];
    }
    for (; z < pieces; ++z) sum += g.partial[(int64_t)(slot + z) * size + q];
    const int64_t slow = q / fast;
    float* at = g.g + (int64_t)j * g.stride_g + slow * g.ldg + (q - slow * fast);
    *at = g.scale[j] * sum + (g.beta != 0.0f ? g.beta * *at : 0.0f);
  }
}

template <typename T, int SRC, int RT> hipError_t launch_grad(const GradArgs& g, dim3 grid, hipStream_t s) {
  if (g.trans) hipLaunchKernelGGL((lora_grad_kernel<T, SRC, RT, true>), grid, dim3(256), 0, s, g);
  else hipLaunchKernelGGL((lora_grad_kernel<T, SRC, RT, false>), grid, dim3(256), 0, s, g);
  return hipGetLastError();
}
template <typename T, int SRC> hipError_t launch_grad_rank(const GradArgs& g, dim3 grid, hipStream_t s) {
  if (g.rank <= 16) return launch_grad<T, SRC, 1>(g, grid, s);
  if (g.rank <= 32) return launch_grad<T, SRC, 2>(g, grid, s);
  return launch_grad<T, SRC, 4>(g, grid, s);
}

}  // namespace

hipError_t lora_plan_device(const int* ids, int64_t n, int64_t adapters, int* d_plan, hipStream_t s) {
  hipLaunchKernelGGL(lora_plan_kernel, dim3((unsigned)(adapters + 1)), dim3(512), 0, s, ids, (int)n, (int)adapters, d_plan,
                     d_plan + n, d_plan + 2 * n);
  return hipGetLastError();
}

int64_t lora_work_bytes(int kind, bool w_trans, int64_t m, int64_t n, int64_t k, const void* w, int64_t ldw, const void* x, int64_t ldx) {
  if (m <= 0 || n <= 0) return 0;
  if (kind == F32) return few_f32(w_trans, m, n, k) ? lora_few_work_bytes(m, n, k) : std::min<int64_t>(16 * m * n * 4, (int64_t)256 << 20);
  const HalfWork need = half_work(w_trans, m, n, k, w, ldw, x, ldx);
  return need.sums + need.w_copy + need.x_copy;
}

hipError_t lora_device(const LoraArgs& c, hipStream_t s) {
  ProjectArgs p;
  p.n = (int)c.n; p.k = (int)c.k; p.rank = (int)c.rank; p.none = c.plan.adapters;
  p.x = c.x; p.ldx = c.ldx;
  p.a = c.a;
  p.a_row = c.a_trans ? c.lda : 1;
  p.a_k = c.a_trans ? 1 : c.lda;
  p.a_stride = c.stride_a;
  p.order = c.plan.order; p.seg = c.plan.seg; p.starts = c.plan.starts;
  p.p = c.p; p.ldp = c.ldp;
  if (c.m > 0 && c.kind == F32 && few_f32(c.w_trans, c.m, c.n, c.k)) {
    HalfGemm g = gemm_args(c);
    g.partial = static_cast<float*>(c.work);
    return lora_few_device(F32, c.w_trans, g, p, s);
  }
  if (c.m > 0 && c.kind == BF16) return launch_half<Bf16>(c, p, s);
  if (c.m > 0 && c.kind == F16K) return launch_half<F16>(c, p, s);
  hipError_t e = hipSuccess;
  if (p.p) {
    e = c.kind == BF16 ? launch_project<Bf16>(p, s) : c.kind == F16K ? launch_project<F16>(p, s) : launch_project<Fp32>(p, s);
  }
  if (e != hipSuccess || c.m == 0) return e;
  GemmCall q;
  q.kind = F32;
  q.opa = c.w_trans ? OP_T : OP_N; q.opb = OP_N;
  q.m = c.m; q.n = c.n; q.k = c.k;
  q.alpha[0] = 1.0; q.alpha[1] = 0.0; q.beta[0] = 0.0; q.beta[1] = 0.0;
  q.A = c.w; q.lda = c.ldw; q.B = c.x; q.ldb = c.ldx; q.C = c.y; q.ldc = c.ldy;
  // (memory of the caller's, or none at all: either way the product allocates nothing and stays on this stream)
  q.partials = c.work ? c.work : c.y;
  q.partials_bytes = c.work ? (size_t)c.work_bytes : 0;
  e = launch_gemm_f32(q, s);
  if (e != hipSuccess || c.plan.adapters == 0) return e;
  const HalfGemm g = gemm_args(c);
  hipLaunchKernelGGL(lora_add_f32_kernel, dim3((unsigned)((c.n + 15) / 16), (unsigned)((c.m + 63) / 64)), dim3(256), 0, s, g);
  return hipGetLastError();
}

int64_t lora_grad_work_bytes(int64_t rows, int64_t n, int64_t rank, int64_t adapters) {
  const int chunk = grad_chunk(std::max<int64_t>(rows, 1), n);
  return n > chunk ? std::min(2 * n / chunk, n / chunk + adapters + 1) * rows * rank * 4 : 0;
}

hipError_t lora_grad_device(const LoraGradArgs& c, hipStream_t s) {
  GradArgs g;
  g.rows = (int)c.rows; g.rank = (int)c.rank; g.n = (int)c.n; g.none = c.plan.adapters;
  g.chunk = grad_chunk(c.rows, c.n);
  g.halves = 2 * c.n / g.chunk < c.n / g.chunk + g.none + 1;
  g.trans = c.trans;
  g.u = c.u; g.ldu = c.ldu; g.exponents = c.exponents; g.lde = c.lde;
  g.p = c.p; g.ldp = c.ldp; g.scale = c.scale;
  g.order = c.plan.order; g.starts = c.plan.starts;
  g.beta = c.beta;
  g.g = c.g; g.ldg = c.ldg; g.stride_g = c.stride_g;
  g.partial = static_cast<float*>(c.work);
  hipError_t e = hipSuccess;
  g.slots = (int)(c.n / g.chunk) + g.none + 1;
  const dim3 grid((unsigned)((c.rows + kGradRows - 1) / kGradRows), (unsigned)(g.slots + g.none), (unsigned)((c.rank + 63) / 64));
  const bool direct = (uintptr_t)c.u % 16 == 0 && c.ldu % 8 == 0 && c.rows % 8 == 0;
  if (c.exponents) {
    e = c.kind == BF16 ? launch_grad_rank<Bf16, QUANT>(g, grid, s)
                       : c.kind == F16K ? launch_grad_rank<F16, QUANT>(g, grid, s) : launch_grad_rank<Fp32, QUANT>(g, grid, s);
  } else if (c.kind == F32) {
    e = launch_grad_rank<Fp32, STAGED>(g, grid, s);
  } else if (direct) {
    e = c.kind == BF16 ? launch_grad_rank<Bf16, DIRECT>(g, grid, s) : launch_grad_rank<F16, DIRECT>(g, grid, s);
  } else {
    e = c.kind == BF16 ? launch_grad_rank<Bf16, STAGED>(g, grid, s) : launch_grad_rank<F16, STAGED>(g, grid, s);
  }
  if (e != hipSuccess || c.n <= g.chunk) return e;
  const unsigned blocks = (unsigned)std::min<int64_t>((c.rows * c.rank + 255) / 256, 1024);
  hipLaunchKernelGGL(lora_grad_join_kernel, dim3(blocks, (unsigned)g.none), dim3(256), 0, s, g);
  return hipGetLastError();
}

}  // namespace eigamd
