// The adapter product for few tokens (one a request while answering): one launch over W and the projection, one that joins.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "gemm_launch.hpp"
#include "half_gemm.hpp"
#include "lora_project.hpp"
#include "lowrank.hpp"

namespace eigamd {

namespace {

template <typename E, int N> using Part = E __attribute__((ext_vector_type(N)));

// Y for few tokens, 16 NG of them a workgroup: the time is that of reading W, from as many compute units as there are.  A
// workgroup owns 64 rows and one piece of the reduction, so that X, which every workgroup reads its piece of, costs little beside
// W (with 16 rows and the whole reduction X was four times the traffic: 64 tokens x 4096 x 4096 took 22 us, now 13).  Its eight
// waves share the piece, 64 (32) positions a turn, turned in the wave's own LDS (W's reduction contiguous: as a RowBlock; its rows: read
// back transposed, single precision one element at a time).  The sums go to memory in 32 bits; the second kernel adds the
// pieces up and the low-rank part to them.
// The projection needs nothing of this, so its workgroups (16 ranks each) are the first ones of the same launch.
template <typename T, int LA, int NG, int FORM> __global__ __launch_bounds__(512) void lora_few_kernel(HalfGemm g, ProjectArgs q, int project, int slots) {
  using E = typename T::elem;
  using x8 = typename T::x8;
  // Products of a turn, one block of each operand: lines of 128 bytes (64 tokens x 8192 x 8192 52 -> 45 us, 192 x 4096 x 4096 27 -> 25; 98 x
  // 7744 x 1088 17.0 -> 17.6).  W's rows contiguous, 64 tokens: no registers for that.
  constexpr int S = T::bytes == 4 || (NG == 4 && LA == MC) ? 1 : 2;
  using Block = RowBlock<T, S>;
  constexpr int red_bytes = 8 * 4 * NG * 64 * 16, blocks_bytes = 8 * (4 + NG) * Block::bytes;
  constexpr int loop_bytes = blocks_bytes > project_lds(1, T::bytes) ? blocks_bytes : project_lds(1, T::bytes);
  constexpr int lds_bytes = red_bytes > loop_bytes ? red_bytes : loop_bytes;
  __shared__ __align__(1024) char lds[lds_bytes];
  if ((int)blockIdx.x < project) {
    project_piece<T, 1, FORM>(q, blockIdx.x % slots, blockIdx.x / slots * 16, lds);
    return;
  }
  const int id = blockIdx.x - project, row_blocks = (g.m + 63) / 64, groups = (g.n + 63) / 64;
  const int part = id / 8 / groups * 8 + id % 8, col0 = id / 8 % groups * 64;
  if (part >= row_blocks * g.splits) return;
  const int row0 = part % row_blocks * 64, z = part / row_blocks;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), l = threadIdx.x & 63;
  const int k_begin = z * g.k_piece, k_end = k_begin + g.k_piece < g.k ? k_begin + g.k_piece : g.k;
  // MC: chunks of CH rows, one that would pass the end holds the last CH, some of them twice
  constexpr int CH = T::bytes == 4 ? 4 : 8;
  const int last = g.m < CH ? 0 : g.m - CH;
  const E* a[4][S];                   // KC: rows of the four row blocks; MC: chunks of 8 lines
  const E* b[NG][S];                  // rows and columns past the end repeat the last one and are not stored
#pragma unroll
  for (int t = 0; t < 4; ++t)
#pragma unroll
    for (int h = 0; h < S; ++h) {
      if constexpr (LA == KC) {
        const int row = row0 + t * 16 + Block::row(h);
        a[t][h] = static_cast<const E*>(g.a) + (int64_t)(row < g.m ? row : g.m - 1) * g.lda;
      } else {
        const int row = row0 + l % (64 / CH) * CH;
        a[t][h] = static_cast<const E*>(g.a) + (int64_t)(h * 32 + t * 8 + l / (64 / CH)) * g.lda + (row < last ? row : last);
      }
    }
#pragma unroll
  for (int c = 0; c < NG; ++c)
#pragma unroll
    for (int h = 0; h < S; ++h) {
      const int at = col0 + c * 16 + Block::row(h);
      b[c][h] = static_cast<const E*>(g.b) + (int64_t)g.order[at < g.n ? at : g.n - 1] * g.ldb;
    }
  f32x4 acc[4][NG] = {};
  // whole turns, then what is left, by one wave (as in project_piece)
  using Whole = std::true_type;
  using Rest = std::false_type;
  auto load = [&](int k0, x8(&fa)[4][S], x8(&fb)[NG][S], auto whole) {
    const int k = k0 + Block::position(), left = k_end - k;
#pragma unroll
    for (int h = 0; h < S; ++h) {
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        if constexpr (LA == KC) {
          fa[t][h] = whole ? load_8<E, x8>(a[t][h] + k) : load_first<E, x8>(a[t][h] + (left > 0 ? k : 0), 1, left);
        } else {
          // 16 bytes of a line; of single precision also of the line 4 further
          constexpr int P = 8 / CH;
          struct { Part<E, CH> part[P]; } v;
#pragma unroll
          for (int p = 0; p < P; ++p) {
            const bool in = whole || k0 + h * 32 + t * 8 + p * 4 + l / (64 / CH) < k_end;
            __builtin_memcpy(&v.part[p], in ? a[t][h] + (int64_t)(k0 + p * 4) * g.lda : static_cast<const E*>(g.a), 16);
#pragma unroll
            for (int e = 0; e < CH; ++e) v.part[p][e] = in ? v.part[p][e] : (E)0.0f;
          }
          fa[t][h] = __builtin_bit_cast(x8, v);
        }
      }
#pragma unroll
      for (int c = 0; c < NG; ++c) fb[c][h] = whole ? load_8<E, x8>(b[c][h] + k) : load_first<E, x8>(b[c][h] + (left > 0 ? k : 0), 1, left);
    }
  };
  auto multiply = [&](const x8(&fa)[4][S], const x8(&fb)[NG][S]) {
    char* mine = lds + w * (4 + NG) * Block::bytes;
    auto own = [&](int t) { return mine + t * Block::bytes; };
    wave_order();
#pragma unroll
    for (int h = 0; h < S; ++h) {
#pragma unroll
      for (int c = 0; c < NG; ++c) Block::put(own(4 + c), fb[c][h], h);
      if constexpr (LA == KC) {
#pragma unroll
        for (int t = 0; t < 4; ++t) Block::put(own(t), fa[t][h], h);
      }
    }
#pragma unroll
    for (int h = 0; h < S; ++h) {
      x8 f[4], y[NG];
      if (LA == KC && h == 0) wave_order();
      if (LA == MC && h > 0) wave_order();
      if constexpr (LA == MC && T::bytes == 4) {
        // lines of 64 rows, 256 bytes, read back one element at a time; the four lines a wave reads together are turned by 16 rows
        // against each other so that they meet all banks once
        float* lines = reinterpret_cast<float*>(mine);
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          struct { f32x4 part[2]; } v = __builtin_bit_cast(decltype(v), fa[t][h]);
#pragma unroll
          for (int p = 0; p < 2; ++p) *reinterpret_cast<f32x4*>(lines + (t * 8 + p * 4 + l / 16) * 64 + ((l % 16 * 4) ^ (t * 16))) = v.part[p];
        }
        wave_order();
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int e = 0; e < 8; ++e) f[t][e] = lines[(l / 16 * 8 + e) * 64 + ((t * 16 + l % 16) ^ (l / 16 * 16))];
      } else if constexpr (LA == MC) {
        // lines of 64 rows, 128 bytes; chunks permuted so that the 8 lines a half wave reads meet all banks once
        auto slot = [](int line, int ch) { return line * 128 + (ch ^ (((line >> 1) & 1) | ((line >> 2) & 2)) << 1) * 16; };
#pragma unroll
        for (int t = 0; t < 4; ++t) *reinterpret_cast<x8*>(mine + slot(t * 8 + l / 8, l % 8)) = fa[t][h];
        wave_order();
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          union { x8 v; typename T::x4 h[2]; } u;
          const int line = (l / 16) * 8 + (l & 15) / 4, ch = t * 2 + (l & 3) / 2;
#pragma unroll
          for (int e = 0; e < 2; ++e) u.h[e] = T::read_transposed(mine + slot(line + 4 * e, ch) + (l & 1) * 8);
          f[t] = u.v;
        }
      } else {
#pragma unroll
        for (int t = 0; t < 4; ++t) f[t] = Block::get(own(t), h);
      }
#pragma unroll
      for (int c = 0; c < NG; ++c) y[c] = Block::get(own(4 + c), h);
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int c = 0; c < NG; ++c) acc[t][c] = T::mma(f[t], y[c], acc[t][c]);
    }
  };
  x8 fa[2][4][S], fb[2][NG][S];
  const int turns = (k_end - k_begin) / (32 * S);
  auto load_turn = [&](int turn, int set) { load(k_begin + turn * 32 * S, fa[set], fb[set], Whole{}); };
  int at = w;
  if (at < turns) load_turn(at, 0);
  for (; at < turns; at += 16) {
    if (at + 8 < turns) load_turn(at + 8, 1);
    multiply(fa[0], fb[0]);
    if (at + 8 >= turns) break;
    if (at + 16 < turns) load_turn(at + 16, 0);
    multiply(fa[1], fb[1]);
  }
  if (const int k0 = k_begin + turns * 32 * S; w == turns % 8 && k0 < k_end) {
    load(k0, fa[0], fb[0], Rest{});
    multiply(fa[0], fb[0]);
  }
  __syncthreads();
  f32x4(&red)[8][4][NG][64] = *reinterpret_cast<f32x4(*)[8][4][NG][64]>(lds);
#pragma unroll
  for (int t = 0; t < 4; ++t)
#pragma unroll
    for (int c = 0; c < NG; ++c) red[w][t][c][l] = acc[t][c];
  __syncthreads();
  float* out = g.partial + (int64_t)z * g.m * g.n;
#pragma unroll
  for (int v = threadIdx.x; v < 4 * NG * 64; v += 512) {
    // 16 neighbouring threads hold the 64 rows of a column
    const int quad = v % 16, in = v / 16, col = col0 + in, t = quad / 4;
    f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int y = 0; y < 8; ++y) sum += red[y][t][in / 16][(quad % 4) * 16 + in % 16];
    int row = row0 + quad * 4;
    const int chunk = row / CH * CH;      // (row0 is a multiple of 64)
    if (col >= g.n || chunk >= g.m) continue;
    if (LA == MC && chunk > last) row = last + row % CH;
    float* at = out + (int64_t)col * g.m + row;
    if (g.m % 4 == 0 && row < g.m) *reinterpret_cast<f32x4*>(at) = sum;
    else
      for (int e = 0; e < 4; ++e)
        if (row + e < g.m) at[e] = sum[e];
  }
}

// Sums of a split reduction in the order of the pieces, and the low-rank part: one output per thread, neighbouring rows side by
// side, 8 ranks at a time.
template <typename T> __global__ __launch_bounds__(256) void lora_few_join_kernel(HalfGemm g) {
  using E = typename T::elem;
  using x8 = typename T::x8;
  using f32x8 = float __attribute__((ext_vector_type(8)));
  const int row = blockIdx.x * 256 + threadIdx.x, col = blockIdx.y;
  if (row >= g.m) return;
  const int token = g.order[col], who = g.seg[col];
  const int64_t total = (int64_t)g.m * g.n;
  const float* from = g.partial + (int64_t)col * g.m + row;
  float sum = 0.0f;
  int z = 0;
  for (; z + 4 <= g.splits; z += 4) {
    float v[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) v[t] = from[(z + t) * total];
#pragma unroll
    for (int t = 0; t < 4; ++t) sum += v[t];
  }
  for (; z < g.splits; ++z) sum += from[z * total];
  if (who != g.none && g.rank > 0) {
    const E* up = static_cast<const E*>(g.up) + (int64_t)who * g.up_stride + (int64_t)row * g.up_row;
    const float* p = g.p + token * g.ldp;
    float d = 0.0f;
    for (int t = 0; t < g.rank; t += 8) {
      const bool whole = t + 8 <= g.rank;
      const f32x8 pv = whole ? load_8<float, f32x8>(p + t) : load_first<float, f32x8>(p + t, 1, g.rank - t);
      const x8 u = whole && g.up_rank == 1 ? load_8<E, x8>(up + t) : load_first<E, x8>(up + (int64_t)t * g.up_rank, g.up_rank, g.rank - t);
#pragma unroll
      for (int e = 0; e < 8; ++e) d += (float)u[e] * pv[e];
    }
    sum += g.scale[who] * d;
  }
  static_cast<E*>(g.c)[token * g.ldc + row] = (E)sum;
}

// The same for 16 columns at a time, the low-rank part on the matrix unit: the columns of one adapter (neighbours in the order of the
// plan) read its factor once.
template <typename T> __global__ __launch_bounds__(256) void lora_few_tile_join_kernel(HalfGemm g) {
  using E = typename T::elem;
  const int w = threadIdx.x / 64, l = threadIdx.x & 63;
  const int row0 = blockIdx.y * 64 + w * 16, col0 = blockIdx.x * 16;
  if (row0 >= g.m) return;
  f32x4 acc[1][1] = {};
  add_adapters<T, 1, 1>(g, row0, col0, acc);
  const int col = col0 + (l & 15), row = row0 + (l / 16) * 4;
  if (col >= g.n || row >= g.m) return;
  const int64_t total = (int64_t)g.m * g.n;
  const float* from = g.partial + (int64_t)col * g.m + row;
  f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
  const bool wide = g.m % 4 == 0;
  for (int z = 0; z < g.splits; ++z) {
    if (wide) {
      sum += *reinterpret_cast<const f32x4*>(from + z * total);
    } else {
      for (int t = 0; t < 4; ++t) sum[t] += from[z * total + (row + t < g.m ? t : 0)];
    }
  }
  sum += acc[0][0];
  E* at = static_cast<E*>(g.c) + (int64_t)g.order[col] * g.ldc + row;
  using e4 = E __attribute__((ext_vector_type(4)));
  if (wide && g.ldc % 4 == 0 && reinterpret_cast<uintptr_t>(g.c) % sizeof(e4) == 0) {
    *reinterpret_cast<e4*>(at) = __builtin_convertvector(sum, e4);
  } else {
    for (int t = 0; t < 4; ++t)
      if (row + t < g.m) at[t] = (E)sum[t];
  }
}

// One token with at most 32 ranks, W and its factor with a contiguous reduction: one launch.  A workgroup owns 16 rows; four of its
// waves take them, 4 rows each, in lines of 1 KB; the other four compute P, every workgroup for itself (from the caches), so that
// nothing has to be waited for and no sums go through memory: 2048 x 2048, rank 16 8.1 -> 6.1 us, 8192 x 8192 38 -> 33, 1024 x 16384
// 23 -> 17; with rank 32 as fast (4096 x 4096 12.9) but for the second launch, beyond slower.
constexpr int kTokenRanks = 32;
template <typename T> __global__ __launch_bounds__(512) void lora_token_kernel(HalfGemm g, ProjectArgs q) {
  using E = typename T::elem;
  using x8 = typename T::x8;
  __shared__ float y[16], p[kTokenRanks];
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), l = threadIdx.x & 63;
  const int row0 = blockIdx.x * 16, chunks = g.k / 8, token = g.order[0], who = g.seg[0], ranks = who != g.none ? g.rank : 0;
  const E* x = static_cast<const E*>(g.b) + (int64_t)token * g.ldb;
  // Sums of four rows with x: chunks of 8, two turns of 64 lanes under way together (four: 2048 x 2048 9.8 us), then what is left, one
  // a lane.
  auto dots = [&](const E* const (&row)[4], float (&sum)[4]) {
    constexpr int TURNS = 2;
    for (int c0 = 0; c0 < chunks; c0 += 64 * TURNS) {
      x8 a[TURNS][4], b[TURNS];
#pragma unroll
      for (int u = 0; u < TURNS; ++u) {
        const int c = c0 + u * 64 + l, at = (c < chunks ? c : chunks - 1) * 8;
#pragma unroll
        for (int v = 0; v < 4; ++v) a[u][v] = load_8<E, x8>(row[v] + at);
        b[u] = load_8<E, x8>(x + at);
      }
#pragma unroll
      for (int u = 0; u < TURNS; ++u) {
        const bool in = c0 + u * 64 + l < chunks;
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          float d = 0.0f;
#pragma unroll
          for (int e = 0; e < 8; ++e) d = __builtin_fmaf((float)a[u][v][e], (float)b[u][e], d);
          sum[v] += in ? d : 0.0f;
        }
      }
    }
    const int k = chunks * 8 + l;
    if (k < g.k) {
#pragma unroll
      for (int v = 0; v < 4; ++v) sum[v] += (float)row[v][k] * (float)x[k];
    }
#pragma unroll
    for (int v = 0; v < 4; ++v)
#pragma unroll
      for (int d = 1; d < 64; d *= 2) sum[v] += __shfl_xor(sum[v], d);
  };
  // this row's part of the other factor, on its way before anything is waited for
  const int row = row0 + threadIdx.x;
  const bool mine = threadIdx.x < 16 && row < g.m;
  x8 up[kTokenRanks / 8];
  if (mine) {
    const E* from = static_cast<const E*>(g.up) + (int64_t)who * g.up_stride + (int64_t)row * g.up_row;
#pragma unroll
    for (int r = 0; r < kTokenRanks; r += 8)
      if (r < ranks) up[r / 8] = load_first<E, x8>(from + (int64_t)r * g.up_rank, g.up_rank, ranks - r);
  }
  const E* rows[4];
  float sum[4] = {};
  if (w < 4) {
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      const int r = row0 + w * 4 + v;
      rows[v] = static_cast<const E*>(g.a) + (int64_t)(r < g.m ? r : g.m - 1) * g.lda;
    }
    dots(rows, sum);
#pragma unroll
    for (int v = 0; v < 4; ++v)
      if (l == 0) y[w * 4 + v] = sum[v];
  } else {
    for (int r0 = (w - 4) * 4; r0 < ranks; r0 += 16) {
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        rows[v] = static_cast<const E*>(q.a) + (int64_t)who * q.a_stride + (int64_t)(r0 + v < ranks ? r0 + v : ranks - 1) * q.a_row;
        sum[v] = 0.0f;
      }
      dots(rows, sum);
#pragma unroll
      for (int v = 0; v < 4; ++v)
        if (l == 0 && r0 + v < ranks) p[r0 + v] = sum[v];
    }
  }
  __syncthreads();
  if (blockIdx.x == 0 && q.p && (int)threadIdx.x < q.rank) q.p[(int64_t)token * q.ldp + threadIdx.x] = ranks ? p[threadIdx.x] : 0.0f;
  if (!mine) return;
  float out = y[threadIdx.x];
  if (ranks) {
    float d = 0.0f;
#pragma unroll
    for (int r = 0; r < kTokenRanks; ++r)
      if (r < ranks) d += (float)up[r / 8][r % 8] * p[r];
    out += g.scale[who] * d;
  }
  static_cast<E*>(g.c)[(int64_t)token * g.ldc + row] = (E)out;
}

// Pieces of the reduction, none shorter than 512 (eight waves, 64 positions each), at most 512 workgroups.
bool piece_allowed(int64_t blocks, int64_t k, int64_t pieces) {
  return pieces == 1 || (pieces <= 16 && k / pieces >= 512 && blocks * pieces <= 512);
}
// A compute unit runs one of these workgroups at a time, so the 64-row blocks times the pieces and the projection's workgroups
// should fill whole rounds of 256; a round costs what its piece does plus the latencies at both ends, about as much as 600
// positions (64 tokens x 4096 x 4096: 13.2 us, the call 17.5; with pieces for 512 at a time 16.8 and 21.9).
int few_pieces(int64_t m, int64_t n, int64_t k, int64_t project, int64_t* k_piece) {
  const int64_t blocks = (m + 63) / 64 * ((n + 63) / 64);
  int64_t best = 1, best_cost = INT64_MAX;
  for (int64_t pieces = 1; piece_allowed(blocks, k, pieces); ++pieces) {
    const int64_t piece = (k + pieces - 1) / pieces, cost = (blocks * pieces + project + 255) / 256 * (piece + 600);
    if (cost < best_cost) { best = pieces; best_cost = cost; }
  }
  *k_piece = std::max<int64_t>(((k + best - 1) / best + 63) / 64 * 64, 64);
  return (int)std::max<int64_t>((k + *k_piece - 1) / *k_piece, 1);
}
template <typename T, int LA, int NG> hipError_t launch_few_tokens(const HalfGemm& g, const ProjectArgs& q, hipStream_t s) {
  const int form = project_form<T>(q), slots = q.p ? (int)project_slots(q) : 0, project = slots * ((q.rank + 15) / 16);
  const dim3 grid((unsigned)(project + ((g.m + 63) / 64 * g.splits + 7) / 8 * 8 * ((g.n + 63) / 64)));
  if (form == A_K) hipLaunchKernelGGL((lora_few_kernel<T, LA, NG, A_K>), grid, dim3(512), 0, s, g, q, project, slots);
  if constexpr (T::bytes == 2) {
    if (form == A_R) hipLaunchKernelGGL((lora_few_kernel<T, LA, NG, A_R>), grid, dim3(512), 0, s, g, q, project, slots);
  }
  if (form == A_ANY) hipLaunchKernelGGL((lora_few_kernel<T, LA, NG, A_ANY>), grid, dim3(512), 0, s, g, q, project, slots);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  // Every output's own product with its factor's row, until that is the most of the call (167 tokens x 3264, 8 adapters: rank 16
  // 15.6 us, 16.7 with the matrix unit; rank 64 31.4, 18.7; 40 x 2048, rank 128 15.2, 17.2).
  if ((int64_t)g.m * g.n * g.rank > (int64_t)1 << 24)
    hipLaunchKernelGGL(lora_few_tile_join_kernel<T>, dim3((unsigned)((g.n + 15) / 16), (unsigned)((g.m + 63) / 64)), dim3(256), 0, s, g);
  else
    hipLaunchKernelGGL(lora_few_join_kernel<T>, dim3((unsigned)((g.m + 255) / 256), (unsigned)g.n), dim3(256), 0, s, g);
  return hipGetLastError();
}
template <typename T, int LA> hipError_t launch_few(HalfGemm g, const ProjectArgs& q, hipStream_t s) {
  if constexpr (LA == KC) {
    if (g.n == 1 && g.rank <= kTokenRanks && (g.rank == 0 || project_form<T>(q) == A_K)) {
      hipLaunchKernelGGL(lora_token_kernel<T>, dim3((unsigned)((g.m + 15) / 16)), dim3(512), 0, s, g, q);
      return hipGetLastError();
    }
  }
  int64_t piece;
  g.splits = few_pieces(g.m, g.n, g.k, q.p ? project_slots(q) * ((q.rank + 15) / 16) : 0, &piece);
  g.k_piece = (int)piece;
  return g.n <= 16 ? launch_few_tokens<T, LA, 1>(g, q, s) : g.n <= 32 ? launch_few_tokens<T, LA, 2>(g, q, s) : launch_few_tokens<T, LA, 4>(g, q, s);
}

}  // namespace

// Up to 64 tokens, and beyond as long as this is one round and quicker than large tiles with the projection in front of them: 3 us,
// and 5 + 4.4 per thousand positions a round, against the plan's time, 6 us and 1.25 per thousand positions for the projection
// (256 tokens x 1024 x 1024 18.7 -> 10.4 us, 142 x 2456 x 4032 29.6 -> 17.9, 192 x 4096 x 4096 31.5 -> 25.1; not 96 x 4096 x 16384,
// 62.5 -> 69.2).
// The projection counts with the workgroups that n tokens of one adapter take, however many there are: with many adapters the large
// tiles lose more than it takes (100 x 4096 x 4096, 48 adapters of rank 128 67 -> 186 us, 200 x 2048 x 2048, rank 64 25 -> 53).
bool lora_few_half(int64_t m, int64_t n, int64_t k) {
  if (n <= 64) return true;
  const int64_t blocks = (m + 63) / 64 * ((n + 63) / 64), project = n / kProjTokens;
  if (blocks + project > 256) return false;
  int64_t piece;
  const int64_t pieces = few_pieces(m, n, k, project, &piece), rounds = (blocks * pieces + project + 255) / 256;
  return 3.0 + (double)rounds * (5.0 + 4.4e-3 * (double)piece) < plan_tiles(m, n, k).us + 6.0 + 1.25e-3 * (double)k;
}
// Single precision, against the library's product with the projection and the low-rank part around it.  Measured: 19 us, 19.5 per
// thousand positions a round where W's reduction is contiguous and 21.8 where its rows are (4 % more in a single round), and the
// projection's workgroups in front, 0.06 per thousand positions each; the product takes 1.02 times its model, 1.27 where tiles are not
// whole, 8 us and 2 per thousand positions around it (777 tokens x 1024 x 1536 72 -> 46 us, 2000 x 1000 x 2048 132 -> 111; not 768 x 2048 x
// 2048, 93 and 109).  Within 3 % it is this one.  More tokens bring more of the projection than of W (8192 x 128 x 2048 80 and 126).
bool lora_few_f32(bool w_trans, int64_t m, int64_t n, int64_t k) {
  const int64_t blocks = (m + 63) / 64 * ((n + 63) / 64), project = n / kProjTokens;
  if (n <= 64) return true;
  if (blocks > (n > 2048 ? 256 : 512) || n > 5120) return false;
  int64_t piece;
  const int64_t pieces = few_pieces(m, n, k, project, &piece);
  const double rounds = blocks * pieces <= 256 ? 1.04 : pieces > 1 ? (double)(blocks * pieces) / 256.0 : 2.0;
  const double us = 19.0 + rounds * (w_trans ? 19.5e-3 : 21.8e-3) * (double)piece + 6e-5 * (double)(project * k);
  const bool whole = m % 128 == 0 && n % 128 == 0;
  return us < 1.03 * (modelled_gemm_f32(m, n, k) * (whole ? 1.02 : 1.27) + 8.0 + 2e-3 * (double)k);
}
int64_t lora_few_work_bytes(int64_t m, int64_t n, int64_t k) {
  int64_t pieces = 1;
  while (piece_allowed((m + 63) / 64 * ((n + 63) / 64), k, pieces + 1)) ++pieces;
  return pieces * m * n * 4;
}

hipError_t lora_few_device(int kind, bool w_trans, const HalfGemm& g, const ProjectArgs& q, hipStream_t s) {
  if (kind != BF16 && kind != F16K) return w_trans ? launch_few<Fp32, KC>(g, q, s) : launch_few<Fp32, MC>(g, q, s);
  if (kind == BF16) return w_trans ? launch_few<Bf16, KC>(g, q, s) : launch_few<Bf16, MC>(g, q, s);
  return w_trans ? launch_few<F16, KC>(g, q, s) : launch_few<F16, MC>(g, q, s);
}

}  // namespace eigamd
