// The projection of the adapter product, P(:,i) = op(A_j) x_i: the body that its own launch and the few-token launch share.
#pragma once
#include "half.hpp"

namespace eigamd {

constexpr int kProjTokens = 32;
struct ProjectArgs {
  int n, k, rank, none;
  const void* x; int64_t ldx;
  const void* a; int64_t a_row, a_k, a_stride;    // strides of op(A_j)(r, k) and of j
  const int* order;
  const int* starts;
  float* p; int64_t ldp;
};

// P for up to 32 tokens of one adapter and 16 RT ranks.  Eight waves share the reduction, 128 (down to 32) positions a turn, each straight
// from memory to the matrix unit: one load of a wave is 64 bytes of each of 16 tokens.  The next turn's loads are under way
// while this one's are multiplied.
//   A_K   the factor's reduction is contiguous: loaded like the tokens
//   A_R   its ranks are (the backward pass): whole 16-byte chunks of ranks go through this wave's own LDS and come back
//         transposed; one element at a time instead, the loads of a 64-rank factor took four times the rest (57 us of 4096 tokens
//         x 4096, now 18)
//   A_ANY element by element: ranks that are no multiple of 8, odd strides
enum { A_K, A_R, A_ANY };
constexpr int project_lds(int rt) { return 8 * rt * 2 * 64 * 16; }
template <typename T, int RT, int FORM> __device__ __forceinline__ void project_piece(const ProjectArgs& g, int slot_id, int r0, char* lds) {
  using E = typename T::elem;
  using x8 = typename T::x8;
  Piece piece;
  if (!find_piece(g.starts, g.none + 1, kProjTokens, slot_id, piece)) return;
  const int w = threadIdx.x / 64, l = threadIdx.x & 63;
  constexpr int line = RT * 32;                      // A_R: 32 positions x 16 RT ranks per wave
  static_assert(8 * 32 * line <= project_lds(RT), "transposition and sums share LDS");
  f32x4(&red)[8][RT][2][64] = *reinterpret_cast<f32x4(*)[8][RT][2][64]>(lds);
  const bool live = piece.adapter != g.none;
  if (live) {
    // lanes past the piece or the rank repeat the last one; what they compute is not stored
    f32x4 acc[RT][2] = {};
    const E* x[2];
    const E* a[RT];
    const E* factor = static_cast<const E*>(g.a) + (int64_t)piece.adapter * g.a_stride;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int at = piece.begin + c * 16 + (l & 15);
      x[c] = static_cast<const E*>(g.x) + (int64_t)g.order[at < piece.end ? at : piece.end - 1] * g.ldx;
    }
    constexpr int per = RT * 2;                              // A_R: 16-byte chunks of a line
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      if constexpr (FORM == A_R) {
        // chunk t * 64 + l of 32 lines
        const int ch = t * 64 + l, r = r0 + (ch % per) * 8;
        a[t] = factor + (int64_t)(ch / per) * g.a_k + (r < g.rank ? r : 0);
      } else {
        const int r = r0 + t * 16 + (l & 15);
        a[t] = factor + (int64_t)(r < g.rank ? r : g.rank - 1) * g.a_row;
      }
    }
    constexpr int S = T::bytes == 4 ? (RT == 1 ? 2 : 1) : RT == 4 ? 2 : 4, turn = 8 * 32 * S;      // products of a turn; positions all waves take in one
    x8 fx[2][S][2], fa[2][S][RT];
    auto load = [&](int k0, int set) {
      const bool whole = k0 + 32 * S <= g.k;
#pragma unroll
      for (int s = 0; s < S; ++s) {
        const int k = k0 + s * 32 + (l / 16) * 8, left = g.k - k;
#pragma unroll
        for (int c = 0; c < 2; ++c) fx[set][s][c] = whole ? load_8<E, x8>(x[c] + k) : load_up_to_8<E, x8>(x[c] + k, left);
#pragma unroll
        for (int t = 0; t < RT; ++t) {
          if constexpr (FORM == A_K) {
            fa[set][s][t] = whole ? load_8<E, x8>(a[t] + k) : load_up_to_8<E, x8>(a[t] + k, left);
          } else if constexpr (FORM == A_R) {
            const int at = k0 + s * 32 + (t * 64 + l) / per;
            fa[set][s][t] = load_up_to_8<E, x8>(a[t] + (int64_t)(k0 + s * 32) * g.a_k, at < g.k ? 8 : 0);
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) fa[set][s][t][e] = e < left ? a[t][(int64_t)(k + e) * g.a_k] : (E)0.0f;
          }
        }
      }
    };
    auto multiply = [&](int set) {
#pragma unroll
      for (int s = 0; s < S; ++s) {
        x8 f[RT];
        if constexpr (FORM == A_R) {
          char* mine = lds + w * 32 * line;
          auto slot = [&](int ln, int ch) { return ln * line + ((ch ^ ((ln & 3) << 1)) & (per - 1)) * 16; };
#pragma unroll
          for (int t = 0; t < RT; ++t) *reinterpret_cast<x8*>(mine + slot((t * 64 + l) / per, (t * 64 + l) % per)) = fa[set][s][t];
#pragma unroll
          for (int t = 0; t < RT; ++t) {
            union { x8 v; typename T::x4 h[2]; } u;
            const int ln = (l / 16) * 8 + (l & 15) / 4, ch = t * 2 + (l & 3) / 2;
#pragma unroll
            for (int h = 0; h < 2; ++h) u.h[h] = T::read_transposed(mine + slot(ln + 4 * h, ch) + (l & 1) * 8);
            f[t] = u.v;
          }
        } else {
#pragma unroll
          for (int t = 0; t < RT; ++t) f[t] = fa[set][s][t];
        }
#pragma unroll
        for (int t = 0; t < RT; ++t)
#pragma unroll
          for (int c = 0; c < 2; ++c) acc[t][c] = T::mma(f[t], fx[set][s][c], acc[t][c]);
      }
    };
    int k0 = w * 32 * S;
    if (k0 < g.k) load(k0, 0);
    for (; k0 < g.k; k0 += 2 * turn) {
      if (k0 + turn < g.k) load(k0 + turn, 1);
      multiply(0);
      if (k0 + turn >= g.k) break;
      if (k0 + 2 * turn < g.k) load(k0 + 2 * turn, 0);
      multiply(1);
    }
    if constexpr (FORM == A_R) __syncthreads();              // (the same LDS; `live` is the workgroup's)
#pragma unroll
    for (int t = 0; t < RT; ++t)
#pragma unroll
      for (int c = 0; c < 2; ++c) red[w][t][c][l] = acc[t][c];
  }
  __syncthreads();
  for (int q = threadIdx.x; q < RT * 2 * 64; q += 512) {
    const int t = q / 128, c = (q / 64) % 2, at = piece.begin + c * 16 + (l & 15);
    if (at >= piece.end) continue;
    f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
    if (live)
      for (int z = 0; z < 8; ++z) sum += red[z][t][c][l];
    const int r = r0 + t * 16 + (l / 16) * 4;
    float* out = g.p + (int64_t)g.order[at] * g.ldp + r;
    for (int e = 0; e < 4; ++e)
      if (r + e < g.rank) out[e] = sum[e];
  }
}

inline int64_t project_slots(const ProjectArgs& g) { return g.n / kProjTokens + g.none + 1; }
template <typename T> int project_form(const ProjectArgs& g) {
  if (g.a_k == 1) return A_K;
  const bool chunks = g.a_row == 1 && g.a_k % 8 == 0 && g.rank % 8 == 0 && g.a_stride % 8 == 0 && (uintptr_t)g.a % 16 == 0;
  return T::bytes == 2 && chunks ? A_R : A_ANY;
}

}  // namespace eigamd
