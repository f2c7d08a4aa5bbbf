// The projection of the adapter product, P(:,i) = op(A_j) x_i: the body that its own launch and the few-token launch share.
#pragma once
#include <type_traits>

#include "half.hpp"

namespace eigamd {

constexpr int kProjTokens = 32, kProjWaves = 8;
struct ProjectArgs {
  int n, k, rank, none;
  const void* x; int64_t ldx;
  const void* a; int64_t a_row, a_k, a_stride;    // strides of op(A_j)(r, k) and of j
  const int* order;
  const int* seg;
  const int* starts;
  float* p; int64_t ldp;                          // nullptr: no adapters, and nobody who wants the zeros
};

// 16 rows x 32 S positions on their way from memory to the matrix unit.  A fragment has neighbouring lanes on different rows; loaded
// so, a load takes the memory pipeline 64 cycles, a row's address at a time.  Here 4 S neighbouring lanes take 64 S bytes (128 of
// single precision) of one row, S loads a block, and the wave's own LDS turns them into fragments (the projection of 32 tokens x 4032
// to 16 ranks: 15 us, now 9); chunks of a row are permuted so that the 16 lanes that read together meet all banks once.
template <typename T, int S = 1> struct RowBlock {
  using x8 = typename T::x8;
  static_assert(S == 1 || (S == 2 && T::bytes == 2), "rows of 64 or 128 bytes");
  static constexpr int bytes = 512 * S * T::bytes;
  static __device__ __forceinline__ int row(int load = 0) { return load * (16 / S) + (threadIdx.x & 63) / (4 * S); }
  static __device__ __forceinline__ int position() { return threadIdx.x % (4 * S) * 8; }
  static __device__ __forceinline__ int at(int row, int chunk) {       // of 16 bytes
    return S * T::bytes == 2 ? row * 64 + (chunk ^ ((row / 4) & 3)) * 16 : row * 128 + (chunk ^ ((row / 2) & 7)) * 16;
  }
  static __device__ __forceinline__ void put(char* lds, x8 v, int load = 0) {
    constexpr int H = T::bytes / 2;
    const Half<x8> u = __builtin_bit_cast(Half<x8>, v);
#pragma unroll
    for (int h = 0; h < H; ++h) *reinterpret_cast<f32x4*>(lds + at(row(load), threadIdx.x % (4 * S) * H + h)) = u.part[h];
  }
  static __device__ __forceinline__ x8 get(const char* lds, int step = 0) {
    const int l = threadIdx.x & 63;
    constexpr int H = T::bytes / 2;
    Half<x8> u;
#pragma unroll
    for (int h = 0; h < H; ++h) u.part[h] = *reinterpret_cast<const f32x4*>(lds + at(l % 16, step * 4 + (l / 16) * H + h));
    return __builtin_bit_cast(x8, u);
  }

 private:
  template <typename V> struct Half { f32x4 part[sizeof(V) / 16]; };
};

// P for up to 32 tokens of one adapter and 16 RT ranks.  Eight waves share the reduction, 128 (down to 32) positions a turn.  The next
// turn's loads are under way while this one's are multiplied.
//   A_K   the factor's reduction is contiguous: loaded like the tokens
//   A_R   its ranks are (the backward pass): whole 16-byte chunks of ranks go through this wave's own LDS and come back
//         transposed; one element at a time instead, the loads of a 64-rank factor took four times the rest (57 us of 4096 tokens
//         x 4096, now 15)
//   A_ANY element by element: ranks that are no multiple of 8, odd strides
enum { A_K, A_R, A_ANY };
constexpr int project_lds(int rt, int bytes) { return kProjWaves * (rt * 2048 > (2 + rt) * 512 * bytes ? rt * 2048 : (2 + rt) * 512 * bytes); }
template <typename T, int RT, int FORM> __device__ __forceinline__ void project_piece(const ProjectArgs& g, int slot_id, int r0, char* lds) {
  using E = typename T::elem;
  using x8 = typename T::x8;
  Piece piece;
  if (!(g.n <= g.none ? find_piece_by_tokens<kProjTokens>(g.seg, g.n, slot_id, piece) : find_piece(g.starts, g.none + 1, kProjTokens, slot_id, piece))) return;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), l = threadIdx.x & 63;
  constexpr int line = RT * 32;                      // A_R: 32 positions x 16 RT ranks per wave
  f32x4(&red)[kProjWaves][RT][2][64] = *reinterpret_cast<f32x4(*)[kProjWaves][RT][2][64]>(lds);
  const bool live = piece.adapter != g.none;
  if (live) {
    // lanes past the piece or the rank repeat the last one; what they compute is not stored
    f32x4 acc[RT][2] = {};
    const E* x[2];
    const E* a[RT];
    const E* factor = static_cast<const E*>(g.a) + (int64_t)piece.adapter * g.a_stride;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int at = piece.begin + c * 16 + RowBlock<T>::row();
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
        const int r = r0 + t * 16 + (FORM == A_K ? RowBlock<T>::row() : l & 15);
        a[t] = factor + (int64_t)(r < g.rank ? r : g.rank - 1) * g.a_row;
      }
    }
    // Turns of S products.  Whole turns and what is left behind the last one (up to S products, one a wave) are loaded by code of
    // their own: a bound on every load of the loop made it several times as long, and fetching it was most of a short call.
    constexpr int S = T::bytes == 4 ? (RT == 1 ? 2 : 1) : RT == 4 ? 2 : 4;
    static_assert(S <= kProjWaves, "one product a wave");
    using Whole = std::true_type;
    using Rest = std::false_type;
    auto load = [&](int k0, x8(&fx)[2], x8(&fa)[RT], auto whole) {
      int k = k0 + RowBlock<T>::position(), left = g.k - k;
#pragma unroll
      for (int c = 0; c < 2; ++c) fx[c] = whole ? load_8<E, x8>(x[c] + k) : load_first<E, x8>(x[c] + (left > 0 ? k : 0), 1, left);
#pragma unroll
      for (int t = 0; t < RT; ++t) {
        if constexpr (FORM == A_R) {
          const bool in = whole || k0 + (t * 64 + l) / per < g.k;
          x8 v = load_8<E, x8>(in ? a[t] + (int64_t)k0 * g.a_k : factor);
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = in ? v[e] : (E)0.0f;
          fa[t] = v;
        } else if constexpr (FORM == A_K && whole) {
          fa[t] = load_8<E, x8>(a[t] + k);
        } else {
          if constexpr (FORM == A_ANY) {
            k = k0 + (l / 16) * 8;
            left = g.k - k;
          }
          fa[t] = load_first<E, x8>(a[t] + (left > 0 ? (int64_t)k * g.a_k : 0), g.a_k, whole ? 8 : left);
        }
      }
    };
    auto multiply = [&](const x8(&fx)[2], const x8(&fa)[RT]) {
      char* mine = lds + w * (2 + RT) * RowBlock<T>::bytes;      // X's two blocks, then the factor's
      x8 f[RT], y[2];
      wave_order();
#pragma unroll
      for (int c = 0; c < 2; ++c) RowBlock<T>::put(mine + c * RowBlock<T>::bytes, fx[c]);
      char* own = mine + 2 * RowBlock<T>::bytes;
      if constexpr (FORM == A_R) {
        auto slot = [&](int ln, int ch) { return ln * line + ((ch ^ ((ln & 3) << 1)) & (per - 1)) * 16; };
#pragma unroll
        for (int t = 0; t < RT; ++t) *reinterpret_cast<x8*>(own + slot((t * 64 + l) / per, (t * 64 + l) % per)) = fa[t];
        wave_order();
#pragma unroll
        for (int t = 0; t < RT; ++t) {
          union { x8 v; typename T::x4 h[2]; } u;
          const int ln = (l / 16) * 8 + (l & 15) / 4, ch = t * 2 + (l & 3) / 2;
#pragma unroll
          for (int h = 0; h < 2; ++h) u.h[h] = T::read_transposed(own + slot(ln + 4 * h, ch) + (l & 1) * 8);
          f[t] = u.v;
        }
      } else if constexpr (FORM == A_K) {
#pragma unroll
        for (int t = 0; t < RT; ++t) RowBlock<T>::put(own + t * RowBlock<T>::bytes, fa[t]);
        wave_order();
#pragma unroll
        for (int t = 0; t < RT; ++t) f[t] = RowBlock<T>::get(own + t * RowBlock<T>::bytes);
      } else {
        wave_order();
#pragma unroll
        for (int t = 0; t < RT; ++t) f[t] = fa[t];
      }
#pragma unroll
      for (int c = 0; c < 2; ++c) y[c] = RowBlock<T>::get(mine + c * RowBlock<T>::bytes);
#pragma unroll
      for (int t = 0; t < RT; ++t)
#pragma unroll
        for (int c = 0; c < 2; ++c) acc[t][c] = T::mma(f[t], y[c], acc[t][c]);
    };
    x8 fx[2][S][2], fa[2][S][RT];
    auto load_turn = [&](int turn, int set) {
#pragma unroll
      for (int s = 0; s < S; ++s) load((turn * S + s) * 32, fx[set][s], fa[set][s], Whole{});
    };
    auto multiply_turn = [&](int set) {
#pragma unroll
      for (int s = 0; s < S; ++s) multiply(fx[set][s], fa[set][s]);
    };
    const int turns = g.k / (32 * S);
    int at = w;
    if (at < turns) load_turn(at, 0);
    for (; at < turns; at += 2 * kProjWaves) {
      if (at + kProjWaves < turns) load_turn(at + kProjWaves, 1);
      multiply_turn(0);
      if (at + kProjWaves >= turns) break;
      if (at + 2 * kProjWaves < turns) load_turn(at + 2 * kProjWaves, 0);
      multiply_turn(1);
    }
    if ((turns * S + w) * 32 < g.k) {
      load((turns * S + w) * 32, fx[0][0], fa[0][0], Rest{});
      multiply(fx[0][0], fa[0][0]);
    }
    __syncthreads();              // (the sums take the same LDS; `live` is the workgroup's)
#pragma unroll
    for (int t = 0; t < RT; ++t)
#pragma unroll
      for (int c = 0; c < 2; ++c) red[w][t][c][l] = acc[t][c];
  }
  __syncthreads();
  const bool wide = g.ldp % 4 == 0 && (reinterpret_cast<uintptr_t>(g.p) & 15) == 0;
  for (int q = threadIdx.x; q < RT * 2 * 64; q += kProjWaves * 64) {
    const int t = q / 128, c = (q / 64) % 2, at = piece.begin + c * 16 + (l & 15);
    if (at >= piece.end) continue;
    f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
    if (live)
      for (int z = 0; z < kProjWaves; ++z) sum += red[z][t][c][l];
    const int r = r0 + t * 16 + (l / 16) * 4;
    float* out = g.p + (int64_t)g.order[at] * g.ldp + r;
    if (wide && r + 4 <= g.rank) {
      *reinterpret_cast<f32x4*>(out) = sum;
    } else {
      for (int e = 0; e < 4; ++e)
        if (r + e < g.rank) out[e] = sum[e];
    }
  }
}

inline int64_t project_slots(const ProjectArgs& g) { return g.n / kProjTokens + (g.n <= g.none ? g.n : g.none + 1); }
template <typename T> int project_form(const ProjectArgs& g) {
  if (g.a_k == 1) return A_K;
  const bool chunks = g.a_row == 1 && g.a_k % 8 == 0 && g.rank % 8 == 0 && g.a_stride % 8 == 0 && (uintptr_t)g.a % 16 == 0;
  return T::bytes == 2 && chunks ? A_R : A_ANY;
}

}  // namespace eigamd
