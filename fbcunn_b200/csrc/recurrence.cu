// A gated linear recurrence along sequences (sm_100a).
//
//   a_t = sigmoid(g_t + bias),  h_t = a_t h_{t-1} + (1 - a_t) x_t,  y_t = h_t z_t sigmoid(z_t)   (y_t = h_t without z)
// and backward, from dy and the gradient by the last state:
//   e_t = dy_t silu(z_t) [+ dstate at a sequence's last row],  D_t = e_t + a_{t+1} D_{t+1} (0 behind the last row)
//   dx = (1 - a) D,  dg = D (h_{t-1} - x) a (1 - a),  dz = dy h silu'(z),  dbias = sum dg,  dstate0 = a_first D_first
//
// All sequences lie one behind the other in one array of rows; a row that begins one takes the initial state instead of
// the row before.  h -> A h + H describes any stretch of rows, so a warp takes `kRows` rows of 64 (fp32: 32) channels,
// a lane two neighbours of them, and the stretches are joined in a block (shared memory), in a cluster of blocks
// (distributed shared memory) and, from one round of rows to the next, in registers: one pass over memory, in an order
// that only the sizes decide.  The rows of the next round are under way (cp.async, by the thread that will use them)
// while this one is computed.  HBM bounds it: some 30 instructions an element against 8 bytes forward, 60 against 14
// backward.  1 - a is formed first where a is the larger, so that a + (1 - a) = 1 to the last place and long memories
// do not drift.
#include <cooperative_groups.h>
#include <math.h>

#include <type_traits>

#include "operators.cuh"

namespace cg = cooperative_groups;

namespace fbfft {
namespace {

constexpr int kWarps = 8, kThreads = 32 * kWarps;
constexpr int kForwardRows = 16, kBackwardRows = 8;  // of a warp, in a round
constexpr int kCheckpoint = 64;                      // rows between the states that forward leaves for backward
constexpr int kMostCluster = 8;
static_assert(kCheckpoint % kForwardRows == 0 && kWarps * kBackwardRows == kCheckpoint && (kWarps * kForwardRows) % kCheckpoint == 0);

struct RecArgs {
  const void* x;
  const void* g;
  const void* z;
  const float* bias;
  const float* state0;   // [sequence][channel] or null
  const void* offsets;   // [sequences + 1], or null: sequences of `length` rows
  // forward
  void* y;
  float* state;          // [sequence][channel] or null
  float* checkpoints;    // [checkpoint][channel] or null
  // backward
  const void* dy;
  const float* dstate;   // or null
  void* dx;
  void* dg;
  void* dz;
  float* dstate0;        // or null
  float* sums;           // [part][channel] of dbias, or null
  long long rows, length, sequences;
  long long x_stride, g_stride, z_stride, y_stride, dy_stride, dx_stride, dg_stride, dz_stride;
  long long per_segment; // sequences of a segment
  long long checkpoints_per_segment;
  int channels, wide_offsets, cluster;
};

__device__ __forceinline__ long long offset_at(const RecArgs& a, long long i) {
  const long long v = a.wide_offsets ? static_cast<const long long*>(a.offsets)[i] : static_cast<const int*>(a.offsets)[i];
  return v < 0 ? 0 : v > a.rows ? a.rows : v;  // a bad offset must not lead out of the tensors
}

// The sequence that a row belongs to, and the rows where it begins and ends.
struct Sequence {
  long long index, begin, end;
};
__device__ __forceinline__ Sequence sequence_of(const RecArgs& a, long long row) {
  if (!a.offsets) {
    const long long i = (a.rows | a.length) >> 32 ? row / a.length : (uint32_t)row / (uint32_t)a.length;
    return {i, i * a.length, (i + 1) * a.length};
  }
  long long lo = 0, hi = a.sequences;  // the last one that begins at or before the row
  while (hi - lo > 1) {
    const long long mid = (lo + hi) >> 1;
    if (offset_at(a, mid) <= row) lo = mid;
    else hi = mid;
  }
  return {lo, offset_at(a, lo), offset_at(a, lo + 1)};
}

// Which of n rows from `row` on begin a sequence, and which end one.
__device__ __forceinline__ void borders(const RecArgs& a, long long row, int n, uint32_t& first, uint32_t& last) {
  first = last = 0;
  if (n <= 0) return;
  Sequence s = sequence_of(a, row);
  if (row == s.begin) first = 1;
  while (s.end > row && s.end - row <= n) {
    const int k = (int)(s.end - row);
    last |= 1u << (k - 1);
    if (k == n) break;
    first |= 1u << k;
    const Sequence next = sequence_of(a, s.end);
    if (next.end <= s.end) break;  // offsets that do not rise
    s = next;
  }
}

// h -> A h + H; A < 0 stands for rows that begin a sequence among them: nothing of h comes through, not even a NaN.
struct Stretch {
  float A, H;
};
__device__ __forceinline__ float apply(const Stretch& s, float h) { return s.A < 0.f ? s.H : fmaf(s.A, h, s.H); }
__device__ __forceinline__ Stretch join(const Stretch& s, const Stretch& next) {
  return {next.A < 0.f || s.A < 0.f ? -1.f : s.A * next.A, apply(next, s.H)};
}

__device__ __forceinline__ float reciprocal(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// a = sigmoid(g) and b = 1 - a, both to the last places: the larger is formed from the smaller.
__device__ __forceinline__ void gate_of(float g, float& a, float& b) {
  const float e = __expf(-fabsf(g));
  const float small = e * reciprocal(1.f + e), big = 1.f - small;
  a = g < 0.f ? small : big;
  b = g < 0.f ? big : small;
}

__device__ __forceinline__ float sigmoid(float x) { return reciprocal(1.f + __expf(-x)); }

// A lane's channels of a row: one 32-bit word, or a single 16-bit value where pairs are not aligned.
template <typename T, int V> __device__ __forceinline__ void unpack(uint32_t w, float (&x)[V]) {
  if constexpr (std::is_same_v<T, float>) {
    x[0] = __uint_as_float(w);
  } else if constexpr (V == 2) {
    const float2 f = unpack2<T>(w);
    x[0] = f.x, x[1] = f.y;
  } else {
    x[0] = unpack2<T>(w).x;
  }
}
template <typename T, int V> __device__ __forceinline__ uint32_t load_word(const T* p) {
  if constexpr (sizeof(T) * V == 4) return __ldg(reinterpret_cast<const uint32_t*>(p));
  else return __ldg(reinterpret_cast<const uint16_t*>(p));
}
template <typename T, int V> __device__ __forceinline__ void store_word(T* p, const float (&x)[V]) {
  if constexpr (std::is_same_v<T, float>) *p = x[0];
  else if constexpr (V == 2) *reinterpret_cast<uint32_t*>(p) = pack2<T>(x[0], x[1]);
  else *p = from_float<T>(x[0]);
}

// The words of a thread's next rows: in shared memory, on their way there while this round is computed.  Single 16-bit
// values, which cp.async does not copy, are loaded where they are read.
template <typename T, int V, int kRows, int kStreams>
struct Words {
  static constexpr bool kAsync = sizeof(T) * V == 4;
  static constexpr int kStage = kStreams * kRows * kThreads * 4;
  char* base;  // this thread's
  const T* at[kStreams];      // the thread's channels of row 0
  long long stride[kStreams];

  __device__ __forceinline__ void fetch(int stage, long long row, int n, bool on) const {
    if constexpr (kAsync) {
      if (on) {
#pragma unroll
        for (int s = 0; s < kStreams; ++s) {
          const T* p = at[s] + row * stride[s];
          const uint32_t to = (uint32_t)__cvta_generic_to_shared(base + stage * kStage + s * kRows * kThreads * 4);
#pragma unroll
          for (int i = 0; i < kRows; ++i)
            if (i < n)
              asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(to + i * kThreads * 4), "l"(p + i * stride[s]) : "memory");
        }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    }
  }
  __device__ __forceinline__ void wait() const {
    if constexpr (kAsync) asm volatile("cp.async.wait_group 1;" ::: "memory");
  }
  // i below the rows that there are
  __device__ __forceinline__ void read(int stage, int s, long long row, int i, float (&x)[V]) const {
    if constexpr (kAsync) unpack<T, V>(*reinterpret_cast<const uint32_t*>(base + stage * kStage + (s * kRows + i) * kThreads * 4), x);
    else unpack<T, V>(load_word<T, V>(at[s] + (row + i) * stride[s]), x);
  }
};

// Joins what the warps and blocks before one have: a block's warps through `part`, a cluster's blocks through `whole`.
// "Before" is in the direction of the scan; `order` counts in it.  Two halves are used in turn.
template <int V>
struct Exchange {
  Stretch part[2][kWarps][32][V];
  Stretch whole[2][kMostCluster][32][V];
};

// `mine`: this warp's stretch; returns the value that enters it and moves `carry` behind the whole round.
template <int V>
__device__ __forceinline__ void exchange(Exchange<V>& x, int half, int order, int rank, int blocks, const Stretch (&mine)[V],
                                         float (&carry)[V], float (&enter)[V]) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int v = 0; v < V; ++v) x.part[half][order][lane][v] = mine[v];
  __syncthreads();
  Stretch before[V], all[V];
#pragma unroll
  for (int v = 0; v < V; ++v) all[v] = before[v] = Stretch{1.f, 0.f};
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      if (w == order) before[v] = all[v];
      all[v] = join(all[v], x.part[half][w][lane][v]);
    }
  }
  if (blocks == 1) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      enter[v] = apply(before[v], carry[v]);
      carry[v] = apply(all[v], carry[v]);
    }
    return;
  }
  cg::cluster_group cluster = cg::this_cluster();
  if (order < blocks) {
    Exchange<V>* const other = cluster.map_shared_rank(&x, order);
#pragma unroll
    for (int v = 0; v < V; ++v) other->whole[half][rank][lane][v] = all[v];
  }
  cluster.sync();
#pragma unroll
  for (int v = 0; v < V; ++v) {
    float h = carry[v];
    enter[v] = h;
    for (int k = 0; k < blocks; ++k) {
      if (k == rank) enter[v] = h;
      h = apply(x.whole[half][k][lane][v], h);
    }
    enter[v] = apply(before[v], enter[v]);
    carry[v] = h;
  }
}

// The rows of this block's segment: [begin, end).
__device__ __forceinline__ void segment_rows(const RecArgs& a, long long& begin, long long& end) {
  if (a.offsets) {
    begin = offset_at(a, 0);
    end = offset_at(a, a.sequences);
  } else {
    const long long first = (long long)blockIdx.y * a.per_segment;
    const long long last = min(first + a.per_segment, a.sequences);
    begin = first * a.length, end = last * a.length;
  }
}

// Sequences without rows hand their state on.
template <int V>
__device__ __forceinline__ void pass_empty(const RecArgs& a, const float* from, float* to, int channel, bool on) {
  if (!to || blockIdx.y || (!a.offsets && a.length > 0)) return;
  for (long long s = threadIdx.x >> 5; s < a.sequences; s += kWarps) {
    if (a.offsets && offset_at(a, s + 1) > offset_at(a, s)) continue;
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (on) to[s * a.channels + channel + v] = from ? from[s * a.channels + channel + v] : 0.f;
  }
}

template <typename T, int V, bool kGate>
__global__ void __launch_bounds__(kThreads, 2) recurrence_forward_kernel(const RecArgs a) {
  constexpr int L = kForwardRows, kTile = kWarps * L, kStreams = kGate ? 3 : 2;
  extern __shared__ __align__(16) char staged[];
  __shared__ Exchange<V> shared;
  grid_dependency_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int blocks = a.cluster, rank = blockIdx.x % blocks;
  const int channel = (blockIdx.x / blocks * 32 + lane) * V;
  const bool on = channel < a.channels;
  const int c = on ? channel : 0;
  long long begin, end;
  segment_rows(a, begin, end);
  if (rank == 0) pass_empty<V>(a, a.state0, a.state, c, on);
  const long long tiles = (end - begin + kTile - 1) / kTile, rounds = (tiles + blocks - 1) / blocks;
  Words<T, V, L, kStreams> words;
  words.base = staged + 4 * threadIdx.x;
  words.at[0] = static_cast<const T*>(a.x) + c, words.stride[0] = a.x_stride;
  words.at[1] = static_cast<const T*>(a.g) + c, words.stride[1] = a.g_stride;
  if (kGate) words.at[kStreams - 1] = static_cast<const T*>(a.z) + c, words.stride[kStreams - 1] = a.z_stride;
  float bias[V], carry[V];
#pragma unroll
  for (int v = 0; v < V; ++v) bias[v] = a.bias ? a.bias[c + v] : 0.f, carry[v] = 0.f;
  const auto row_of = [&](long long round) { return begin + ((round * blocks + rank) * kWarps + warp) * L; };
  const auto rows_at = [&](long long row) { return (int)max(0ll, min((long long)L, end - row)); };
  for (int k = 0; k < 2; ++k) words.fetch(k, row_of(k), rows_at(row_of(k)), on);
  for (long long round = 0; round < rounds; ++round) {
    const int stage = (int)(round & 1);
    const long long row = row_of(round);
    const int n = rows_at(row);
    words.wait();
    uint32_t first, last;
    borders(a, row, n, first, last);
    float A[L][V], B[L][V];
    Stretch mine[V];
#pragma unroll
    for (int v = 0; v < V; ++v) mine[v] = Stretch{1.f, 0.f};
#pragma unroll
    for (int i = 0; i < L; ++i) {
      if (i < n) {
        float x[V], g[V];
        words.read(stage, 0, row, i, x);
        words.read(stage, 1, row, i, g);
#pragma unroll
        for (int v = 0; v < V; ++v) {
          gate_of(g[v] + bias[v], A[i][v], B[i][v]);
          B[i][v] *= x[v];
        }
        if (first >> i & 1) {  // the row takes the initial state, whatever comes before it
          const float* const h0 = a.state0 ? a.state0 + sequence_of(a, row + i).index * a.channels + c : nullptr;
#pragma unroll
          for (int v = 0; v < V; ++v) {
            B[i][v] = h0 ? fmaf(A[i][v], h0[v], B[i][v]) : B[i][v];
            mine[v] = Stretch{-1.f, B[i][v]};
          }
        } else {
#pragma unroll
          for (int v = 0; v < V; ++v) mine[v] = Stretch{mine[v].A < 0.f ? -1.f : mine[v].A * A[i][v], fmaf(A[i][v], mine[v].H, B[i][v])};
        }
      } else {
#pragma unroll
        for (int v = 0; v < V; ++v) A[i][v] = 1.f, B[i][v] = 0.f;
      }
    }
    float h[V];
    exchange(shared, stage, warp, rank, blocks, mine, carry, h);
    if (a.checkpoints && n > 0 && on && (row - begin) % kCheckpoint == 0) {
      float* const to = a.checkpoints + (blockIdx.y * a.checkpoints_per_segment + (row - begin) / kCheckpoint) * a.channels + c;
#pragma unroll
      for (int v = 0; v < V; ++v) to[v] = h[v];
    }
    T* y = static_cast<T*>(a.y) + row * a.y_stride + c;
#pragma unroll
    for (int i = 0; i < L; ++i) {
      if (i >= n) continue;
      const bool start = first >> i & 1;
#pragma unroll
      for (int v = 0; v < V; ++v) h[v] = start ? B[i][v] : fmaf(A[i][v], h[v], B[i][v]);
      float out[V];
      if (kGate) {
        float z[V];
        words.read(stage, kStreams - 1, row, i, z);
#pragma unroll
        for (int v = 0; v < V; ++v) out[v] = h[v] * (z[v] * sigmoid(z[v]));
      } else {
#pragma unroll
        for (int v = 0; v < V; ++v) out[v] = h[v];
      }
      if (on) store_word<T, V>(y + i * a.y_stride, out);
      if ((last >> i & 1) && a.state && on) {
        float* const to = a.state + sequence_of(a, row + i).index * a.channels + c;
#pragma unroll
        for (int v = 0; v < V; ++v) to[v] = h[v];
      }
    }
    words.fetch(stage, row_of(round + 2), rows_at(row_of(round + 2)), on);
  }
}

template <typename T, int V, bool kGate>
__global__ void __launch_bounds__(kThreads, 2) recurrence_backward_kernel(const RecArgs a) {
  constexpr int L = kBackwardRows, kTile = kWarps * L, kStreams = kGate ? 4 : 3;
  extern __shared__ __align__(16) char staged[];
  __shared__ Exchange<V> shared;
  __shared__ Stretch states[2][kWarps][32][V];
  grid_dependency_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int blocks = a.cluster, rank = blockIdx.x % blocks;
  const int channel = (blockIdx.x / blocks * 32 + lane) * V;
  const bool on = channel < a.channels;
  const int c = on ? channel : 0;
  long long begin, end;
  segment_rows(a, begin, end);
  if (rank == 0) pass_empty<V>(a, a.dstate, a.dstate0, c, on);
  const long long tiles = (end - begin + kTile - 1) / kTile, rounds = (tiles + blocks - 1) / blocks;
  Words<T, V, L, kStreams> words;
  words.base = staged + 4 * threadIdx.x;
  words.at[0] = static_cast<const T*>(a.x) + c, words.stride[0] = a.x_stride;
  words.at[1] = static_cast<const T*>(a.g) + c, words.stride[1] = a.g_stride;
  words.at[2] = static_cast<const T*>(a.dy) + c, words.stride[2] = a.dy_stride;
  if (kGate) words.at[kStreams - 1] = static_cast<const T*>(a.z) + c, words.stride[kStreams - 1] = a.z_stride;
  float bias[V], carry[V], dbias[V];
#pragma unroll
  for (int v = 0; v < V; ++v) bias[v] = a.bias ? a.bias[c + v] : 0.f, carry[v] = dbias[v] = 0.f;
  // the last rows come first
  const auto tile_of = [&](long long round) { return tiles - 1 - (round * blocks + rank); };
  const auto row_of = [&](long long round) { return begin + (tile_of(round) * kWarps + warp) * L; };
  const auto rows_at = [&](long long round) { return tile_of(round) < 0 ? 0 : (int)max(0ll, min((long long)L, end - row_of(round))); };
  for (int k = 0; k < 2; ++k) words.fetch(k, row_of(k), rows_at(k), on);
  for (long long round = 0; round < rounds; ++round) {
    const int stage = (int)(round & 1);
    const long long row = row_of(round), tile = tile_of(round);
    const int n = rows_at(round);
    float entered[V];  // the state before the tile
#pragma unroll
    for (int v = 0; v < V; ++v)
      entered[v] = tile < 0 ? 0.f : a.checkpoints[(blockIdx.y * a.checkpoints_per_segment + tile) * a.channels + c + v];
    words.wait();
    uint32_t first, last;
    borders(a, row, n, first, last);
    // the states of the warp's rows: its stretch, those of the warps before it, and from row to row
    float A[L][V], B[L][V], P[L][V], E[L][V];  // gates, states before each row, what enters each row from its output
    Stretch mine[V];
#pragma unroll
    for (int v = 0; v < V; ++v) mine[v] = Stretch{1.f, 0.f};
#pragma unroll
    for (int i = 0; i < L; ++i) {
      if (i < n) {
        float x[V], g[V];
        words.read(stage, 0, row, i, x);
        words.read(stage, 1, row, i, g);
#pragma unroll
        for (int v = 0; v < V; ++v) gate_of(g[v] + bias[v], A[i][v], B[i][v]);
        if (first >> i & 1) {
          const float* const h0 = a.state0 ? a.state0 + sequence_of(a, row + i).index * a.channels + c : nullptr;
#pragma unroll
          for (int v = 0; v < V; ++v) {
            P[i][v] = h0 ? h0[v] : 0.f;
            mine[v] = Stretch{-1.f, fmaf(A[i][v], P[i][v], B[i][v] * x[v])};
          }
        } else {
#pragma unroll
          for (int v = 0; v < V; ++v)
            mine[v] = Stretch{mine[v].A < 0.f ? -1.f : mine[v].A * A[i][v], fmaf(A[i][v], mine[v].H, B[i][v] * x[v])};
        }
      } else {
#pragma unroll
        for (int v = 0; v < V; ++v) A[i][v] = 1.f, B[i][v] = 0.f;
      }
    }
#pragma unroll
    for (int v = 0; v < V; ++v) states[stage][warp][lane][v] = mine[v];
    __syncthreads();
    float h[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      h[v] = entered[v];
      for (int w = 0; w < warp; ++w) h[v] = apply(states[stage][w][lane][v], h[v]);
    }
    T* dz = static_cast<T*>(a.dz) + row * a.dz_stride + c;
#pragma unroll
    for (int i = 0; i < L; ++i) {
#pragma unroll
      for (int v = 0; v < V; ++v) E[i][v] = 0.f;
      if (i >= n) continue;
      float x[V], dy[V];
      words.read(stage, 0, row, i, x);
      words.read(stage, 2, row, i, dy);
      const bool start = first >> i & 1;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        P[i][v] = start ? P[i][v] : h[v];
        h[v] = fmaf(A[i][v], P[i][v], B[i][v] * x[v]);
        E[i][v] = dy[v];
      }
      if (kGate) {
        float z[V];
        words.read(stage, kStreams - 1, row, i, z);
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const float s = sigmoid(z[v]);
          E[i][v] = dy[v] * (z[v] * s);
          z[v] = dy[v] * h[v] * (s * fmaf(z[v], 1.f - s, 1.f));
        }
        if (a.dz && on) store_word<T, V>(dz + i * a.dz_stride, z);
      }
      if ((last >> i & 1) && a.dstate) {
        const float* const from = a.dstate + sequence_of(a, row + i).index * a.channels + c;
#pragma unroll
        for (int v = 0; v < V; ++v) E[i][v] += from[v];
      }
    }
    // what flows to the rows before: d -> A (E + d), nothing across the beginning of a sequence
#pragma unroll
    for (int v = 0; v < V; ++v) mine[v] = Stretch{1.f, 0.f};
#pragma unroll
    for (int i = L - 1; i >= 0; --i) {
      if (i >= n) continue;
      const bool start = first >> i & 1;
#pragma unroll
      for (int v = 0; v < V; ++v)
        mine[v] = start ? Stretch{-1.f, 0.f}
                        : Stretch{mine[v].A < 0.f ? -1.f : mine[v].A * A[i][v], A[i][v] * (E[i][v] + mine[v].H)};
    }
    float d[V];
    exchange(shared, stage, kWarps - 1 - warp, rank, blocks, mine, carry, d);
    T* dx = static_cast<T*>(a.dx) + row * a.dx_stride + c;
    T* dg = static_cast<T*>(a.dg) + row * a.dg_stride + c;
#pragma unroll
    for (int i = L - 1; i >= 0; --i) {
      if (i >= n) continue;
      float x[V], out[V];
      words.read(stage, 0, row, i, x);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        d[v] += E[i][v];
        out[v] = B[i][v] * d[v];
        x[v] = out[v] * A[i][v] * (P[i][v] - x[v]);
        dbias[v] += x[v];
        d[v] *= A[i][v];
      }
      if (a.dx && on) store_word<T, V>(dx + i * a.dx_stride, out);
      if (a.dg && on) store_word<T, V>(dg + i * a.dg_stride, x);
      if (first >> i & 1) {
        if (a.dstate0 && on) {
          float* const to = a.dstate0 + sequence_of(a, row + i).index * a.channels + c;
#pragma unroll
          for (int v = 0; v < V; ++v) to[v] = d[v];
        }
#pragma unroll
        for (int v = 0; v < V; ++v) d[v] = 0.f;
      }
    }
    words.fetch(stage, row_of(round + 2), rows_at(round + 2), on);
  }
  if (!a.sums) return;
  __syncthreads();
#pragma unroll
  for (int v = 0; v < V; ++v) states[0][warp][lane][v].H = dbias[v];
  __syncthreads();
  if (warp == 0 && on) {
    float* const to = a.sums + ((long long)blockIdx.y * blocks + rank) * a.channels + c;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      float s = 0.f;
      for (int w = 0; w < kWarps; ++w) s += states[0][w][lane][v].H;
      to[v] = s;
    }
  }
}

// dbias (=|+=) scale * the parts' sums, in their order.
__global__ void __launch_bounds__(128)
recurrence_sum_kernel(const float* sums, float* dbias, int parts, int channels, float scale, int accumulate) {
  grid_dependency_wait();
  const int c = blockIdx.x * 128 + threadIdx.x;
  if (c >= channels) return;
  float s = 0.f;
  for (int p = 0; p < parts; ++p) s += sums[(long long)p * channels + c];
  s *= scale;
  dbias[c] = accumulate ? dbias[c] + s : s;
}

// One token of every sequence, the states in place.
template <typename T, int V, bool kGate>
__global__ void __launch_bounds__(128) recurrence_step_kernel(const RecArgs a) {
  grid_dependency_wait();
  const int c = (blockIdx.x * 128 + threadIdx.x) * V;
  if (c >= a.channels) return;
  for (long long s = blockIdx.y; s < a.sequences; s += gridDim.y) {
    float x[V], g[V], z[V], out[V];
    unpack<T, V>(load_word<T, V>(static_cast<const T*>(a.x) + s * a.x_stride + c), x);
    unpack<T, V>(load_word<T, V>(static_cast<const T*>(a.g) + s * a.g_stride + c), g);
    if (kGate) unpack<T, V>(load_word<T, V>(static_cast<const T*>(a.z) + s * a.z_stride + c), z);
    float* const state = a.state + s * a.channels + c;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      float fa, fb;
      gate_of(g[v] + (a.bias ? a.bias[c + v] : 0.f), fa, fb);
      const float h = fmaf(fa, state[v], fb * x[v]);
      state[v] = h;
      out[v] = kGate ? h * (z[v] * sigmoid(z[v])) : h;
    }
    store_word<T, V>(static_cast<T*>(a.y) + s * a.y_stride + c, out);
  }
}

// ---- host -------------------------------------------------------------------------------------------
struct Division {
  int tiles, segments, cluster;  // of channels; of sequences; blocks that share a segment's rows
  long long per_segment, checkpoints;
};

// Blocks for the whole GPU, two to an SM: over channels, then over sequences of known borders, then over time.
Division split_of(const fbfftconv_recurrence_desc& d, int V) {
  Division s{};
  s.tiles = (d.channels + 32 * V - 1) / (32 * V);
  const long long want = 2ll * sm_count();
  long long segments = d.offsets ? 1 : want / s.tiles;
  if (segments > d.sequences) segments = d.sequences;
  if (segments < 1) segments = 1;
  s.per_segment = d.sequences > 0 ? (d.sequences + segments - 1) / segments : 1;
  s.segments = (int)(d.sequences > 0 ? (d.sequences + s.per_segment - 1) / s.per_segment : 1);
  const long long rows = d.offsets ? d.rows : s.per_segment * d.length;
  s.checkpoints = (rows + kCheckpoint - 1) / kCheckpoint;
  s.cluster = 1;
  while (s.cluster < kMostCluster && (long long)s.tiles * s.segments * s.cluster * 2 <= want &&
         (long long)s.cluster * 2 * kCheckpoint <= rows)
    s.cluster *= 2;
  return s;
}

template <typename K>
cudaError_t launch_split(K kernel, const RecArgs& a, const Division& s, size_t smem, cudaStream_t stream) {
  const cudaError_t e = ensure_dynamic_smem(reinterpret_cast<const void*>(kernel), (int)smem);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(s.tiles * s.cluster, s.segments);
  config.blockDim = dim3(kThreads);
  config.dynamicSmemBytes = smem;
  config.stream = stream;
  cudaLaunchAttribute attrs[2]{};
  attrs[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attrs[0].val.programmaticStreamSerializationAllowed = 1;
  attrs[1].id = cudaLaunchAttributeClusterDimension;
  attrs[1].val.clusterDim.x = s.cluster, attrs[1].val.clusterDim.y = attrs[1].val.clusterDim.z = 1;
  config.attrs = attrs;
  config.numAttrs = s.cluster > 1 ? 2 : 1;
  const cudaError_t r = cudaLaunchKernelEx(&config, kernel, a);
  if (r != cudaSuccess) cudaGetLastError();
  return r;
}

template <typename T, int V>
cudaError_t forward(const RecArgs& a, const Division& s, cudaStream_t stream) {
  const size_t row = sizeof(T) * V == 4 ? 2ull * kForwardRows * kThreads * 4 : 0;
  return a.z ? launch_split(recurrence_forward_kernel<T, V, true>, a, s, 3 * row, stream)
             : launch_split(recurrence_forward_kernel<T, V, false>, a, s, 2 * row, stream);
}

template <typename T, int V>
cudaError_t backward(const RecArgs& a, const Division& s, cudaStream_t stream) {
  const size_t row = sizeof(T) * V == 4 ? 2ull * kBackwardRows * kThreads * 4 : 0;
  return a.z ? launch_split(recurrence_backward_kernel<T, V, true>, a, s, 4 * row, stream)
             : launch_split(recurrence_backward_kernel<T, V, false>, a, s, 3 * row, stream);
}

template <typename T, int V>
cudaError_t step(const RecArgs& a, cudaStream_t stream) {
  const dim3 grid((a.channels + 128 * V - 1) / (128 * V), (unsigned)(a.sequences < 65535 ? a.sequences : 65535));
  return a.z ? launch_dependent(recurrence_step_kernel<T, V, true>, grid, 128, 0, stream, a)
             : launch_dependent(recurrence_step_kernel<T, V, false>, grid, 128, 0, stream, a);
}

#define BY_TYPE(call)                                                                            \
  (d.type == FBFFTCONV_FLOAT32 ? call(float, 1)                                                  \
   : d.type == FBFFTCONV_BFLOAT16 ? (pairs ? call(__nv_bfloat16, 2) : call(__nv_bfloat16, 1))    \
                                  : (pairs ? call(__half, 2) : call(__half, 1)))

int check_desc(const fbfftconv_recurrence_desc* d) {
  if (!d) return op_fail(FBFFTCONV_ERR_INVALID_ARGUMENT, "null argument");
  if (d->channels <= 0 || d->channels > (1 << 22)) return op_fail(FBFFTCONV_ERR_INVALID_ARGUMENT, "1 to 2^22 channels");
  if (d->sequences < 0 || d->length < 0 || d->rows < 0) return op_fail(FBFFTCONV_ERR_INVALID_ARGUMENT, "negative size");
  if (d->sequences > (1ll << 31) || d->length > (1ll << 40) || d->rows > (1ll << 40))
    return op_fail(FBFFTCONV_ERR_UNSUPPORTED_SIZE, "more than 2^31 sequences or 2^40 rows");
  if (!known_type(d->type)) return op_fail(FBFFTCONV_ERR_INVALID_ARGUMENT, "unknown element type");
  if (!d->offsets && ((d->length > 0 && d->sequences > d->rows / d->length) || d->rows != d->sequences * d->length))
    return op_fail(FBFFTCONV_ERR_INVALID_ARGUMENT, "rows are not sequences times length");
  if (d->offsets && !aligned_to(d->offsets, d->wide_offsets ? 8 : 4))
    return op_fail(FBFFTCONV_ERR_INVALID_ARGUMENT, "offsets are not aligned");
  return FBFFTCONV_OK;
}

struct RowPointer {
  const void* p;
  const char* name;
  bool needed;
  long long stride;
};

template <int N, int M>
int check_rec_pointers(const RowPointer (&rows)[N], const RowPointer (&floats)[M], const fbfftconv_recurrence_desc& d,
                       int device, bool* pairs) {
  *pairs = d.channels % 2 == 0;
  for (const RowPointer& q : rows) {
    if (!q.p && q.needed) return op_fail(FBFFTCONV_ERR_INVALID_ARGUMENT, "%s is null", q.name);
    if (!aligned_to(q.p, type_bytes(d.type))) return op_fail(FBFFTCONV_ERR_INVALID_ARGUMENT, "%s is not aligned to its element", q.name);
    if (q.p && q.stride < d.channels) return op_fail(FBFFTCONV_ERR_INVALID_ARGUMENT, "the rows of %s overlap", q.name);
    if (q.p && (q.stride % 2 || !aligned_to(q.p, 2 * type_bytes(d.type)))) *pairs = false;
  }
  for (const RowPointer& q : floats) {
    if (!q.p && q.needed) return op_fail(FBFFTCONV_ERR_INVALID_ARGUMENT, "%s is null", q.name);
    if (!aligned_to(q.p, 4)) return op_fail(FBFFTCONV_ERR_INVALID_ARGUMENT, "%s is not aligned to its element", q.name);
  }
  for (const RowPointer& q : rows) OP_TRY(validate_device_pointer(device, q.p, q.name));
  for (const RowPointer& q : floats) OP_TRY(validate_device_pointer(device, q.p, q.name));
  return validate_device_pointer(device, d.offsets, "offsets");
}

RecArgs common_args(const fbfftconv_recurrence_desc& d) {
  const auto or_dense = [&](int64_t s) { return s ? (long long)s : (long long)d.channels; };
  RecArgs a{};
  a.rows = d.rows, a.length = d.length, a.sequences = d.sequences, a.channels = d.channels;
  a.offsets = d.offsets, a.wide_offsets = d.wide_offsets;
  a.x_stride = or_dense(d.x_stride), a.g_stride = or_dense(d.g_stride), a.z_stride = or_dense(d.z_stride);
  a.y_stride = or_dense(d.y_stride), a.dy_stride = or_dense(d.grad_y_stride);
  a.dx_stride = or_dense(d.grad_x_stride), a.dg_stride = or_dense(d.grad_g_stride), a.dz_stride = or_dense(d.grad_z_stride);
  return a;
}

// 16-bit channels travel in pairs or alone, which changes how many blocks share the channels; what is kept between the
// passes must not depend on that.
Division split_for(const fbfftconv_recurrence_desc& d, bool pairs) {
  const int V = d.type == FBFFTCONV_FLOAT32 ? 1 : 2;
  Division s = split_of(d, V);
  if (V == 2 && !pairs) s.tiles = (d.channels + 31) / 32;
  return s;
}

}  // namespace
}  // namespace fbfft

using namespace fbfft;

extern "C" {

size_t fbfftconv_recurrence_checkpoint_bytes(const fbfftconv_recurrence_desc* desc) {
  if (check_desc(desc) != FBFFTCONV_OK) return 0;
  int device;
  if (resolve_device(desc->device, &device) != FBFFTCONV_OK) return 0;
  const OnDevice on(device);
  const Division s = split_for(*desc, true);
  return (size_t)(s.segments * s.checkpoints) * desc->channels * sizeof(float);
}

size_t fbfftconv_recurrence_workspace_bytes(const fbfftconv_recurrence_desc* desc) {
  if (check_desc(desc) != FBFFTCONV_OK) return 0;
  int device;
  if (resolve_device(desc->device, &device) != FBFFTCONV_OK) return 0;
  const OnDevice on(device);
  const Division s = split_for(*desc, true);
  return (size_t)s.segments * s.cluster * desc->channels * sizeof(float);
}

int fbfftconv_recurrence(const fbfftconv_recurrence_desc* desc, const void* x, const void* g, const void* z,
                         const float* bias, const float* state0, void* y, float* state, float* checkpoints,
                         fbfftconv_stream stream) {
  OP_TRY(check_desc(desc));
  const fbfftconv_recurrence_desc& d = *desc;
  RecArgs a = common_args(d);
  const bool some = d.rows > 0;
  const RowPointer rows[] = {{x, "x", some, a.x_stride}, {g, "g", some, a.g_stride}, {z, "z", false, a.z_stride}, {y, "y", some, a.y_stride}};
  const RowPointer floats[] = {{bias, "bias", false, 0}, {state0, "the initial state", false, 0}, {state, "the final state", false, 0},
                               {checkpoints, "checkpoints", false, 0}};
  int device;
  bool pairs;
  if (state0 && state0 == state && d.sequences > 0)
    return op_fail(FBFFTCONV_ERR_INVALID_ARGUMENT, "the final state must not overwrite the initial one");
  OP_TRY(resolve_device(d.device, &device));
  OP_TRY(check_rec_pointers(rows, floats, d, device, &pairs));
  if (d.sequences == 0) return FBFFTCONV_OK;
  const OnDevice on(device);
  if (on.error() != cudaSuccess) return op_cuda_fail(on.error(), "cudaSetDevice");
  const Division s = split_for(d, pairs);
  a.x = x, a.g = g, a.z = z, a.bias = bias, a.state0 = state0, a.y = y, a.state = state, a.checkpoints = checkpoints;
  a.per_segment = s.per_segment, a.checkpoints_per_segment = s.checkpoints, a.cluster = s.cluster;
  count_launch();
#define FORWARD(T, V) forward<T, V>(a, s, static_cast<cudaStream_t>(stream))
  const cudaError_t e = BY_TYPE(FORWARD);
#undef FORWARD
  return e == cudaSuccess ? FBFFTCONV_OK : op_cuda_fail(e, "recurrence");
}

int fbfftconv_recurrence_backward(const fbfftconv_recurrence_desc* desc, const void* x, const void* g, const void* z,
                                  const float* bias, const float* state0, const float* checkpoints, const void* grad_y,
                                  const float* grad_state, void* grad_x, void* grad_g, void* grad_z, float* grad_state0,
                                  float* grad_bias, float scale, int accumulate, void* workspace, size_t workspace_bytes,
                                  fbfftconv_stream stream) {
  OP_TRY(check_desc(desc));
  const fbfftconv_recurrence_desc& d = *desc;
  if (!isfinite(scale)) return op_fail(FBFFTCONV_ERR_INVALID_ARGUMENT, "the scale must be finite");
  if (grad_z && !z) return op_fail(FBFFTCONV_ERR_INVALID_ARGUMENT, "a gradient by z without z");
  RecArgs a = common_args(d);
  const bool some = d.rows > 0;
  const RowPointer rows[] = {{x, "x", some, a.x_stride}, {g, "g", some, a.g_stride}, {z, "z", false, a.z_stride},
                             {grad_y, "gradOutput", some, a.dy_stride}, {grad_x, "gradInput of x", false, a.dx_stride},
                             {grad_g, "gradInput of g", false, a.dg_stride}, {grad_z, "gradInput of z", false, a.dz_stride}};
  const RowPointer floats[] = {{bias, "bias", false, 0}, {state0, "the initial state", false, 0}, {checkpoints, "checkpoints", some, 0},
                               {grad_state, "the final state's gradient", false, 0}, {grad_state0, "the initial state's gradient", false, 0},
                               {grad_bias, "gradBias", false, 0}, {workspace, "the workspace", grad_bias != nullptr && d.sequences > 0, 0}};
  int device;
  bool pairs;
  if (grad_state && grad_state == grad_state0 && d.sequences > 0)
    return op_fail(FBFFTCONV_ERR_INVALID_ARGUMENT, "the states' gradients must not share memory");
  OP_TRY(resolve_device(d.device, &device));
  OP_TRY(check_rec_pointers(rows, floats, d, device, &pairs));
  const OnDevice on(device);
  if (on.error() != cudaSuccess) return op_cuda_fail(on.error(), "cudaSetDevice");
  const Division s = split_for(d, pairs);
  const int parts = d.sequences > 0 ? s.segments * s.cluster : 0;
  if (grad_bias && workspace_bytes < (size_t)parts * d.channels * sizeof(float))
    return op_fail(FBFFTCONV_ERR_INVALID_ARGUMENT, "the workspace is smaller than fbfftconv_recurrence_workspace_bytes");
  const cudaStream_t cuda_stream = static_cast<cudaStream_t>(stream);
  if (d.sequences > 0) {
    a.x = x, a.g = g, a.z = z, a.bias = bias, a.state0 = state0, a.checkpoints = const_cast<float*>(checkpoints);
    a.dy = grad_y, a.dstate = grad_state, a.dx = grad_x, a.dg = grad_g, a.dz = grad_z, a.dstate0 = grad_state0;
    a.sums = grad_bias ? static_cast<float*>(workspace) : nullptr;
    a.per_segment = s.per_segment, a.checkpoints_per_segment = s.checkpoints, a.cluster = s.cluster;
    count_launch();
#define BACKWARD(T, V) backward<T, V>(a, s, cuda_stream)
    const cudaError_t e = BY_TYPE(BACKWARD);
#undef BACKWARD
    if (e != cudaSuccess) return op_cuda_fail(e, "recurrence, backward");
  }
  if (!grad_bias) return FBFFTCONV_OK;
  count_launch();
  const cudaError_t e = launch_dependent(recurrence_sum_kernel, dim3((d.channels + 127) / 128), 128, 0, cuda_stream,
                                         static_cast<const float*>(workspace), grad_bias, parts, d.channels, scale, accumulate);
  return e == cudaSuccess ? FBFFTCONV_OK : op_cuda_fail(e, "recurrence, sums");
}

int fbfftconv_recurrence_step(const fbfftconv_recurrence_desc* desc, const void* x, const void* g, const void* z,
                              const float* bias, float* state, void* y, fbfftconv_stream stream) {
  OP_TRY(check_desc(desc));
  const fbfftconv_recurrence_desc& d = *desc;
  if (d.offsets || (d.sequences > 0 && d.length != 1))
    return op_fail(FBFFTCONV_ERR_INVALID_ARGUMENT, "a step takes one row of every sequence");
  RecArgs a = common_args(d);
  const bool some = d.sequences > 0;
  const RowPointer rows[] = {{x, "x", some, a.x_stride}, {g, "g", some, a.g_stride}, {z, "z", false, a.z_stride}, {y, "y", some, a.y_stride}};
  const RowPointer floats[] = {{bias, "bias", false, 0}, {state, "the state", some, 0}};
  int device;
  bool pairs;
  OP_TRY(resolve_device(d.device, &device));
  OP_TRY(check_rec_pointers(rows, floats, d, device, &pairs));
  if (!some) return FBFFTCONV_OK;
  const OnDevice on(device);
  if (on.error() != cudaSuccess) return op_cuda_fail(on.error(), "cudaSetDevice");
  a.x = x, a.g = g, a.z = z, a.bias = bias, a.y = y, a.state = state;
  count_launch();
#define STEP(T, V) step<T, V>(a, static_cast<cudaStream_t>(stream))
  const cudaError_t e = BY_TYPE(STEP);
#undef STEP
  return e == cudaSuccess ? FBFFTCONV_OK : op_cuda_fail(e, "recurrence step");
}

}  // extern "C"
