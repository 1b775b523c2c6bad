// The norms before and after a residual block, fused with the block's gate and the residual's scale (sm_100a).
//
//   n = post(u),  r' = alpha r + beta act(g) n,  v = pre(r')          rms(x) = x / sqrt(mean x^2 + eps) w + b
//                                                                     layer(x) = rms(x - mean x)
// and backward, with hat the normalised rows and s their reciprocal deviation:
//   D = dr' + s2 (dv w2 - hat2 mean(dv w2 hat2) [- mean(dv w2)]),  dr = alpha D,  dn = beta act D
//   du = s1 (dn w1 - hat1 mean(dn w1 hat1) [- mean(dn w1)]),  dact = beta D n
//   dw2 = sum dv hat2, db2 = sum dv, dw1 = sum dn hat1, db1 = sum dn;  dg summed over the rows that share a gate row
//
// A row is held in the registers of one warp or one block between its sums, so each tensor moves once; 16384 x 4096 bf16
// with a gate per token takes 413 us both ways where its bytes would take 266, bound by the latency of a row's sums and
// by issue (38 and 92 instructions an element).  Sums over a row go by shuffles and one exchange through shared memory; a
// layer norm's deviation is taken about the mean, in a sum of its own.  Sums over rows stay in registers while a block
// walks its rows, and a second kernel adds the blocks' sums in a fixed order: the same call gives the same bits.
#include <math.h>

#include <type_traits>

#include "operators.cuh"

namespace fbfft {
namespace {

constexpr int kMostChannels = 16384;
constexpr long long kMostRows = 1ll << 30, kMostStride = 1ll << 30;  // rows and strides are 32 bits wide in the kernels

struct NormArgs {
  const void* u;
  const void* r;
  const void* gate;
  const float* w1;
  const float* b1;
  const float* w2;
  const float* b2;
  void* r_out;
  void* v;
  float4* stats;      // mean and reciprocal deviation of u, and of r'
  // backward
  const void* dr_out;
  const void* dv;
  void* du;
  void* dr;
  void* dgate;
  float* sums;        // a worker's sums: [kind][worker][channel]
  float* gate_sums;   // [worker][channel], or null: a worker has whole gate rows to itself
  int rows, u_stride, r_stride, gate_stride, per_gate;  // per_gate: rows that share a gate row
  int channels, lanes, post, pre, gate_kind;
  int splits;         // workers to a gate row, where rows share it
  int stages;         // rows under way in the ring
  bool vectors;
  float eps, alpha, beta;
};

template <typename E> __device__ __forceinline__ E* row_of(const void* p, int row, int stride) {
  return static_cast<E*>(const_cast<void*>(p)) + (long long)row * stride;
}

// A thread's columns of a row: chunks of neighbours one vector wide, or single ones a row's lanes apart where a
// pointer, a stride or the width does not allow vectors.
template <int C, int kVec, bool kRing>
struct Columns {
  int lane, lanes, channels;
  bool vectors;
  uint32_t valid;  // bit i: column i is one of the row's
  __device__ __forceinline__ Columns(int lane, int lanes, int channels, bool vectors)
      : lane(lane), lanes(lanes), channels(channels), vectors(vectors), valid(0) {
#pragma unroll
    for (int i = 0; i < C; ++i) valid |= (at(i) < channels ? 1u : 0u) << i;
  }
  __device__ __forceinline__ bool has(int i) const { return valid >> i & 1u; }
  __device__ __forceinline__ int at(int i) const {
    return kRing || vectors ? ((i / kVec) * lanes + lane) * kVec + i % kVec : i * lanes + lane;
  }
};

template <typename T, int kVec>
__device__ __forceinline__ void load_vector(const T* p, float* x) {
  if constexpr (std::is_same_v<T, float>) {
#pragma unroll
    for (int i = 0; i < kVec; i += 4) {
      const float4 q = __ldg(reinterpret_cast<const float4*>(p + i));
      x[i] = q.x, x[i + 1] = q.y, x[i + 2] = q.z, x[i + 3] = q.w;
    }
  } else {
    static_assert(kVec == 8);
    const uint4 q = __ldg(reinterpret_cast<const uint4*>(p));
    const uint32_t u[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = unpack2<T>(u[i]);
      x[2 * i] = f.x, x[2 * i + 1] = f.y;
    }
  }
}

template <typename T, int kVec>
__device__ __forceinline__ void store_vector(T* p, const float* x) {
  if constexpr (std::is_same_v<T, float>) {
#pragma unroll
    for (int i = 0; i < kVec; i += 4)
      *reinterpret_cast<float4*>(p + i) = make_float4(x[i], x[i + 1], x[i + 2], x[i + 3]);
  } else {
    static_assert(kVec == 8);
    *reinterpret_cast<uint4*>(p) = make_uint4(pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]), pack2<T>(x[4], x[5]), pack2<T>(x[6], x[7]));
  }
}

// x = the row's columns as fp32.  Where there is none: zero; in the ring's kernels, whose threads have whole vectors or
// none, any other of the row's, which keeps the loads free of branches (sum_of leaves it out).
template <typename T, int C, int kVec, bool kRing>
__device__ __forceinline__ void load_row(const T* row, const Columns<C, kVec, kRing>& c, float (&x)[C]) {
  if constexpr (kRing) {
#pragma unroll
    for (int i = 0; i < C; i += kVec) load_vector<T, kVec>(row + (c.has(i) ? c.at(i) : 0), x + i);
  } else {
#pragma unroll
    for (int i = 0; i < C; ++i) x[i] = 0.f;
    if (c.vectors) {
#pragma unroll
      for (int i = 0; i < C; i += kVec)
        if (c.has(i)) load_vector<T, kVec>(row + c.at(i), x + i);
    } else {
#pragma unroll
      for (int i = 0; i < C; ++i)
        if (c.has(i)) x[i] = to_float(row[c.at(i)]);
    }
  }
}

template <typename T, int C, int kVec, bool kRing>
__device__ __forceinline__ void store_row(T* row, const Columns<C, kVec, kRing>& c, const float (&x)[C]) {
  if (kRing || c.vectors) {
#pragma unroll
    for (int i = 0; i < C; i += kVec)
      if (c.has(i)) store_vector<T, kVec>(row + c.at(i), x + i);
  } else {
#pragma unroll
    for (int i = 0; i < C; ++i)
      if (c.has(i)) row[c.at(i)] = from_float<T>(x[i]);
  }
}

// A thread's own columns of the next rows, on their way from memory to shared memory: cp.async by the thread that will
// read them, so that no other thread has to be waited for, and no register holds what is in flight.  A stream is one of
// the row's tensors; its 16-byte pieces of a block's threads lie side by side, free of bank conflicts.
template <int C, int kVec, bool kRing>
struct Ring {
  char* base;  // of this thread, stage 0
  int pitch;   // bytes of a stage
  int step;    // bytes between a thread's pieces: 16 for every thread of the block
  int stages;  // rows under way, 1 or 2

  template <typename E>
  __device__ __forceinline__ void fetch(int stage, int piece, const E* row, const Columns<C, kVec, kRing>& c) const {
    constexpr int kPer = 16 / (int)sizeof(E);  // elements of a piece
#pragma unroll
    for (int i = 0; i < C; i += kPer)
      if (c.has(i))
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(
                         base + stage * pitch + (piece + i / kPer) * step)), "l"(row + c.at(i)) : "memory");
  }
  __device__ __forceinline__ void commit() const { asm volatile("cp.async.commit_group;" ::: "memory"); }
  // until the oldest of the rows that are under way has arrived
  __device__ __forceinline__ void wait() const {
    if (stages == 1) asm volatile("cp.async.wait_group 0;" ::: "memory");
    else asm volatile("cp.async.wait_group 1;" ::: "memory");
  }

  template <typename E>
  __device__ __forceinline__ void read(int stage, int piece, const Columns<C, kVec, kRing>& c, float (&x)[C]) const {
    constexpr int kPer = 16 / (int)sizeof(E);
#pragma unroll
    for (int i = 0; i < C; i += kPer) {
      const uint4 q = *reinterpret_cast<const uint4*>(base + stage * pitch + (piece + i / kPer) * step);
      if constexpr (std::is_same_v<E, float>) {
        x[i] = __uint_as_float(q.x), x[i + 1] = __uint_as_float(q.y), x[i + 2] = __uint_as_float(q.z), x[i + 3] = __uint_as_float(q.w);
      } else {
        const uint32_t u[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float2 f = unpack2<E>(u[k]);
          x[i + 2 * k] = f.x, x[i + 2 * k + 1] = f.y;
        }
      }
    }
  }
};

// Without the ring: a row's lines on their way to the L1 cache while the row before it is computed.
template <typename T, int C, int kVec, bool kRing>
__device__ __forceinline__ void prefetch_row(const T* row, const Columns<C, kVec, kRing>& c) {
  constexpr int kLine = 128 / (int)sizeof(T);
  for (int i = c.lane * kLine; i < c.channels; i += c.lanes * kLine) asm volatile("prefetch.global.L1 [%0];" ::"l"(row + i));
}

// The sum of a thread's columns of a row: what lies in vectors that are not the row's stays out, whatever it holds.
template <int C, int kVec, bool kRing, typename F>
__device__ __forceinline__ float sum_of(const Columns<C, kVec, kRing>& c, F term) {
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < C; i += kVec) {
    float t = 0.f;
#pragma unroll
    for (int k = i; k < i + kVec; ++k) t = term(k, t);
    s += !kRing || c.has(i) ? t : 0.f;
  }
  return s;
}

// Sums over the lanes of a row, for everyone: shuffles within a warp, then every thread adds the warps' sums in their
// order.  Two exchanges in turn use the two halves of `part`: a warp that is through with one cannot reach the next but
// one before all have left the first.  What lies behind the last warp's sums must be zero.
template <int kThreads>
struct RowSums {
  float (*part)[2][32];
  int lanes, turn;
  template <int N>
  __device__ __forceinline__ void operator()(float (&x)[N]) {
#pragma unroll
    for (int k = 0; k < N; ++k)
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) x[k] += __shfl_xor_sync(0xffffffffu, x[k], o);
    if (lanes <= 32) return;
    float(*const mine)[32] = part[turn];
    turn ^= 1;
    if ((threadIdx.x & 31) == 0) {
#pragma unroll
      for (int k = 0; k < N; ++k) mine[k][threadIdx.x >> 5] = x[k];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < N; ++k) {
      float s = 0.f;
#pragma unroll
      for (int w = 0; w < (kThreads + 31) / 32; w += 4) {
        if (w >= 8 && w >= lanes / 32) break;
        const float4 q = *reinterpret_cast<const float4*>(&mine[k][w]);
        s += (q.x + q.y) + (q.z + q.w);
      }
      x[k] = s;
    }
  }
};

__device__ __forceinline__ void clear_sums(float (*part)[2][32]) {
  if (threadIdx.x < 128) (&part[0][0][0])[threadIdx.x] = 0.f;
  for (int i = threadIdx.x + blockDim.x; i < 128; i += blockDim.x) (&part[0][0][0])[i] = 0.f;
  __syncthreads();
}

// x becomes x - mean; returns (mean, 1 / deviation).
template <int C, int kVec, bool kRing, typename S>
__device__ __forceinline__ float2 normalise(float (&x)[C], int kind, const Columns<C, kVec, kRing>& c, S& sums, float eps) {
  const float per = 1.f / (float)c.channels;
  float mean = 0.f;
  if (kind == FBFFTCONV_NORM_LAYER) {
    float one[1] = {sum_of(c, [&](int i, float t) { return t + x[i]; })};
    sums(one);
    mean = one[0] * per;
#pragma unroll
    for (int i = 0; i < C; ++i) x[i] = kRing || c.has(i) ? x[i] - mean : 0.f;
  }
  float one[1] = {sum_of(c, [&](int i, float t) { return fmaf(x[i], x[i], t); })};
  sums(one);
  return make_float2(mean, rsqrtf(fmaf(one[0], per, eps)));
}

__device__ __forceinline__ float sigmoid(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + __expf(-x)));
  return r;
}

// y = act(y), in one loop for each kind of gate
template <int C> __device__ __forceinline__ void activate(float (&y)[C], int kind) {
  if (kind != FBFFTCONV_GATE_SIGMOID) return;
#pragma unroll
  for (int i = 0; i < C; ++i) y[i] = sigmoid(y[i]);
}

template <typename T, int C> constexpr int pieces_of() { return C * (int)sizeof(T) / 16; }

template <typename T, typename TR, int C, int kThreads, bool kRing>
__global__ void __launch_bounds__(kThreads, kThreads <= 256 ? 4 : kThreads <= 320 ? 2 : 1) norm_forward_kernel(const NormArgs a) {
  constexpr int kVec = std::is_same_v<T, float> ? 4 : 8;
  constexpr int kT = pieces_of<T, C>(), kTR = pieces_of<TR, C>();
  __shared__ __align__(16) float part[2][2][32];
  extern __shared__ __align__(16) char staged[];
  clear_sums(part);
  grid_dependency_wait();
  const int slot = threadIdx.x / a.lanes, slots = blockDim.x / a.lanes;
  const Columns<C, kVec, kRing> c((int)threadIdx.x % a.lanes, a.lanes, a.channels, a.vectors);
  RowSums<kThreads> sums{part, a.lanes, 0};
  const int stride = gridDim.x * slots;
  const Ring<C, kVec, kRing> ring{staged + 16 * threadIdx.x, (2 * kT + kTR) * 16 * (int)blockDim.x, 16 * (int)blockDim.x, a.stages};
  const auto gate_row_of = [&](int row) { return a.per_gate == 1 ? row : row / a.per_gate; };
  const auto fetch = [&](int row, int stage) {
    if (row < a.rows) {
      const int gate_row = gate_row_of(row);
      ring.fetch(stage, 0, row_of<const TR>(a.r, row, a.r_stride), c);
      if (a.u) ring.fetch(stage, kTR, row_of<const T>(a.u, row, a.u_stride), c);
      if (a.gate_kind) ring.fetch(stage, kTR + kT, row_of<const T>(a.gate, gate_row, a.gate_stride), c);
    }
    ring.commit();
  };
  int row = blockIdx.x * slots + slot;
  if (kRing)
    for (int k = 0; k < a.stages; ++k) fetch(row + k * stride, k);
  for (int stage = 0; row < a.rows; row += stride, stage = stage + 1 < a.stages ? stage + 1 : 0) {
    float x[C], r[C], w[C], b[C];
    if (kRing) {
      ring.wait();
      if (a.u) ring.template read<T>(stage, kTR, c, x);
      ring.template read<TR>(stage, 0, c, r);
    } else {
      if (a.u) load_row(row_of<const T>(a.u, row, a.u_stride), c, x);
      load_row(row_of<const TR>(a.r, row, a.r_stride), c, r);
      if (row + stride < a.rows) {
        if (a.u) prefetch_row(row_of<const T>(a.u, row + stride, a.u_stride), c);
        prefetch_row(row_of<const TR>(a.r, row + stride, a.r_stride), c);
        if (a.u && a.gate_kind) prefetch_row(row_of<const T>(a.gate, gate_row_of(row + stride), a.gate_stride), c);
      }
    }
    float2 first = make_float2(0.f, 1.f), second = first;
    if (a.u) {
      float g[C];
      if (a.gate_kind) {
        if (kRing) ring.template read<T>(stage, kTR + kT, c, g);
        else load_row(row_of<const T>(a.gate, gate_row_of(row), a.gate_stride), c, g);
      }
      if (kRing) fetch(row + a.stages * stride, stage);
      if (a.post) {
        load_row(a.w1, c, w);  // on its way during the sums
        first = normalise(x, a.post, c, sums, a.eps);
#pragma unroll
        for (int i = 0; i < C; ++i) x[i] *= first.y * w[i];
        if (a.b1) {
          load_row(a.b1, c, b);
#pragma unroll
          for (int i = 0; i < C; ++i) x[i] += b[i];
        }
      }
      if (a.gate_kind) {
        activate(g, a.gate_kind);
#pragma unroll
        for (int i = 0; i < C; ++i) x[i] *= g[i];
      }
#pragma unroll
      for (int i = 0; i < C; ++i) r[i] = fmaf(a.beta, x[i], a.alpha * r[i]);
      if (a.pre) load_row(a.w2, c, w);
      store_row(row_of<TR>(a.r_out, row, a.channels), c, r);
    } else {
      if (kRing) fetch(row + a.stages * stride, stage);
      load_row(a.w2, c, w);
    }
    if (a.pre) {
      second = normalise(r, a.pre, c, sums, a.eps);
#pragma unroll
      for (int i = 0; i < C; ++i) r[i] *= second.y * w[i];
      if (a.b2) {
        load_row(a.b2, c, b);
#pragma unroll
        for (int i = 0; i < C; ++i) r[i] += b[i];
      }
      store_row(row_of<T>(a.v, row, a.channels), c, r);
    }
    if (a.stats && c.lane == 0) a.stats[row] = make_float4(first.x, first.y, second.x, second.y);
  }
}

// A worker is the lanes of one row: a block, or a warp of a block where rows are short.  r' is formed again from u, r
// and the gate: the one that was stored is rounded, and the weights' gradients would carry that.
template <typename T, typename TR, int C, int kThreads, bool kAll, bool kRing>
__global__ void __launch_bounds__(kThreads) norm_backward_kernel(const NormArgs a) {
  constexpr int kVec = std::is_same_v<T, float> ? 4 : 8;
  constexpr int kT = pieces_of<T, C>(), kTR = pieces_of<TR, C>();
  __shared__ __align__(16) float part[2][2][32];
  extern __shared__ __align__(16) char staged[];
  clear_sums(part);
  grid_dependency_wait();
  const int slots = blockDim.x / a.lanes;
  const int worker = blockIdx.x * slots + threadIdx.x / a.lanes, workers = gridDim.x * slots;
  const Columns<C, kVec, kRing> c((int)threadIdx.x % a.lanes, a.lanes, a.channels, a.vectors);
  RowSums<kThreads> sums{part, a.lanes, 0};
  const float per = 1.f / (float)a.channels;
  const bool shared_gate = kAll && a.gate_kind && a.per_gate > 1;
  // without shared gate rows all rows are one stretch, dealt out in turn; else `splits` workers deal out a gate row's
  const int stretch = shared_gate ? a.per_gate : a.rows, stretches = a.rows / stretch;
  const int splits = shared_gate ? a.splits : workers;
  const Ring<C, kVec, kRing> ring{staged + 16 * threadIdx.x, (3 * kT + 2 * kTR) * 16 * (int)blockDim.x, 16 * (int)blockDim.x, a.stages};
  enum { kR = 0, kDr = kTR, kU = 2 * kTR, kGate = kU + kT, kDv = kGate + kT };  // pieces of a stage
  const bool need_u = a.u && (a.post || a.gate_kind || a.pre);
  const auto fetch = [&](int row, int end, int gate_row, int stage) {
    if (row < end) {
      if (a.pre) ring.fetch(stage, kR, row_of<const TR>(a.r, row, a.r_stride), c);
      if (a.dr_out) ring.fetch(stage, kDr, row_of<const TR>(a.dr_out, row, a.channels), c);
      if (need_u) ring.fetch(stage, kU, row_of<const T>(a.u, row, a.u_stride), c);
      if (a.gate_kind) ring.fetch(stage, kGate, row_of<const T>(a.gate, gate_row, a.gate_stride), c);
      if (a.pre) ring.fetch(stage, kDv, row_of<const T>(a.dv, row, a.channels), c);
    }
    ring.commit();
  };
  float sw1[C], sw2[C], sb1[kAll ? C : 1], sb2[kAll ? C : 1], sg[kAll ? C : 1];
#pragma unroll
  for (int i = 0; i < C; ++i) {
    sw1[i] = sw2[i] = 0.f;
    if (kAll) sb1[i] = sb2[i] = sg[i] = 0.f;
  }
  // means over a row, the second of a layer norm alone
  const auto mean_of = [&](float (&p)[2], int kind) {
    if (kind == FBFFTCONV_NORM_LAYER) {
      sums(p);
      p[1] *= per;
    } else {
      float one[1] = {p[0]};
      sums(one);
      p[0] = one[0], p[1] = 0.f;
    }
    p[0] *= per;
  };
  int stage = 0;
  for (int s = worker / splits; s < stretches; s += workers / splits) {
    const int end = (s + 1) * stretch;
    int row = s * stretch + worker % splits;
    if (kRing)
      for (int k = 0; k < a.stages; ++k) fetch(row + k * splits, end, shared_gate ? s : row + k * splits, stage + k < a.stages ? stage + k : 0);
    float4 next_stat = row < end ? a.stats[row] : make_float4(0.f, 0.f, 0.f, 0.f);
    for (; row < end; row += splits, stage = stage + 1 < a.stages ? stage + 1 : 0) {
      const float4 stat = next_stat;
      if (row + splits < end) {
        next_stat = a.stats[row + splits];  // a row ahead: nothing of a row can begin without it
        if (!kRing) {
          const int next = row + splits;
          if (need_u) prefetch_row(row_of<const T>(a.u, next, a.u_stride), c);
          if (a.gate_kind && !shared_gate) prefetch_row(row_of<const T>(a.gate, next, a.gate_stride), c);
          if (a.dr_out) prefetch_row(row_of<const TR>(a.dr_out, next, a.channels), c);
          if (a.pre) {
            prefetch_row(row_of<const TR>(a.r, next, a.r_stride), c);
            prefetch_row(row_of<const T>(a.dv, next, a.channels), c);
          }
        }
      }
      if (kRing) ring.wait();
      float x[C], d[C], w[C], act[C];  // x: the block's output, normalised
      if (need_u) {
        if (kRing) ring.template read<T>(stage, kU, c, x);
        else load_row(row_of<const T>(a.u, row, a.u_stride), c, x);
      }
      if (a.gate_kind) {
        if (kRing) ring.template read<T>(stage, kGate, c, act);
        else load_row(row_of<const T>(a.gate, shared_gate ? s : row, a.gate_stride), c, act);
        activate(act, a.gate_kind);
      }
      if (a.post) {
#pragma unroll
        for (int i = 0; i < C; ++i) x[i] = (x[i] - stat.x) * stat.y;
      }
      // n: the branch before its gate, which is what the gate's gradient takes; needs w1 in n
      const auto branch = [&](float (&n)[C]) {
        if (a.post) {
          if (a.b1) {
            float b[C];
            load_row(a.b1, c, b);
#pragma unroll
            for (int i = 0; i < C; ++i) n[i] = fmaf(n[i], x[i], b[i]);
          } else {
#pragma unroll
            for (int i = 0; i < C; ++i) n[i] *= x[i];
          }
        } else {
#pragma unroll
          for (int i = 0; i < C; ++i) n[i] = x[i];
        }
      };
      if (a.dr_out) {
        if (kRing) ring.template read<TR>(stage, kDr, c, d);
        else load_row(row_of<const TR>(a.dr_out, row, a.channels), c, d);
      } else {
#pragma unroll
        for (int i = 0; i < C; ++i) d[i] = 0.f;
      }
      if (a.pre) {
        float r[C], y[C];
        if (kRing) ring.template read<TR>(stage, kR, c, r);
        else load_row(row_of<const TR>(a.r, row, a.r_stride), c, r);
        if (a.u) {
          if (a.post) load_row(a.w1, c, w);
          branch(w);
          if (a.gate_kind) {
#pragma unroll
            for (int i = 0; i < C; ++i) w[i] *= act[i];
          }
#pragma unroll
          for (int i = 0; i < C; ++i) r[i] = fmaf(a.beta, w[i], a.alpha * r[i]);
        }
        load_row(a.w2, c, w);
        if (kRing) ring.template read<T>(stage, kDv, c, y);
        else load_row(row_of<const T>(a.dv, row, a.channels), c, y);
#pragma unroll
        for (int i = 0; i < C; ++i) {
          r[i] = (r[i] - stat.z) * stat.w;
          sw2[i] = fmaf(y[i], r[i], sw2[i]);
          if (kAll) sb2[i] += y[i];
          y[i] *= w[i];
        }
        float p[2] = {sum_of(c, [&](int i, float t) { return fmaf(y[i], r[i], t); }), 0.f};
        if (a.pre == FBFFTCONV_NORM_LAYER) p[1] = sum_of(c, [&](int i, float t) { return t + y[i]; });
        if (kRing) fetch(row + a.stages * splits, end, shared_gate ? s : row + a.stages * splits, stage);
        if (a.post) load_row(a.w1, c, w);  // on its way during the sums
        mean_of(p, a.pre);
#pragma unroll
        for (int i = 0; i < C; ++i) d[i] = fmaf(stat.w, y[i] - fmaf(r[i], p[0], p[1]), d[i]);
      } else {
        if (kRing) fetch(row + a.stages * splits, end, shared_gate ? s : row + a.stages * splits, stage);
        load_row(a.w1, c, w);
      }
      {
        float out[C];
#pragma unroll
        for (int i = 0; i < C; ++i) out[i] = a.alpha * d[i];
        store_row(row_of<TR>(a.dr, row, a.channels), c, out);
      }
      if (!a.u) continue;
#pragma unroll
      for (int i = 0; i < C; ++i) d[i] *= a.beta;
      if (a.gate_kind) {
        float n[C];
#pragma unroll
        for (int i = 0; i < C; ++i) n[i] = w[i];
        branch(n);
#pragma unroll
        for (int i = 0; i < C; ++i) n[i] *= d[i];
        if (a.gate_kind == FBFFTCONV_GATE_SIGMOID) {
#pragma unroll
          for (int i = 0; i < C; ++i) n[i] *= fmaf(-act[i], act[i], act[i]);
        }
#pragma unroll
        for (int i = 0; i < C; ++i) {
          d[i] *= act[i];
          if (kAll) sg[i] += n[i];
        }
        if (!shared_gate) store_row(row_of<T>(a.dgate, row, a.channels), c, n);
      }
      if (a.post) {
#pragma unroll
        for (int i = 0; i < C; ++i) {
          sw1[i] = fmaf(d[i], x[i], sw1[i]);
          if (kAll) sb1[i] += d[i];
          d[i] *= w[i];
        }
        float p[2] = {sum_of(c, [&](int i, float t) { return fmaf(d[i], x[i], t); }), 0.f};
        if (a.post == FBFFTCONV_NORM_LAYER) p[1] = sum_of(c, [&](int i, float t) { return t + d[i]; });
        mean_of(p, a.post);
#pragma unroll
        for (int i = 0; i < C; ++i) d[i] = stat.y * (d[i] - fmaf(x[i], p[0], p[1]));
      }
      store_row(row_of<T>(a.du, row, a.channels), c, d);
    }
    if constexpr (kAll) {
      if (shared_gate) {
        if (a.gate_sums) store_row(a.gate_sums + (long long)worker * a.channels, c, sg);
        else store_row(row_of<T>(a.dgate, s, a.channels), c, sg);
#pragma unroll
        for (int i = 0; i < C; ++i) sg[i] = 0.f;
      }
    }
  }
  const long long one = (long long)workers * a.channels;
  float* at = a.sums + (long long)worker * a.channels;
  if (a.post) store_row(at, c, sw1);
  if (a.pre) store_row(at + one, c, sw2);
  if constexpr (kAll) {
    if (a.post) store_row(at + 2 * one, c, sb1);
    if (a.pre) store_row(at + 3 * one, c, sb2);
  }
}

// out[column] = (accumulate: +) scale * sum of the workers' sums, a fixed order: eight strands of rows, then the strands.
struct SumJob {
  const float* src;  // [count][channels]
  void* dst;
  int count, type;
  float scale;
  int accumulate;
};
struct SumArgs {
  SumJob job[5];
  int jobs, channels;
  long long gate_rows;  // of the last job, if it is the gate's: one sum for each
};

constexpr int kStrands = 32;
__global__ void __launch_bounds__(1024) norm_sum_kernel(const SumArgs a) {
  __shared__ float part[kStrands][33];
  grid_dependency_wait();
  const int lane = threadIdx.x & 31, strand = threadIdx.x >> 5;
  const int column = blockIdx.x * 32 + lane;
  const bool gate = blockIdx.y >= a.jobs;
  const SumJob& j = a.job[gate ? a.jobs : blockIdx.y];
  const long long group = gate ? blockIdx.y - a.jobs : 0;
  const float* src = j.src + group * j.count * a.channels;
  float s = 0.f;
  if (column < a.channels)
    for (int i = strand; i < j.count; i += kStrands) s += src[(long long)i * a.channels + column];
  part[strand][lane] = s;
  __syncthreads();
  if (strand != 0 || column >= a.channels) return;
  s = 0.f;
#pragma unroll
  for (int i = 0; i < kStrands; ++i) s += part[i][lane];
  s *= j.scale;
  const long long at = group * a.channels + column;
  if (j.type == FBFFTCONV_FLOAT32) {
    float* const d = static_cast<float*>(j.dst) + at;
    *d = j.accumulate ? *d + s : s;
  } else if (j.type == FBFFTCONV_BFLOAT16) {
    static_cast<__nv_bfloat16*>(j.dst)[at] = from_float<__nv_bfloat16>(s);
  } else {
    static_cast<__half*>(j.dst)[at] = from_float<__half>(s);
  }
}

// ---- host -------------------------------------------------------------------------------------------
struct Shape {
  int lanes, threads, columns;  // threads of a row, of a block; columns of a thread
  bool ring;
};

// Short rows share a block, a warp each; a longer row has a block to itself, whose lanes meet at its barriers.  Rows of
// whole vectors go through the ring (8192 x 7000 f16 with a gate: 150 and 351 us forward and backward; 7001, without the
// ring: 475 and 1112) where one row of every tensor fits shared memory.  Sixteen columns a thread are more than the
// registers hold with the sums over rows: eight in the backward pass (16384 x 4096 with a gate 285 us, sixteen 319), until
// a row is wider than 512 threads; from there on it spills.  Forward, eight keep more blocks on an SM until a row is wider
// than 256 threads (16384 x 2048 bf16 57 us, sixteen 59).
Shape shape_of(int channels, int columns, bool ring) {
  const int lanes = (channels + 32 * columns - 1) / (32 * columns) * 32;
  return {lanes, lanes == 32 ? 128 : lanes, columns, ring};
}
constexpr size_t kMostShared = 226 * 1024;  // of a block, less what the kernels hold besides

Shape forward_shape(int channels, int type_size, int residual_size, bool vectors) {
  if (vectors && (size_t)channels * (2 * type_size + residual_size) <= kMostShared - 16 * 1024)
    return shape_of(channels, channels > 2048 ? 16 : 8, true);
  return shape_of(channels, channels > 8192 ? 16 : 8, false);
}
Shape backward_shape(int channels, int type_size, int residual_size, bool vectors) {
  if (vectors && (size_t)channels * (3 * type_size + 2 * residual_size) <= kMostShared - 16 * 1024)
    return shape_of(channels, channels > 4096 ? 16 : 8, true);
  return shape_of(channels, channels > 4096 ? 16 : 8, false);
}

int check_desc(const fbfftconv_norm_desc* d) {
  if (!d) return op_fail(FBFFTCONV_ERR_INVALID_ARGUMENT, "null argument");
  if (d->rows < 0 || d->channels <= 0) return op_fail(FBFFTCONV_ERR_INVALID_ARGUMENT, "rows and channels must be positive");
  if (d->rows > kMostRows || d->u_stride > kMostStride || d->r_stride > kMostStride || d->gate_stride > kMostStride)
    return op_fail(FBFFTCONV_ERR_UNSUPPORTED_SIZE, "more than 2^30 rows, or elements between rows");
  if (d->u_stride < 0 || d->r_stride < 0 || d->gate_stride < 0) return op_fail(FBFFTCONV_ERR_INVALID_ARGUMENT, "negative stride");
  if (d->channels > kMostChannels) return op_fail(FBFFTCONV_ERR_UNSUPPORTED_SIZE, "more than %d channels", kMostChannels);
  if (!known_type(d->type) || !known_type(d->residual_type) ||
      (d->residual_type != d->type && d->residual_type != FBFFTCONV_FLOAT32))
    return op_fail(FBFFTCONV_ERR_INVALID_ARGUMENT, "the residual stream has the block's element type, or fp32");
  if (d->post < 0 || d->post > FBFFTCONV_NORM_LAYER || d->pre < 0 || d->pre > FBFFTCONV_NORM_LAYER)
    return op_fail(FBFFTCONV_ERR_INVALID_ARGUMENT, "unknown norm");
  if (!d->post && !d->pre) return op_fail(FBFFTCONV_ERR_INVALID_ARGUMENT, "neither norm is there");
  if (d->gate < 0 || d->gate > FBFFTCONV_GATE_SIGMOID) return op_fail(FBFFTCONV_ERR_INVALID_ARGUMENT, "unknown gate");
  if (d->gate && (d->gate_rows < 0 || (d->rows > 0 && (d->gate_rows == 0 || d->rows % d->gate_rows))))
    return op_fail(FBFFTCONV_ERR_INVALID_ARGUMENT, "the gate's rows must divide the rows");
  if (!(d->eps >= 0) || !isfinite(d->eps) || !isfinite(d->residual_scale) || !isfinite(d->branch_scale))
    return op_fail(FBFFTCONV_ERR_INVALID_ARGUMENT, "eps and the scales must be finite, eps not negative");
  return FBFFTCONV_OK;
}

NormArgs common_args(const fbfftconv_norm_desc& d) {
  NormArgs a{};
  a.rows = (int)d.rows, a.channels = d.channels;
  a.post = d.post, a.pre = d.pre, a.gate_kind = d.gate;
  a.u_stride = d.u_stride ? (int)d.u_stride : d.channels;
  a.r_stride = d.r_stride ? (int)d.r_stride : d.channels;
  a.gate_stride = d.gate_stride ? (int)d.gate_stride : d.channels;
  a.per_gate = d.gate && d.gate_rows ? (int)(d.rows / d.gate_rows) : 1;
  a.eps = d.eps, a.alpha = d.residual_scale, a.beta = d.branch_scale;
  return a;
}

struct Pointer {
  const void* p;
  const char* name;
  int type;
  bool needed;
  long long stride;  // of its rows, in elements
};

// Null where it is needed, misaligned, or of another device; clears `vectors` where 16-byte loads are not possible.
template <int N>
int check_pointers(const Pointer (&all)[N], int device, int channels, int type, bool* vectors) {
  for (const Pointer& q : all) {
    if (!q.p && q.needed) return op_fail(FBFFTCONV_ERR_INVALID_ARGUMENT, "%s is null", q.name);
    if (!aligned_to(q.p, type_bytes(q.type))) return op_fail(FBFFTCONV_ERR_INVALID_ARGUMENT, "%s is not aligned to its element", q.name);
    const int vector = type == FBFFTCONV_FLOAT32 ? 4 : 8;  // elements that travel together
    if (q.p && (!aligned_to(q.p, 16) || q.stride % vector)) *vectors = false;
  }
  if (channels % (type == FBFFTCONV_FLOAT32 ? 4 : 8)) *vectors = false;
  for (const Pointer& q : all) OP_TRY(validate_device_pointer(device, q.p, q.name));
  return FBFFTCONV_OK;
}

template <typename K>
cudaError_t launch_rows(K kernel, NormArgs a, const Shape& s, int grid, size_t stage_bytes, cudaStream_t stream) {
  a.stages = 2 * stage_bytes <= kMostShared ? 2 : 1;
  const size_t smem = a.stages * stage_bytes;
  if (smem > 40 * 1024) {  // 48 KB, less what the kernel holds besides, need no leave
    const cudaError_t e = ensure_dynamic_smem(reinterpret_cast<const void*>(kernel), (int)smem);
    if (e != cudaSuccess) return e;
  }
  return launch_dependent(kernel, dim3(grid), s.threads, smem, stream, a);
}

template <typename T, typename TR>
cudaError_t forward(const NormArgs& a, const Shape& s, cudaStream_t stream) {
  const long long slots = s.threads / s.lanes, need = (a.rows + slots - 1) / slots;
  // Blocks that walk several rows each: four an SM from 256 threads up, 1024 threads an SM below.  Those are one or more
  // full sets of what an SM holds; other numbers leave a set half empty (8192 x 5120 bf16 with an fp32 stream 112 us, five
  // an SM 130, seven 124), fewer threads leave loads too few (131072 x 256 bf16 50 us, half as many 62, 12312 x 1000 f32 42
  // and 57), and more are more starts (8192 x 8192 bf16 122 us, eight an SM 126, sixteen 137).
  const long long most = (long long)sm_count() * (s.threads >= 256 ? 4 : 1024 / s.threads);
  const int grid = (int)(need < most ? need : most);
  if (!s.ring)
    return s.columns == 8 ? launch_rows(norm_forward_kernel<T, TR, 8, 1024, false>, a, s, grid, 0, stream)
                          : launch_rows(norm_forward_kernel<T, TR, 16, 1024, false>, a, s, grid, 0, stream);
  const size_t stage = (size_t)s.threads * s.columns * (2 * sizeof(T) + sizeof(TR));
  if (s.columns == 8) return launch_rows(norm_forward_kernel<T, TR, 8, 256, true>, a, s, grid, stage, stream);
  // Above 256 threads an SM holds one block at the 118 registers of sixteen columns, but two of up to 320 threads at 96,
  // which 16-bit values do with (16384 rows with a gate: 4352 wide 150 us instead of 207, 5120 wide 162 instead of 215).
  // Up to 256 it holds two or more anyway, and 96 are only fewer (2560 wide 133 us instead of 108 with an fp32 stream,
  // 4096 wide with a gate 137 instead of 129); fp32 spills more at 96 (5120 wide 288 us instead of 249).
  if constexpr (sizeof(T) == 2)
    if (s.threads > 256 && s.threads <= 320) return launch_rows(norm_forward_kernel<T, TR, 16, 320, true>, a, s, grid, stage, stream);
  return s.threads <= 512 ? launch_rows(norm_forward_kernel<T, TR, 16, 512, true>, a, s, grid, stage, stream)
                          : launch_rows(norm_forward_kernel<T, TR, 16, 1024, true>, a, s, grid, stage, stream);
}

template <typename T, typename TR, bool kAll>
cudaError_t backward(const NormArgs& a, const Shape& s, int grid, cudaStream_t stream) {
  if (!s.ring)
    return s.columns == 8      ? launch_rows(norm_backward_kernel<T, TR, 8, 512, kAll, false>, a, s, grid, 0, stream)
           : s.threads <= 512 ? launch_rows(norm_backward_kernel<T, TR, 16, 512, kAll, false>, a, s, grid, 0, stream)
                              : launch_rows(norm_backward_kernel<T, TR, 16, 1024, kAll, false>, a, s, grid, 0, stream);
  const size_t stage = (size_t)s.threads * s.columns * (3 * sizeof(T) + 2 * sizeof(TR));
  return s.columns == 8      ? launch_rows(norm_backward_kernel<T, TR, 8, 512, kAll, true>, a, s, grid, stage, stream)
         : s.threads <= 512 ? launch_rows(norm_backward_kernel<T, TR, 16, 512, kAll, true>, a, s, grid, stage, stream)
                            : launch_rows(norm_backward_kernel<T, TR, 16, 1024, kAll, true>, a, s, grid, stage, stream);
}

template <typename T, typename TR>
cudaError_t backward(const NormArgs& a, const Shape& s, int grid, bool all, cudaStream_t stream) {
  return all ? backward<T, TR, true>(a, s, grid, stream) : backward<T, TR, false>(a, s, grid, stream);
}

#define BY_TYPES(call)                                                                                            \
  (d.type == FBFFTCONV_FLOAT32 ? call(float, float)                                                               \
   : d.type == FBFFTCONV_BFLOAT16                                                                                 \
       ? (d.residual_type == FBFFTCONV_FLOAT32 ? call(__nv_bfloat16, float) : call(__nv_bfloat16, __nv_bfloat16)) \
       : (d.residual_type == FBFFTCONV_FLOAT32 ? call(__half, float) : call(__half, __half)))

// Backward holds more sums where biases have gradients or rows share a gate's.
bool shared_gate(const fbfftconv_norm_desc& d) { return d.gate && d.gate_rows < d.rows; }

// How the backward pass deals its rows out: workers, and workers to a gate row that rows share.
struct Deal {
  int grid, slots, splits;
  bool shared;
};

Deal deal_of(const fbfftconv_norm_desc& d, const Shape& s) {
  Deal q{};
  q.slots = s.threads / s.lanes;
  // threads that an SM holds of these kernels, in blocks
  const int per_sm = s.threads >= 512 ? 1 : 512 / s.threads;
  const long long most = (long long)sm_count() * per_sm;
  q.shared = shared_gate(d);
  if (!q.shared) {
    const long long need = (d.rows + q.slots - 1) / q.slots;
    q.grid = (int)(need < most ? need : most);
    return q;
  }
  const long long workers = most * q.slots, per_gate = d.rows / d.gate_rows;
  long long splits = workers / d.gate_rows;
  if (splits > per_gate) splits = per_gate;
  if (splits < 1) splits = 1;
  // whole blocks of workers; a gate row's workers stay together
  long long total = splits > 1 ? splits * d.gate_rows : (d.gate_rows < workers ? d.gate_rows : workers);
  q.splits = (int)splits;
  q.grid = (int)((total + q.slots - 1) / q.slots);
  return q;
}

size_t sum_floats(const fbfftconv_norm_desc& d, const Deal& q) {
  const long long workers = (long long)q.grid * q.slots;
  return (size_t)workers * d.channels * (q.shared && q.splits > 1 ? 5 : 4);
}

}  // namespace
}  // namespace fbfft

using namespace fbfft;

extern "C" {

int fbfftconv_residual_norm(const fbfftconv_norm_desc* desc, const void* u, const void* r, const void* gate,
                            const float* post_weight, const float* post_bias, const float* pre_weight,
                            const float* pre_bias, void* r_out, void* v, float* stats, fbfftconv_stream stream) {
  OP_TRY(check_desc(desc));
  const fbfftconv_norm_desc& d = *desc;
  if (!u && d.rows > 0 && (d.post || d.gate)) return op_fail(FBFFTCONV_ERR_INVALID_ARGUMENT, "a post-norm or a gate without a block's output");
  int device;
  bool vectors = true;
  NormArgs a = common_args(d);
  OP_TRY(resolve_device(d.device, &device));
  const bool some = d.rows > 0;
  const Pointer all[] = {
      {u, "u", d.type, false, a.u_stride}, {r, "r", d.residual_type, some, a.r_stride},
      {d.gate ? gate : nullptr, "the gate", d.type, some && d.gate, a.gate_stride},
      {post_weight, "the post-norm's weight", FBFFTCONV_FLOAT32, some && d.post, 0},
      {post_bias, "the post-norm's bias", FBFFTCONV_FLOAT32, false, 0},
      {pre_weight, "the pre-norm's weight", FBFFTCONV_FLOAT32, some && d.pre, 0},
      {pre_bias, "the pre-norm's bias", FBFFTCONV_FLOAT32, false, 0},
      {u ? r_out : nullptr, "the residual's output", d.residual_type, some && u, d.channels},
      {d.pre ? v : nullptr, "the norm's output", d.type, some && d.pre, d.channels},
      {stats, "stats", FBFFTCONV_FLOAT32, false, 0}};
  if (!aligned_to(stats, 16)) return op_fail(FBFFTCONV_ERR_INVALID_ARGUMENT, "stats are not aligned to 16 bytes");
  OP_TRY(check_pointers(all, device, d.channels, d.type, &vectors));
  if (!some) return FBFFTCONV_OK;
  const OnDevice on(device);
  if (on.error() != cudaSuccess) return op_cuda_fail(on.error(), "cudaSetDevice");
  const Shape s = forward_shape(d.channels, type_bytes(d.type), type_bytes(d.residual_type), vectors);
  a.lanes = s.lanes;
  a.u = u, a.r = r, a.gate = gate, a.w1 = post_weight, a.b1 = post_bias, a.w2 = pre_weight, a.b2 = pre_bias;
  a.r_out = r_out, a.v = v, a.stats = reinterpret_cast<float4*>(stats), a.vectors = vectors;
  count_launch();
#define FORWARD(T, TR) forward<T, TR>(a, s, static_cast<cudaStream_t>(stream))
  const cudaError_t e = BY_TYPES(FORWARD);
#undef FORWARD
  return e == cudaSuccess ? FBFFTCONV_OK : op_cuda_fail(e, "residual norm");
}

size_t fbfftconv_residual_norm_workspace_bytes(const fbfftconv_norm_desc* desc) {
  if (check_desc(desc) != FBFFTCONV_OK || desc->rows == 0) return 0;
  int device;
  if (resolve_device(desc->device, &device) != FBFFTCONV_OK) return 0;
  const OnDevice on(device);
  size_t most = 0;  // of the shapes that the pointers' alignment may lead to
  for (int i = 0; i < 2; ++i) {
    const Shape s = backward_shape(desc->channels, type_bytes(desc->type), type_bytes(desc->residual_type), i);
    const size_t n = sum_floats(*desc, deal_of(*desc, s));
    most = n > most ? n : most;
  }
  return most * sizeof(float);
}

int fbfftconv_residual_norm_backward(const fbfftconv_norm_desc* desc, const void* u, const void* r, const void* gate,
                                     const float* stats, const float* post_weight, const float* post_bias,
                                     const float* pre_weight, const void* grad_r, const void* grad_v, void* grad_u,
                                     void* grad_r_in, void* grad_gate, float* grad_post_weight, float* grad_post_bias,
                                     float* grad_pre_weight, float* grad_pre_bias, float scale, int accumulate,
                                     void* workspace, size_t workspace_bytes, fbfftconv_stream stream) {
  OP_TRY(check_desc(desc));
  const fbfftconv_norm_desc& d = *desc;
  if (!u && d.rows > 0 && (d.post || d.gate)) return op_fail(FBFFTCONV_ERR_INVALID_ARGUMENT, "a post-norm or a gate without a block's output");
  if (!isfinite(scale)) return op_fail(FBFFTCONV_ERR_INVALID_ARGUMENT, "the scale must be finite");
  int device;
  bool vectors = true;
  NormArgs a = common_args(d);
  OP_TRY(resolve_device(d.device, &device));
  const bool some = d.rows > 0;
  const Pointer all[] = {
      {u, "u", d.type, false, a.u_stride}, {d.gate ? gate : nullptr, "the gate", d.type, some && d.gate, a.gate_stride},
      {d.pre ? r : nullptr, "r", d.residual_type, some && d.pre, a.r_stride},
      {stats, "stats", FBFFTCONV_FLOAT32, some, 0},
      {post_weight, "the post-norm's weight", FBFFTCONV_FLOAT32, some && d.post, 0},
      {post_bias, "the post-norm's bias", FBFFTCONV_FLOAT32, false, 0},
      {pre_weight, "the pre-norm's weight", FBFFTCONV_FLOAT32, some && d.pre, 0},
      {grad_r, "the residual's gradient", d.residual_type, some && u, d.channels},
      {d.pre ? grad_v : nullptr, "the norm's gradient", d.type, some && d.pre, d.channels},
      {u ? grad_u : nullptr, "gradInput of u", d.type, some && u, d.channels},
      {grad_r_in, "gradInput of r", d.residual_type, some, d.channels},
      {d.gate ? grad_gate : nullptr, "gradInput of the gate", d.type, some && d.gate, d.channels},
      {grad_post_weight, "gradPostWeight", FBFFTCONV_FLOAT32, false, 0}, {grad_post_bias, "gradPostBias", FBFFTCONV_FLOAT32, false, 0},
      {grad_pre_weight, "gradPreWeight", FBFFTCONV_FLOAT32, false, 0}, {grad_pre_bias, "gradPreBias", FBFFTCONV_FLOAT32, false, 0},
      {workspace, "the workspace", FBFFTCONV_FLOAT32, some, 0}};
  if (!aligned_to(stats, 16)) return op_fail(FBFFTCONV_ERR_INVALID_ARGUMENT, "stats are not aligned to 16 bytes");
  OP_TRY(check_pointers(all, device, d.channels, d.type, &vectors));
  const OnDevice on(device);
  if (on.error() != cudaSuccess) return op_cuda_fail(on.error(), "cudaSetDevice");
  const cudaStream_t cuda_stream = static_cast<cudaStream_t>(stream);
  SumArgs sum{};
  sum.channels = d.channels;
  float* const outs[4] = {d.post ? grad_post_weight : nullptr, d.pre ? grad_pre_weight : nullptr,
                          d.post ? grad_post_bias : nullptr, d.pre ? grad_pre_bias : nullptr};
  const bool every = shared_gate(d) || outs[2] || outs[3];
  const Shape s = backward_shape(d.channels, type_bytes(d.type), type_bytes(d.residual_type), vectors);
  Deal q{};
  if (some) {
    q = deal_of(d, s);
    if (workspace_bytes < sum_floats(d, q) * sizeof(float))
      return op_fail(FBFFTCONV_ERR_INVALID_ARGUMENT, "the workspace is smaller than fbfftconv_residual_norm_workspace_bytes");
  }
  const long long workers = (long long)q.grid * q.slots, one = workers * d.channels;
  float* const sums = static_cast<float*>(workspace);
  for (int i = 0; i < 4; ++i)
    if (outs[i]) sum.job[sum.jobs++] = SumJob{sums + i * one, outs[i], (int)workers, FBFFTCONV_FLOAT32, scale, accumulate};
  int groups = 0;
  if (some) {
    a.lanes = s.lanes, a.u = u, a.r = r, a.gate = gate, a.w1 = post_weight, a.b1 = post_bias, a.w2 = pre_weight;
    if (!u) a.alpha = 1.f;  // the forward pass takes r itself there
    a.stats = reinterpret_cast<float4*>(const_cast<float*>(stats));
    a.dr_out = grad_r, a.dv = grad_v, a.du = grad_u, a.dr = grad_r_in, a.dgate = grad_gate, a.vectors = vectors;
    a.sums = sums, a.splits = q.splits;
    if (q.shared && q.splits > 1) {
      a.gate_sums = sums + 4 * one;
      sum.job[sum.jobs] = SumJob{a.gate_sums, grad_gate, q.splits, d.type, 1.f, 0};
      groups = (int)d.gate_rows;  // no more than there are workers
    }
    count_launch();
#define BACKWARD(T, TR) backward<T, TR>(a, s, q.grid, every, cuda_stream)
    const cudaError_t e = BY_TYPES(BACKWARD);
#undef BACKWARD
    if (e != cudaSuccess) return op_cuda_fail(e, "residual norm, backward");
  }
  if (!some && d.gate && grad_gate && d.gate_rows > 0) {  // gate rows that no rows share
    const cudaError_t e = cudaMemsetAsync(grad_gate, 0, (size_t)d.gate_rows * d.channels * type_bytes(d.type), cuda_stream);
    if (e != cudaSuccess) return op_cuda_fail(e, "residual norm, backward");
  }
  if (sum.jobs + groups == 0) return FBFFTCONV_OK;
  count_launch();
  const cudaError_t e = launch_dependent(norm_sum_kernel, dim3((d.channels + 31) / 32, sum.jobs + groups), 1024, 0, cuda_stream, sum);
  return e == cudaSuccess ? FBFFTCONV_OK : op_cuda_fail(e, "residual norm, sums");
}

}  // extern "C"
