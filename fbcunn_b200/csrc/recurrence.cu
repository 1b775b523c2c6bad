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
// while this one is computed.  Bytes would allow 8 x 4096 x 2048 bf16 both ways in 226 us; it takes 418, bound by issue
// and latency: 40 to 46 instructions an element forward, 83 backward, with 128 registers and so 16 warps an SM.  1 - a is
// formed first where a is the larger, so that a + (1 - a) = 1 to the last place and long memories do not drift.
#include <cooperative_groups.h>
#include <math.h>
#include <string.h>

#include <atomic>
#include <mutex>
#include <type_traits>

#include "operators.cuh"

namespace cg = cooperative_groups;

namespace fbfft {
namespace {

constexpr int kWarps = 8, kThreads = 32 * kWarps;
constexpr int kForwardRows = 16, kBackwardRows = 8;  // of a warp, in a round
constexpr int kCheckpoint = 64;                      // rows between the states that forward leaves for backward
constexpr int kMostCluster = 16;
constexpr long long kMostRows = 1ll << 30;             // rows are 32 bits wide in the kernels
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
  int rows, length, sequences;
  int x_stride, g_stride, z_stride, y_stride, dy_stride, dx_stride, dg_stride, dz_stride;
  int per_segment;       // sequences of a segment
  int checkpoints_per_segment;
  int channels, wide_offsets, cluster;
  bool wide;             // rows begin on 16 bytes
  uint32_t polls;        // of a wait for a cluster's stretches, after the first
  uint32_t never;        // bytes that a wait is for and nobody sends: none, unless waits are to run out
  int* wait_error;       // set when one ran out: the device's word in host memory
};

// Offsets of up to this many sequences are kept in shared memory: a search is a chain of loads.
constexpr int kKeptOffsets = 512;

__device__ __forceinline__ int load_offset(const RecArgs& a, int i) {
  const long long v = a.wide_offsets ? static_cast<const long long*>(a.offsets)[i] : static_cast<const int*>(a.offsets)[i];
  return (int)(v < 0 ? 0 : v > a.rows ? a.rows : v);  // a bad offset must not lead out of the tensors
}

__device__ __forceinline__ int offset_at(const RecArgs& a, const int* kept, int i) {
  return a.sequences <= kKeptOffsets ? kept[i] : load_offset(a, i);
}
__device__ __forceinline__ void keep_offsets(const RecArgs& a, int* kept) {
  if (a.offsets && a.sequences <= kKeptOffsets)
    for (int i = threadIdx.x; i <= a.sequences; i += kThreads) kept[i] = load_offset(a, i);
  __syncthreads();
}

// The sequence that a row belongs to, and the rows where it begins and ends.
struct Sequence {
  int index, begin, end;
};
__device__ __forceinline__ Sequence sequence_of(const RecArgs& a, const int* kept, int row) {
  if (!a.offsets) {
    const int i = row / a.length;
    return {i, i * a.length, (i + 1) * a.length};
  }
  int lo = 0, hi = a.sequences;  // the last one that begins at or before the row
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (offset_at(a, kept, mid) <= row) lo = mid;
    else hi = mid;
  }
  return {lo, offset_at(a, kept, lo), offset_at(a, kept, lo + 1)};
}

// The sequence that a row belongs to, for the few rows that begin or end one: kept out of the loops' code.
__device__ __noinline__ int index_of(const RecArgs& a, const int* kept, int row) { return sequence_of(a, kept, row).index; }

// Which of a warp's rows begin a sequence, and which end one.  `in`, the sequence that its rows were in last, is looked
// up anew only where they have left it; most rounds lie within one sequence.
struct Borders {
  uint32_t first, last;
};
__device__ __forceinline__ Borders borders(const RecArgs& a, const int* kept, int row, int n, Sequence& in) {
  Borders b{0, 0};
  if (n <= 0) return b;
  if (row < in.begin || row >= in.end) in = sequence_of(a, kept, row);
  if (row > in.begin && in.end - row > n) return b;
  if (row == in.begin) b.first = 1;
  while (in.end > row && in.end - row <= n) {
    const int k = in.end - row;
    b.last |= 1u << (k - 1);
    if (k == n) break;
    b.first |= 1u << k;
    const Sequence next = sequence_of(a, kept, in.end);
    if (next.end <= in.end) break;  // offsets that do not rise
    in = next;
  }
  return b;
}

// A lane's channels: one value, or two whose sums and products are single instructions (the issue slots are what runs
// out first here).
template <int V> struct Vec;
template <> struct Vec<1> {
  float x;
  __device__ __forceinline__ float get(int) const { return x; }
  __device__ __forceinline__ void set(int, float v) { x = v; }
};
template <> struct Vec<2> {
  float x, y;
  __device__ __forceinline__ float get(int i) const { return i ? y : x; }
  __device__ __forceinline__ void set(int i, float v) { (i ? y : x) = v; }
  __device__ __forceinline__ unsigned long long bits() const {
    unsigned long long b;
    asm("mov.b64 %0, {%1, %2};" : "=l"(b) : "f"(x), "f"(y));
    return b;
  }
  static __device__ __forceinline__ Vec from(unsigned long long b) {
    Vec v;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(v.x), "=f"(v.y) : "l"(b));
    return v;
  }
};
template <int V> __device__ __forceinline__ Vec<V> all_of(float v) {
  Vec<V> r;
#pragma unroll
  for (int i = 0; i < V; ++i) r.set(i, v);
  return r;
}
__device__ __forceinline__ Vec<1> fma(Vec<1> a, Vec<1> b, Vec<1> c) { return {fmaf(a.x, b.x, c.x)}; }
__device__ __forceinline__ Vec<1> operator*(Vec<1> a, Vec<1> b) { return {a.x * b.x}; }
__device__ __forceinline__ Vec<1> operator+(Vec<1> a, Vec<1> b) { return {a.x + b.x}; }
__device__ __forceinline__ Vec<2> fma(Vec<2> a, Vec<2> b, Vec<2> c) {
  unsigned long long d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a.bits()), "l"(b.bits()), "l"(c.bits()));
  return Vec<2>::from(d);
}
__device__ __forceinline__ Vec<2> operator*(Vec<2> a, Vec<2> b) {
  unsigned long long d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a.bits()), "l"(b.bits()));
  return Vec<2>::from(d);
}
__device__ __forceinline__ Vec<2> operator+(Vec<2> a, Vec<2> b) {
  unsigned long long d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a.bits()), "l"(b.bits()));
  return Vec<2>::from(d);
}

// h -> A h + H; A < 0 stands for rows that begin a sequence among them: nothing of h comes through, not even a NaN.
template <int V> struct Stretch {
  Vec<V> A, H;
};
template <int V> __device__ __forceinline__ Vec<V> apply(const Stretch<V>& s, Vec<V> h) {
  Vec<V> r = fma(s.A, h, s.H);
#pragma unroll
  for (int v = 0; v < V; ++v)
    if (s.A.get(v) < 0.f) r.set(v, s.H.get(v));
  return r;
}
template <int V> __device__ __forceinline__ Stretch<V> join(const Stretch<V>& s, const Stretch<V>& next) {
  Stretch<V> r{s.A * next.A, apply(next, s.H)};
#pragma unroll
  for (int v = 0; v < V; ++v)
    if (s.A.get(v) < 0.f || next.A.get(v) < 0.f) r.A.set(v, -1.f);
  return r;
}
template <int V> __device__ __forceinline__ Stretch<V> nothing() { return {all_of<V>(1.f), all_of<V>(0.f)}; }

__device__ __forceinline__ float reciprocal(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float exp2_fast(float x) {  // results below the normal numbers are zero
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

constexpr float kLog2e = 1.4426950408889634f;

// a = sigmoid(g) and b = 1 - a, both to the last places: the larger is formed from the smaller.
template <int V> __device__ __forceinline__ void gate_of(Vec<V> g, Vec<V>& a, Vec<V>& b) {
  Vec<V> e, r;
#pragma unroll
  for (int v = 0; v < V; ++v) e.set(v, exp2_fast(-kLog2e * fabsf(g.get(v))));
  const Vec<V> d = e + all_of<V>(1.f);
#pragma unroll
  for (int v = 0; v < V; ++v) r.set(v, reciprocal(d.get(v)));
  const Vec<V> small = e * r, big = fma(small, all_of<V>(-1.f), all_of<V>(1.f));
#pragma unroll
  for (int v = 0; v < V; ++v) {
    a.set(v, g.get(v) < 0.f ? small.get(v) : big.get(v));
    b.set(v, g.get(v) < 0.f ? big.get(v) : small.get(v));
  }
}

template <int V> __device__ __forceinline__ Vec<V> sigmoid(Vec<V> x) {
  const Vec<V> t = x * all_of<V>(-kLog2e);
  Vec<V> e, r;
#pragma unroll
  for (int v = 0; v < V; ++v) e.set(v, exp2_fast(t.get(v)));
  e = e + all_of<V>(1.f);
#pragma unroll
  for (int v = 0; v < V; ++v) r.set(v, reciprocal(e.get(v)));
  return r;
}

// z sigmoid(z) by itself: with another factor the product of a mask's lowest z would be infinite before it meets its zero.
template <int V> __device__ __forceinline__ Vec<V> silu(Vec<V> z) { return z * sigmoid(z); }

template <int V> __device__ __forceinline__ Vec<V> load_floats(const float* p) {
  Vec<V> r;
#pragma unroll
  for (int v = 0; v < V; ++v) r.set(v, p[v]);
  return r;
}
template <int V> __device__ __forceinline__ void store_floats(float* p, Vec<V> x) {
#pragma unroll
  for (int v = 0; v < V; ++v) p[v] = x.get(v);
}

// A lane's channels of a row: one 32-bit word, or a single 16-bit value where pairs are not aligned.
template <typename T, int V> __device__ __forceinline__ Vec<V> unpack(uint32_t w) {
  if constexpr (std::is_same_v<T, float>) {
    return Vec<1>{__uint_as_float(w)};
  } else if constexpr (V == 2) {
    const float2 f = unpack2<T>(w);
    return Vec<2>{f.x, f.y};
  } else {
    return Vec<1>{unpack2<T>(w).x};
  }
}
template <typename T, int V> __device__ __forceinline__ uint32_t load_word(const T* p) {
  if constexpr (sizeof(T) * V == 4) return __ldg(reinterpret_cast<const uint32_t*>(p));
  else return __ldg(reinterpret_cast<const uint16_t*>(p));
}
template <typename T, int V> __device__ __forceinline__ void store_word(T* p, Vec<V> x) {
  if constexpr (std::is_same_v<T, float>) *p = x.x;
  else if constexpr (V == 2) *reinterpret_cast<uint32_t*>(p) = pack2<T>(x.x, x.y);
  else *p = from_float<T>(x.x);
}

// The words of a warp's next rows: in shared memory, on their way there while this round is computed.  A slot holds
// one tensor's rows, 128 bytes each; it is filled anew as soon as the round has read it, one group of copies after the
// scan and one after the outputs, so that the oldest group but one is always the one that is waited for.  Where rows
// begin on 16 bytes a lane copies such pieces of its warp's rows, past the L1 cache (`wide`; 8 x 4096 x 1024 bf16 takes 84
// and 153 us forward and backward, 1026 channels, whose rows begin on 4 bytes, 115 and 176); else each its own words.
// Single 16-bit values, which cp.async does not copy, are loaded where they are read (1025 channels: 127 and 261).
template <typename T, int V, int kRows>
struct Words {
  static constexpr bool kAsync = sizeof(T) * V == 4;
  static constexpr int kSlot = kRows * kThreads * 4;
  static constexpr int kPiece = 16 / sizeof(T);  // channels of a piece
  char* base;      // this warp's
  bool wide;
  int channel, channels;  // of the warp's first lane; of a row

  // `p`: the warp's channels of its first row
  __device__ __forceinline__ void fetch(int slot, const T* p, int stride, int n) const {
    if constexpr (kAsync) {
      const int lane = threadIdx.x & 31;
      const uint32_t to = (uint32_t)__cvta_generic_to_shared(base + slot * kSlot);
      if (wide) {
        const int first = lane >> 3, piece = lane & 7;
        const T* from = p + first * stride + piece * kPiece;
        const uint32_t at = to + first * 128 + piece * 16;
        const int rows = channel + piece * kPiece < channels ? n : 0;
#pragma unroll
        for (int i = 0; i < kRows; i += 4)
          if (first + i < rows)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(at + i * 128), "l"(from + i * stride) : "memory");
      } else {
        const T* from = p + lane * V;
        const int rows = channel + lane * V < channels ? n : 0;
#pragma unroll
        for (int i = 0; i < kRows; ++i)
          if (i < rows)
            asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(to + i * 128 + lane * 4), "l"(from + i * stride) : "memory");
      }
    } else {
      // to the L1 cache: a row's 32 values lie in one or two lines, and two lanes see to each row
      const int lane = threadIdx.x & 31, row = lane >> 1;
      if (row < kRows && row < n)
        asm volatile("prefetch.global.L1 [%0];" ::"l"(p + row * stride + (lane & 1 ? min(31, channels - 1 - channel) : 0)));
    }
  }
  __device__ __forceinline__ void commit() const {
    if constexpr (kAsync) asm volatile("cp.async.commit_group;" ::: "memory");
  }
  __device__ __forceinline__ void wait() const {
    if constexpr (kAsync) {
      asm volatile("cp.async.wait_group 1;" ::: "memory");
      __syncwarp();
    }
  }
  // before a slot is filled anew: every lane has read it
  __device__ __forceinline__ void release() const {
    if constexpr (kAsync) __syncwarp();
  }
  // row i of the slot, which is that of `p`
  __device__ __forceinline__ Vec<V> read(int slot, const T* p, int stride, int i) const {
    if constexpr (kAsync) return unpack<T, V>(*reinterpret_cast<const uint32_t*>(base + slot * kSlot + i * 128 + (threadIdx.x & 31) * 4));
    else return unpack<T, V>(load_word<T, V>(p + (channel + (threadIdx.x & 31) * V < channels ? (threadIdx.x & 31) * V : 0) + i * stride));
  }
};

// Joins what the warps and blocks before one have: a block's warps through `part`, a cluster's blocks through `whole`.
// "Before" is in the direction of the scan; `order` counts in it.  Each has a buffer for even and one for odd rounds: a
// warp that is through with a round may write the next one's while others still read, and what orders those reads is the
// barrier of the round after, which it passes before it writes the same buffer again.
constexpr int kTurns = 2;
template <int V>
struct Exchange {
  Stretch<V> part[kTurns][kWarps][32];
  Stretch<V> whole[kTurns][kMostCluster][32];
  uint64_t arrived[kTurns];  // mbarriers: the cluster's stretches of a round are there
  int gave_up;
};

constexpr uint32_t kPolls = 1u << 20;  // of a microsecond: about a second, where a round takes some microseconds

__device__ __forceinline__ uint32_t shared_address(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

// Polls of a microsecond: one, and up to `more` of them.  (A loop that asks before its first poll cost 8 of 418 us
// at 8 x 4096 x 2048 both ways, where there is no cluster at all.)
__device__ __forceinline__ bool wait_phase(uint32_t barrier, uint32_t parity, uint32_t more) {
  uint32_t done;
  do {
    asm volatile("{ .reg .pred p; mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3; selp.u32 %0, 1, 0, p; }"
                 : "=r"(done) : "r"(barrier), "r"(parity), "r"(1000u) : "memory");
  } while (!done && more-- != 0);
  return done;
}

template <int V>
__device__ __forceinline__ void start_exchange(Exchange<V>& x, int blocks) {
  if (blocks == 1) return;
  if (threadIdx.x == 0) {
    x.gave_up = 0;
    for (int h = 0; h < kTurns; ++h) asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(shared_address(&x.arrived[h])) : "memory");
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  cg::this_cluster().sync();
}

// Writes a stretch into another block's shared memory and counts its bytes there.
__device__ __forceinline__ void send(uint32_t to, uint32_t barrier, int block, const Stretch<2>& s) {
  asm volatile(
      "{ .reg .b32 a, b; mapa.shared::cluster.u32 a, %0, %2; mapa.shared::cluster.u32 b, %1, %2;\n"
      "st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v4.f32 [a], {%3, %4, %5, %6}, [b]; }"
      ::"r"(to), "r"(barrier), "r"(block), "f"(s.A.x), "f"(s.A.y), "f"(s.H.x), "f"(s.H.y) : "memory");
}
__device__ __forceinline__ void send(uint32_t to, uint32_t barrier, int block, const Stretch<1>& s) {
  asm volatile(
      "{ .reg .b32 a, b; mapa.shared::cluster.u32 a, %0, %2; mapa.shared::cluster.u32 b, %1, %2;\n"
      "st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v2.f32 [a], {%3, %4}, [b]; }"
      ::"r"(to), "r"(barrier), "r"(block), "f"(s.A.x), "f"(s.H.x) : "memory");
}

// `mine`: this warp's stretch; returns the value that enters it and moves `carry` behind the whole round.  A block's
// stretch goes to all blocks of the cluster with the bytes counted on their mbarriers: a cluster's barrier would have
// waited for the outputs that are on their way to memory too.  A block sends a round's stretch after all of its warps
// have read the round's before, so that nothing arrives in a buffer that is still read.  A block whose wait has run out
// goes on as one without a cluster: it neither sends, counts nor waits any more, and the others' waits run out in turn.
template <int V>
__device__ __forceinline__ Vec<V> exchange(Exchange<V>& x, uint32_t round, int order, int rank, int blocks,
                                           const RecArgs& a, const Stretch<V>& mine, Vec<V>& carry) {
  const int lane = threadIdx.x & 31, half = round % kTurns;
  Stretch<V>(*const part)[32] = x.part[half];
  part[order][lane] = mine;
  __syncthreads();
  Stretch<V> before = nothing<V>();
#pragma unroll 4
  for (int w = 0; w < order; ++w) before = join(before, part[w][lane]);
  Stretch<V> all = join(before, mine);
#pragma unroll 4
  for (int w = order + 1; w < kWarps; ++w) all = join(all, part[w][lane]);
  if (blocks == 1 || *reinterpret_cast<volatile int*>(&x.gave_up)) {
    const Vec<V> enter = apply(before, carry);
    carry = apply(all, carry);
    return enter;
  }
  const uint32_t barrier = shared_address(&x.arrived[half]);
  if (threadIdx.x == 0)
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(barrier), "r"((uint32_t)(blocks * 32 * sizeof(Stretch<V>)) + a.never) : "memory");
  for (int k = order; k < blocks; k += kWarps) send(shared_address(&x.whole[half][rank][lane]), barrier, k, all);
  if (!wait_phase(barrier, round / kTurns & 1, a.polls)) {
    *reinterpret_cast<volatile int*>(&x.gave_up) = 1;
    asm volatile("st.global.u32 [%0], %1;" ::"l"(a.wait_error), "r"(1));
  }
#pragma unroll 4
  for (int k = 0; k < rank; ++k) carry = apply(x.whole[half][k][lane], carry);
  const Vec<V> enter = apply(before, carry);
#pragma unroll 4
  for (int k = rank; k < blocks; ++k) carry = apply(x.whole[half][k][lane], carry);
  return enter;
}

// Ends a block's part: nothing may arrive in the memory of a block that has left.  One whose waits have all ended has what
// is sent to it; one whose wait ran out stays until no other block can send any more, and then for as long as what was
// sent may be under way.
template <int V>
__device__ __forceinline__ void finish_exchange(Exchange<V>& x, int blocks) {
  if (blocks == 1) return;
  cg::this_cluster().sync();  // every block comes here: all waits before it are bounded
  if (*reinterpret_cast<volatile int*>(&x.gave_up)) __nanosleep(1000000);
}

// Starts a wait that nothing ends, with a limit of a few polls: 1 when it gave up.
__global__ void wait_probe_kernel(int* gave_up) {
  __shared__ uint64_t barrier;
  asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(shared_address(&barrier)) : "memory");
  *gave_up = !wait_phase(shared_address(&barrier), 0, 4);
}

// The rows of this block's segment: [begin, end).
__device__ __forceinline__ void segment_rows(const RecArgs& a, const int* kept, int& begin, int& end) {
  if (a.offsets) {
    begin = offset_at(a, kept, 0);
    end = offset_at(a, kept, a.sequences);
  } else {
    const int first = blockIdx.y * a.per_segment;
    const int last = min(first + a.per_segment, a.sequences);
    begin = first * a.length, end = last * a.length;
  }
}

// Sequences without rows hand their state on.
template <int V>
__device__ __forceinline__ void pass_empty(const RecArgs& a, const int* kept, const float* from, float* to, int channel, bool on) {
  if (!to || blockIdx.y || (!a.offsets && a.length > 0)) return;
  for (int s = threadIdx.x >> 5; s < a.sequences; s += kWarps) {
    if (a.offsets && offset_at(a, kept, s + 1) > offset_at(a, kept, s)) continue;
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (on) to[(long long)s * a.channels + channel + v] = from ? from[(long long)s * a.channels + channel + v] : 0.f;
  }
}

template <typename T, int V, bool kGate>
__global__ void __launch_bounds__(kThreads, 2) recurrence_forward_kernel(const __grid_constant__ RecArgs a) {
  constexpr int L = kForwardRows, kTile = kWarps * L;
  extern __shared__ __align__(16) char staged[];
  __shared__ __align__(16) Exchange<V> shared;
  __shared__ int kept[kKeptOffsets + 1];
  grid_dependency_wait();
  keep_offsets(a, kept);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int blocks = a.cluster, rank = blockIdx.x % blocks;
  const int channel = (blockIdx.x / blocks * 32 + lane) * V;
  const bool on = channel < a.channels;
  const int c = on ? channel : 0;
  int begin, end;
  segment_rows(a, kept, begin, end);
  if (rank == 0) pass_empty<V>(a, kept, a.state0, a.state, c, on);
  const int tiles = (end - begin + kTile - 1) / kTile, rounds = (tiles + blocks - 1) / blocks;
  const int group = blockIdx.x / blocks * 32 * V;  // the first lane's channel
  const Words<T, V, L> words{staged + warp * (L * 128), a.wide, group, a.channels};
  enum { kX, kG, kZ };  // slots
  const T* const x0 = static_cast<const T*>(a.x) + group;
  const T* const g0 = static_cast<const T*>(a.g) + group;
  const T* const z0 = static_cast<const T*>(a.z) + group;
  const Vec<V> bias = a.bias ? load_floats<V>(a.bias + c) : all_of<V>(0.f);
  Vec<V> carry = all_of<V>(0.f);
  start_exchange(shared, blocks);
  const auto row_of = [&](int round) { return begin + ((round * blocks + rank) * kWarps + warp) * L; };
  const auto rows_at = [&](int row) { return max(0, min(L, end - row)); };
  const auto fetch_inputs = [&](int round) {
    words.release();
    const int row = row_of(round);
    const int n = rows_at(row);
    words.fetch(kX, x0 + (long long)row * a.x_stride, a.x_stride, n);
    words.fetch(kG, g0 + (long long)row * a.g_stride, a.g_stride, n);
    words.commit();
  };
  const auto fetch_outputs = [&](int round) {
    words.release();
    const int row = row_of(round);
    if (kGate) words.fetch(kZ, z0 + (long long)row * a.z_stride, a.z_stride, rows_at(row));
    words.commit();
  };
  fetch_inputs(0);
  fetch_outputs(0);
  Sequence in{0, 0, 0};
  for (int round = 0; round < rounds; ++round) {
    const int row = row_of(round);
    const int n = rows_at(row);
    const T* const xs = x0 + (long long)row * a.x_stride;
    const T* const gs = g0 + (long long)row * a.g_stride;
    const T* const zs = z0 + (long long)row * a.z_stride;
    words.wait();
    const Borders at = borders(a, kept, row, n, in);
    const bool within = n == L && at.first == 0 && at.last == 0;  // all rows there, none at a sequence's border
    Vec<V> A[L], B[L];
    Stretch<V> mine = nothing<V>();
    const auto scan = [&](auto plain) {
#pragma unroll
      for (int i = 0; i < L; ++i) {
        if (plain || i < n) {
          gate_of(words.read(kG, gs, a.g_stride, i) + bias, A[i], B[i]);
          B[i] = B[i] * words.read(kX, xs, a.x_stride, i);
          if (!plain && (at.first >> i & 1)) {  // the row takes the initial state, whatever comes before it
            if (a.state0) B[i] = fma(A[i], load_floats<V>(a.state0 + (long long)index_of(a, kept, row + i) * a.channels + c), B[i]);
            mine = Stretch<V>{all_of<V>(-1.f), B[i]};
          } else {
            const bool cut = !plain && mine.A.x < 0.f;
            mine = Stretch<V>{cut ? mine.A : mine.A * A[i], fma(A[i], mine.H, B[i])};
          }
        } else {
          A[i] = all_of<V>(1.f), B[i] = all_of<V>(0.f);
        }
      }
    };
    if (within) scan(std::true_type{});
    else scan(std::false_type{});
    fetch_inputs(round + 1);
    Vec<V> h = exchange(shared, (uint32_t)round, warp, rank, blocks, a, mine, carry);
    words.wait();
    if (a.checkpoints && n > 0 && on && (row - begin) % kCheckpoint == 0)
      store_floats(a.checkpoints + (long long)(blockIdx.y * a.checkpoints_per_segment + (row - begin) / kCheckpoint) * a.channels + c, h);
    T* y = static_cast<T*>(a.y) + (long long)row * a.y_stride + c;
    const auto emit = [&](auto plain) {
#pragma unroll
      for (int i = 0; i < L; ++i) {
        if (!plain && i >= n) continue;
        const bool start = !plain && (at.first >> i & 1);
        h = start ? B[i] : fma(A[i], h, B[i]);
        Vec<V> out = h;
        if (kGate) {
          const Vec<V> z = words.read(kZ, zs, a.z_stride, i);
          out = h * silu(z);
        }
        if (on) store_word<T, V>(y + i * a.y_stride, out);
        if (!plain && (at.last >> i & 1) && a.state && on)
          store_floats(a.state + (long long)index_of(a, kept, row + i) * a.channels + c, h);
      }
    };
    if (within) emit(std::true_type{});
    else emit(std::false_type{});
    fetch_outputs(round + 1);
  }
  finish_exchange(shared, blocks);
}

template <typename T, int V, bool kGate>
__global__ void __launch_bounds__(kThreads, 2) recurrence_backward_kernel(const __grid_constant__ RecArgs a) {
  constexpr int L = kBackwardRows, kTile = kWarps * L;
  extern __shared__ __align__(16) char staged[];
  __shared__ __align__(16) Exchange<V> shared;
  __shared__ Stretch<V> states[2][kWarps][32];
  __shared__ int kept[kKeptOffsets + 1];
  grid_dependency_wait();
  keep_offsets(a, kept);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int blocks = a.cluster, rank = blockIdx.x % blocks;
  const int channel = (blockIdx.x / blocks * 32 + lane) * V;
  const bool on = channel < a.channels;
  const int c = on ? channel : 0;
  int begin, end;
  segment_rows(a, kept, begin, end);
  if (rank == 0) pass_empty<V>(a, kept, a.dstate, a.dstate0, c, on);
  const int tiles = (end - begin + kTile - 1) / kTile, rounds = (tiles + blocks - 1) / blocks;
  const int group = blockIdx.x / blocks * 32 * V;  // the first lane's channel
  const Words<T, V, L> words{staged + warp * (L * 128), a.wide, group, a.channels};
  enum { kX, kG = 2, kDy, kZ };  // slots: x has two, it is read to the end of its round
  const T* const x0 = static_cast<const T*>(a.x) + group;
  const T* const g0 = static_cast<const T*>(a.g) + group;
  const T* const dy0 = static_cast<const T*>(a.dy) + group;
  const T* const z0 = static_cast<const T*>(a.z) + group;
  const Vec<V> bias = a.bias ? load_floats<V>(a.bias + c) : all_of<V>(0.f);
  Vec<V> carry = all_of<V>(0.f), dbias = all_of<V>(0.f);
  start_exchange(shared, blocks);
  // the last rows come first
  const auto tile_of = [&](int round) { return tiles - 1 - (round * blocks + rank); };
  const auto row_of = [&](int round) { return begin + (tile_of(round) * kWarps + warp) * L; };
  const auto rows_at = [&](int round) { return tile_of(round) < 0 ? 0 : max(0, min(L, end - row_of(round))); };
  const auto fetch_inputs = [&](int round) {
    words.release();
    const int row = row_of(round);
    const int n = rows_at(round);
    words.fetch(kX + (int)(round & 1), x0 + (long long)row * a.x_stride, a.x_stride, n);
    words.fetch(kG, g0 + (long long)row * a.g_stride, a.g_stride, n);
    words.commit();
  };
  const auto fetch_outputs = [&](int round) {
    words.release();
    const int row = row_of(round);
    const int n = rows_at(round);
    words.fetch(kDy, dy0 + (long long)row * a.dy_stride, a.dy_stride, n);
    if (kGate) words.fetch(kZ, z0 + (long long)row * a.z_stride, a.z_stride, n);
    words.commit();
  };
  fetch_inputs(0);
  fetch_outputs(0);
  Sequence in{0, 0, 0};
  for (int round = 0; round < rounds; ++round) {
    const int stage = (int)(round & 1);
    const int row = row_of(round), tile = tile_of(round);
    const int n = rows_at(round);
    const T* const xs = x0 + (long long)row * a.x_stride;
    const T* const gs = g0 + (long long)row * a.g_stride;
    const T* const dys = dy0 + (long long)row * a.dy_stride;
    const T* const zs = z0 + (long long)row * a.z_stride;
    // the state before the tile
    Vec<V> h = tile < 0 ? all_of<V>(0.f)
                        : load_floats<V>(a.checkpoints + (long long)(blockIdx.y * a.checkpoints_per_segment + tile) * a.channels + c);
    words.wait();
    const Borders at = borders(a, kept, row, n, in);
    const bool within = n == L && at.first == 0 && at.last == 0;  // all rows there, none at a sequence's border
    // the states of the warp's rows: its stretch, those of the warps before it, and from row to row
    Vec<V> A[L], B[L], P[L], E[L];  // gates, states before each row, what enters each row from its output
    Stretch<V> mine = nothing<V>();
    const auto scan = [&](auto plain) {
#pragma unroll
      for (int i = 0; i < L; ++i) {
        if (plain || i < n) {
          gate_of(words.read(kG, gs, a.g_stride, i) + bias, A[i], B[i]);
          const Vec<V> in_x = B[i] * words.read(kX + stage, xs, a.x_stride, i);
          if (!plain && (at.first >> i & 1)) {
            P[i] = a.state0 ? load_floats<V>(a.state0 + (long long)index_of(a, kept, row + i) * a.channels + c) : all_of<V>(0.f);
            mine = Stretch<V>{all_of<V>(-1.f), fma(A[i], P[i], in_x)};
          } else {
            const bool cut = !plain && mine.A.x < 0.f;
            mine = Stretch<V>{cut ? mine.A : mine.A * A[i], fma(A[i], mine.H, in_x)};
          }
        } else {
          A[i] = all_of<V>(1.f), B[i] = all_of<V>(0.f);
        }
      }
    };
    if (within) scan(std::true_type{});
    else scan(std::false_type{});
    fetch_inputs(round + 1);
    states[stage][warp][lane] = mine;
    __syncthreads();
    for (int w = 0; w < warp; ++w) h = apply(states[stage][w][lane], h);
    words.wait();
    T* dz = static_cast<T*>(a.dz) + (long long)row * a.dz_stride + c;
    // forward from row to row; then back, what flows to the rows before: d -> A (E + d), nothing across the beginning
    // of a sequence
    mine = nothing<V>();
    const auto through = [&](auto plain) {
#pragma unroll
      for (int i = 0; i < L; ++i) {
        E[i] = all_of<V>(0.f);
        if (!plain && i >= n) continue;
        const Vec<V> dy = words.read(kDy, dys, a.dy_stride, i);
        const bool start = !plain && (at.first >> i & 1);
        P[i] = start ? P[i] : h;
        h = fma(A[i], P[i], B[i] * words.read(kX + stage, xs, a.x_stride, i));
        E[i] = dy;
        if (kGate) {
          const Vec<V> z = words.read(kZ, zs, a.z_stride, i), s = sigmoid(z), ds = dy * s;
          E[i] = ds * z;
          // dy h s (1 + z (1 - s))
          const Vec<V> slope = fma(z, fma(s, all_of<V>(-1.f), all_of<V>(1.f)), all_of<V>(1.f));
          if (a.dz && on) store_word<T, V>(dz + i * a.dz_stride, (ds * h) * slope);
        }
        if (!plain && (at.last >> i & 1) && a.dstate)
          E[i] = E[i] + load_floats<V>(a.dstate + (long long)index_of(a, kept, row + i) * a.channels + c);
      }
#pragma unroll
      for (int i = L - 1; i >= 0; --i) {
        if (!plain && i >= n) continue;
        const bool start = !plain && (at.first >> i & 1), cut = !plain && mine.A.x < 0.f;
        mine = start ? Stretch<V>{all_of<V>(-1.f), all_of<V>(0.f)}
                     : Stretch<V>{cut ? mine.A : mine.A * A[i], A[i] * (E[i] + mine.H)};
      }
    };
    if (within) through(std::true_type{});
    else through(std::false_type{});
    fetch_outputs(round + 1);
    Vec<V> d = exchange(shared, (uint32_t)round, kWarps - 1 - warp, rank, blocks, a, mine, carry);
    T* dx = static_cast<T*>(a.dx) + (long long)row * a.dx_stride + c;
    T* dg = static_cast<T*>(a.dg) + (long long)row * a.dg_stride + c;
    const auto emit = [&](auto plain) {
#pragma unroll
      for (int i = L - 1; i >= 0; --i) {
        if (!plain && i >= n) continue;
        d = d + E[i];
        const Vec<V> out = B[i] * d;
        const Vec<V> way = fma(words.read(kX + stage, xs, a.x_stride, i), all_of<V>(-1.f), P[i]);
        const Vec<V> gate = (out * A[i]) * way;
        dbias = dbias + gate;
        d = d * A[i];
        if (a.dx && on) store_word<T, V>(dx + i * a.dx_stride, out);
        if (a.dg && on) store_word<T, V>(dg + i * a.dg_stride, gate);
        if (!plain && (at.first >> i & 1)) {
          if (a.dstate0 && on) store_floats(a.dstate0 + (long long)index_of(a, kept, row + i) * a.channels + c, d);
          d = all_of<V>(0.f);
        }
      }
    };
    if (within) emit(std::true_type{});
    else emit(std::false_type{});
  }
  finish_exchange(shared, blocks);
  if (!a.sums) return;
  __syncthreads();
  states[0][warp][lane].H = dbias;
  __syncthreads();
  if (warp == 0 && on) {
    Vec<V> s = all_of<V>(0.f);
    for (int w = 0; w < kWarps; ++w) s = s + states[0][w][lane].H;
    store_floats(a.sums + ((long long)blockIdx.y * blocks + rank) * a.channels + c, s);
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
    const Vec<V> x = unpack<T, V>(load_word<T, V>(static_cast<const T*>(a.x) + s * a.x_stride + c));
    const Vec<V> g = unpack<T, V>(load_word<T, V>(static_cast<const T*>(a.g) + s * a.g_stride + c));
    float* const state = a.state + s * a.channels + c;
    Vec<V> fa, fb;
    gate_of(a.bias ? g + load_floats<V>(a.bias + c) : g, fa, fb);
    const Vec<V> h = fma(fa, load_floats<V>(state), fb * x);
    Vec<V> out = h;
    if (kGate) {
      const Vec<V> z = unpack<T, V>(load_word<T, V>(static_cast<const T*>(a.z) + s * a.z_stride + c));
      out = h * silu(z);
    }
    store_floats(state, h);
    store_word<T, V>(static_cast<T*>(a.y) + s * a.y_stride + c, out);
  }
}

// ---- host -------------------------------------------------------------------------------------------
struct Division {
  int tiles, segments;  // of channels; of sequences
  long long rows, per_segment, checkpoints;  // of a segment
};

// Blocks over channels, then over sequences of known borders, two to an SM; what is left goes to clusters over time.
Division division_of(const fbfftconv_recurrence_desc& d, int V) {
  Division s{};
  s.tiles = (d.channels + 32 * V - 1) / (32 * V);
  long long segments = d.offsets ? 1 : 2ll * sm_count() / s.tiles;
  if (segments > d.sequences) segments = d.sequences;
  if (segments < 1) segments = 1;
  s.per_segment = d.sequences > 0 ? (d.sequences + segments - 1) / segments : 1;
  s.segments = (int)(d.sequences > 0 ? (d.sequences + s.per_segment - 1) / s.per_segment : 1);
  s.rows = d.offsets ? d.rows : s.per_segment * d.length;
  s.checkpoints = (s.rows + kCheckpoint - 1) / kCheckpoint;
  return s;
}

cudaLaunchConfig_t config_of(const Division& s, int cluster, size_t smem, cudaStream_t stream, cudaLaunchAttribute (&attrs)[2]) {
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(s.tiles * cluster, s.segments);
  config.blockDim = dim3(kThreads);
  config.dynamicSmemBytes = smem;
  config.stream = stream;
  attrs[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attrs[0].val.programmaticStreamSerializationAllowed = 1;
  attrs[1].id = cudaLaunchAttributeClusterDimension;
  attrs[1].val.clusterDim.x = cluster, attrs[1].val.clusterDim.y = attrs[1].val.clusterDim.z = 1;
  config.attrs = attrs;
  config.numAttrs = cluster > 1 ? 2 : 1;
  return config;
}

// Clusters of a size that the current GPU holds at once, asked once for each kernel and device.
constexpr int kMostDevices = 64;     // of a process
constexpr int kDividedKernels = 20;  // those below: two directions, five element layouts, with and without the output gate
int resident_clusters(const void* kernel, int cluster, size_t smem) {
  struct Known {
    const void* kernel;
    int16_t clusters[kMostCluster + 1];
  };
  static Known known[kMostDevices][kDividedKernels];
  static std::mutex lock;
  const std::lock_guard<std::mutex> hold(lock);
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess || device < 0 || device >= kMostDevices) return 0;
  Known* k = known[device];
  while (k < known[device] + kDividedKernels - 1 && k->kernel && k->kernel != kernel) ++k;
  if (k->kernel != kernel) *k = Known{kernel, {}};
  if (k->clusters[cluster] == 0) {
    Division one{};
    one.tiles = one.segments = 1;
    cudaLaunchAttribute attrs[2]{};
    const cudaLaunchConfig_t config = config_of(one, cluster, smem, nullptr, attrs);
    int n = 0;
    cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);  // clusters of more than 8 blocks
    if (cudaOccupancyMaxActiveClusters(&n, kernel, &config) != cudaSuccess) cudaGetLastError(), n = 0;
    k->clusters[cluster] = n > 0 ? (int16_t)n : -1;
  }
  return k->clusters[cluster];
}

// The widest cluster of which the GPU holds as many at once as there are: those that are left would begin when the others
// have ended (131072 x 1024 f16 forward by 16 clusters: of 16 blocks, of which 14 are held, 545 us, of 13 blocks 420).
// Narrower ones are slower, a round takes as long with fewer rows (8, 9, 11 and 12 blocks: 620, 556, 490 and 452 us).  A
// block has at least one round of rows.
template <typename K>
cudaError_t launch_divided(K kernel, RecArgs a, const Division& s, int tile_rows, size_t smem, int* parts, cudaStream_t stream) {
  const void* const pointer = reinterpret_cast<const void*>(kernel);
  cudaError_t e = ensure_dynamic_smem(pointer, (int)smem);
  const long long groups = (long long)s.tiles * s.segments, tiles = (s.rows + tile_rows - 1) / tile_rows;
  a.cluster = 1;
  if (e != cudaSuccess) return e;
  if (tiles > 1 && groups < 2ll * sm_count())
    for (int c = (int)(tiles < kMostCluster ? tiles : kMostCluster); c > 1 && a.cluster == 1; --c)
      if (resident_clusters(pointer, c, smem) >= groups) a.cluster = c;
  if (parts) *parts = s.segments * a.cluster;
  cudaLaunchAttribute attrs[2]{};
  const cudaLaunchConfig_t config = config_of(s, a.cluster, smem, stream, attrs);
  e = cudaLaunchKernelEx(&config, kernel, a);
  if (e != cudaSuccess) cudaGetLastError();  // returned here; the next launch must not report it again
  return e;
}

template <typename T, int V>
cudaError_t forward(const RecArgs& a, const Division& s, cudaStream_t stream) {
  constexpr size_t slot = sizeof(T) * V == 4 ? kForwardRows * kThreads * 4 : 0;
  constexpr int tile = kWarps * kForwardRows;
  return a.z ? launch_divided(recurrence_forward_kernel<T, V, true>, a, s, tile, 3 * slot, nullptr, stream)
             : launch_divided(recurrence_forward_kernel<T, V, false>, a, s, tile, 2 * slot, nullptr, stream);
}

template <typename T, int V>
cudaError_t backward(const RecArgs& a, const Division& s, int* parts, cudaStream_t stream) {
  constexpr size_t slot = sizeof(T) * V == 4 ? kBackwardRows * kThreads * 4 : 0;
  constexpr int tile = kWarps * kBackwardRows;
  return a.z ? launch_divided(recurrence_backward_kernel<T, V, true>, a, s, tile, 5 * slot, parts, stream)
             : launch_divided(recurrence_backward_kernel<T, V, false>, a, s, tile, 4 * slot, parts, stream);
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
  if (d->sequences > kMostRows || d->length > kMostRows || d->rows > kMostRows)
    return op_fail(FBFFTCONV_ERR_UNSUPPORTED_SIZE, "more than 2^30 sequences or rows");
  const int64_t strides[] = {d->x_stride, d->g_stride, d->z_stride, d->y_stride, d->grad_y_stride, d->grad_x_stride,
                             d->grad_g_stride, d->grad_z_stride};
  for (const int64_t s : strides)
    if (s < 0) return op_fail(FBFFTCONV_ERR_INVALID_ARGUMENT, "negative stride");
    else if (s > (1ll << 26)) return op_fail(FBFFTCONV_ERR_UNSUPPORTED_SIZE, "more than 2^26 elements between rows");
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
                       int device, bool* pairs, bool* wide) {
  const int piece = 16 / type_bytes(d.type);
  *pairs = d.channels % 2 == 0;
  *wide = d.channels % piece == 0;
  for (const RowPointer& q : rows) {
    if (!q.p && q.needed) return op_fail(FBFFTCONV_ERR_INVALID_ARGUMENT, "%s is null", q.name);
    if (!aligned_to(q.p, type_bytes(d.type))) return op_fail(FBFFTCONV_ERR_INVALID_ARGUMENT, "%s is not aligned to its element", q.name);
    if (q.p && q.stride < d.channels) return op_fail(FBFFTCONV_ERR_INVALID_ARGUMENT, "the rows of %s overlap", q.name);
    if (q.p && (q.stride % 2 || !aligned_to(q.p, 2 * type_bytes(d.type)))) *pairs = false;
    if (q.p && (q.stride % piece || !aligned_to(q.p, 16))) *wide = false;
  }
  for (const RowPointer& q : floats) {
    if (!q.p && q.needed) return op_fail(FBFFTCONV_ERR_INVALID_ARGUMENT, "%s is null", q.name);
    if (!aligned_to(q.p, 4)) return op_fail(FBFFTCONV_ERR_INVALID_ARGUMENT, "%s is not aligned to its element", q.name);
  }
  for (const RowPointer& q : rows) OP_TRY(validate_device_pointer(device, q.p, q.name));
  for (const RowPointer& q : floats) OP_TRY(validate_device_pointer(device, q.p, q.name));
  return validate_device_pointer(device, d.offsets, "offsets");
}

std::atomic<uint32_t> wait_polls{kPolls};

// A word for each device, in host memory that its kernels write: what a call lost is known to the next one without a wait
// for the device.  Null where there is none to be had.
int* wait_error_of(int device) {
  static std::atomic<int*> known{nullptr};
  static std::mutex lock;
  int* words = known.load(std::memory_order_acquire);
  if (!words) {
    const std::lock_guard<std::mutex> hold(lock);
    words = known.load(std::memory_order_acquire);
    if (!words) {
      // the first call of a process may be one that is captured, which does not concern this allocation
      cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
      cudaThreadExchangeStreamCaptureMode(&mode);
      void* p = nullptr;
      const cudaError_t e = cudaHostAlloc(&p, kMostDevices * sizeof(int), cudaHostAllocPortable | cudaHostAllocMapped);
      cudaThreadExchangeStreamCaptureMode(&mode);
      if (e != cudaSuccess) {
        cudaGetLastError();
        return nullptr;
      }
      words = static_cast<int*>(p);
      memset(words, 0, kMostDevices * sizeof(int));
      known.store(words, std::memory_order_release);
    }
  }
  return device >= 0 && device < kMostDevices ? words + device : nullptr;
}

int take_wait_error(int device, int** out) {
  *out = wait_error_of(device);
  if (!*out) return op_fail(FBFFTCONV_ERR_NOMEM, "no host memory for the waits' status");
  if (*static_cast<volatile int*>(*out))
    return op_fail(FBFFTCONV_ERR_CUDA, "a recurrence gave up a bounded wait: results since the last fbfftconv_recurrence_status(1) are incomplete");
  return FBFFTCONV_OK;
}

RecArgs common_args(const fbfftconv_recurrence_desc& d) {
  const auto or_dense = [&](int64_t s) { return s ? (int)s : d.channels; };
  RecArgs a{};
  a.rows = (int)d.rows, a.length = (int)d.length, a.sequences = (int)d.sequences, a.channels = d.channels;
  a.offsets = d.offsets, a.wide_offsets = d.wide_offsets, a.polls = wait_polls.load(std::memory_order_relaxed);
  a.never = a.polls ? 0 : 16;
  a.x_stride = or_dense(d.x_stride), a.g_stride = or_dense(d.g_stride), a.z_stride = or_dense(d.z_stride);
  a.y_stride = or_dense(d.y_stride), a.dy_stride = or_dense(d.grad_y_stride);
  a.dx_stride = or_dense(d.grad_x_stride), a.dg_stride = or_dense(d.grad_g_stride), a.dz_stride = or_dense(d.grad_z_stride);
  return a;
}

// 16-bit channels travel in pairs or alone, which changes how many blocks share the channels; what is kept between the
// passes must not depend on that.
Division division_for(const fbfftconv_recurrence_desc& d, bool pairs) {
  const int V = d.type == FBFFTCONV_FLOAT32 ? 1 : 2;
  Division s = division_of(d, V);
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
  const Division s = division_for(*desc, true);
  return (size_t)(s.segments * s.checkpoints) * desc->channels * sizeof(float);
}

size_t fbfftconv_recurrence_workspace_bytes(const fbfftconv_recurrence_desc* desc) {
  if (check_desc(desc) != FBFFTCONV_OK) return 0;
  int device;
  if (resolve_device(desc->device, &device) != FBFFTCONV_OK) return 0;
  const OnDevice on(device);
  const Division s = division_for(*desc, true);
  return (size_t)s.segments * kMostCluster * desc->channels * sizeof(float);
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
  OP_TRY(check_rec_pointers(rows, floats, d, device, &pairs, &a.wide));
  if (d.sequences == 0) return FBFFTCONV_OK;
  const OnDevice on(device);
  if (on.error() != cudaSuccess) return op_cuda_fail(on.error(), "cudaSetDevice");
  OP_TRY(take_wait_error(device, &a.wait_error));
  const Division s = division_for(d, pairs);
  a.x = x, a.g = g, a.z = z, a.bias = bias, a.state0 = state0, a.y = y, a.state = state, a.checkpoints = checkpoints;
  a.per_segment = (int)s.per_segment, a.checkpoints_per_segment = (int)s.checkpoints;
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
  OP_TRY(check_rec_pointers(rows, floats, d, device, &pairs, &a.wide));
  const OnDevice on(device);
  if (on.error() != cudaSuccess) return op_cuda_fail(on.error(), "cudaSetDevice");
  const Division s = division_for(d, pairs);
  int parts = 0;
  if (grad_bias && d.sequences > 0 && workspace_bytes < (size_t)s.segments * kMostCluster * d.channels * sizeof(float))
    return op_fail(FBFFTCONV_ERR_INVALID_ARGUMENT, "the workspace is smaller than fbfftconv_recurrence_workspace_bytes");
  const cudaStream_t cuda_stream = static_cast<cudaStream_t>(stream);
  if (d.sequences > 0) {
    OP_TRY(take_wait_error(device, &a.wait_error));
    a.x = x, a.g = g, a.z = z, a.bias = bias, a.state0 = state0, a.checkpoints = const_cast<float*>(checkpoints);
    a.dy = grad_y, a.dstate = grad_state, a.dx = grad_x, a.dg = grad_g, a.dz = grad_z, a.dstate0 = grad_state0;
    a.sums = grad_bias ? static_cast<float*>(workspace) : nullptr;
    a.per_segment = (int)s.per_segment, a.checkpoints_per_segment = (int)s.checkpoints;
    count_launch();
#define BACKWARD(T, V) backward<T, V>(a, s, &parts, cuda_stream)
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

int fbfftconv_recurrence_status(int reset) {
  int device;
  if (cudaGetDevice(&device) != cudaSuccess || cudaDeviceSynchronize() != cudaSuccess) {
    cudaGetLastError();
    return -1;
  }
  volatile int* const word = wait_error_of(device);
  if (!word) return -1;
  const int code = *word;
  if (reset) *word = 0;
  return code;
}

uint32_t fbfftconv_recurrence_wait_limit(uint32_t microseconds) { return wait_polls.exchange(microseconds); }

int fbfftconv_recurrence_wait_selftest(fbfftconv_stream stream) {
  int* out = nullptr;
  cudaError_t e = cudaMalloc(&out, sizeof(int));
  int gave_up = 0;
  if (e == cudaSuccess) {
    count_launch();
    wait_probe_kernel<<<1, 1, 0, static_cast<cudaStream_t>(stream)>>>(out);
    e = cudaGetLastError();
    if (e == cudaSuccess) e = cudaStreamSynchronize(static_cast<cudaStream_t>(stream));
    if (e == cudaSuccess) e = cudaMemcpy(&gave_up, out, sizeof(int), cudaMemcpyDeviceToHost);
    cudaFree(out);
  }
  if (e != cudaSuccess) return op_cuda_fail(e, "recurrence, wait");
  return gave_up ? FBFFTCONV_OK : op_fail(FBFFTCONV_ERR_CUDA, "the wait did not give up");
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
  OP_TRY(check_rec_pointers(rows, floats, d, device, &pairs, &a.wide));
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
