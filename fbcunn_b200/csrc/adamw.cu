// One AdamW step over many tensors (sm_100a).
//
//   m = b1 m + (1 - b1) g        v = b2 v + (1 - b2) g^2
//   p = p (1 - lr wd) - lr (m / (1 - b1^t)) / (sqrt(v / (1 - b2^t)) + eps)
//
// Every element is read and written once, so HBM bounds it.  A warp takes a block of 256 elements of one tensor at a
// time, eight to a lane: with 8-bit moments those are the elements that share a scale, whose largest magnitude is then
// one redux.sync away, and nothing passes through shared memory.  The table of tensors travels in the kernel's
// parameters: a captured step holds its own copy, and no upload can be overtaken by the next step's.
//
// 8-bit moments: m and sqrt(v) in e4m3, 448 standing for the block's largest magnitude.  The root is held, not v,
// because its exponents span half as many powers of two.  Both are rounded up or down at random, by a hash of (seed,
// step, tensor, element), in proportion to what is cut off: with b2 = 0.999 a step moves sqrt(v) by some 5e-4 of
// itself, a code by 6e-2 or more, so rounding to nearest would never move it.  A root that is not zero is never stored
// as zero: the type's lowest value (block maximum / 2.3e5) bounds the next step's m / sqrt(v).
#include <cuda_fp8.h>
#include <float.h>
#include <math.h>

#include <algorithm>
#include <atomic>
#include <memory>
#include <new>
#include <type_traits>
#include <utility>
#include <vector>

#include "operators.cuh"

struct fbfftconv_adamw {
  std::vector<fbfftconv_adamw_tensor> tensors;
  fbfftconv_adamw_options options;
  int device;
};

namespace fbfft {
namespace {

constexpr int kBlock = 256;           // elements that share a scale, and a warp's share
constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr long long kMostElements = 1ll << 38, kMostBlocks = 1ll << 30;  // of a tensor, of a launch
constexpr float kTiny = 7.8886090522101181e-31f;  // 2^-100: a block below it is stored as zeros, its scale would overflow

struct Entry {
  void* param;
  float* master;
  const void* grad;
  void* moment1;
  void* moment2;
  float* scale1;
  float* scale2;
  long long count;
  int first;          // first block of this tensor among the launch's
  uint8_t param_type, grad_type, vectors, pad;
  uint32_t index;     // in the caller's list: part of the hash
};

struct Common {
  float beta1, beta2, rest1, rest2, eps;  // rest = 1 - beta, rounded from 64 bits
  float log_beta1, log_beta2;
  float lr, weight_decay, grad_scale;
  const float* scalars;  // lr and grad_scale on the device, or null
  long long* steps;      // steps done; blocks that are through with this launch
  uint32_t seed;
  int tensors, blocks, advance;
  int run;               // blocks in a row that a warp takes, or 0: every so many-th, as many as there are warps
};

// 4 KB of parameters reach every device; larger tables take the extended limit.
constexpr int kFew = 44, kSome = 128, kMany = 400;
template <int N> struct Table {
  Common c;
  Entry entry[N];
};
static_assert(sizeof(Table<kFew>) <= 4096 && sizeof(Table<kMany>) <= 32764, "kernel parameters");

__device__ __forceinline__ uint32_t mix(uint32_t x) {
  x ^= x >> 16;
  x *= 0x6A09E667u;
  x ^= x >> 15;
  x *= 0xBB67AE85u;
  return x ^ (x >> 16);
}

// Eight neighbours of a lane, where all of the tensor's pointers are aligned.
template <typename T>
__device__ __forceinline__ void load8(const void* base, long long at, float (&x)[8]) {
  const uint4 q = *reinterpret_cast<const uint4*>(static_cast<const T*>(base) + at);
  const uint32_t u[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = unpack2<T>(u[i]);
    x[2 * i] = f.x, x[2 * i + 1] = f.y;
  }
}
template <>
__device__ __forceinline__ void load8<float>(const void* base, long long at, float (&x)[8]) {
  const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(base) + at);
  const float4 a = p[0], b = p[1];
  x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
}

template <typename T>
__device__ __forceinline__ void store8(void* base, long long at, const float (&x)[8]) {
  *reinterpret_cast<uint4*>(static_cast<T*>(base) + at) =
      make_uint4(pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]), pack2<T>(x[4], x[5]), pack2<T>(x[6], x[7]));
}
template <>
__device__ __forceinline__ void store8<float>(void* base, long long at, const float (&x)[8]) {
  float4* p = reinterpret_cast<float4*>(static_cast<float*>(base) + at);
  p[0] = make_float4(x[0], x[1], x[2], x[3]);
  p[1] = make_float4(x[4], x[5], x[6], x[7]);
}

// Elsewhere a lane has every 32nd element, which is coalesced at any alignment; `left` elements of the block exist.
__device__ __forceinline__ void load_each(const void* base, long long at, int left, int type, float (&x)[8]) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int j = lane + 32 * i;
    x[i] = 0.f;
    if (j >= left) continue;
    if (type == FBFFTCONV_FLOAT32) x[i] = static_cast<const float*>(base)[at + j];
    else if (type == FBFFTCONV_BFLOAT16) x[i] = to_float(static_cast<const __nv_bfloat16*>(base)[at + j]);
    else x[i] = to_float(static_cast<const __half*>(base)[at + j]);
  }
}

__device__ __forceinline__ void store_each(void* base, long long at, int left, int type, const float (&x)[8]) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int j = lane + 32 * i;
    if (j >= left) continue;
    if (type == FBFFTCONV_FLOAT32) static_cast<float*>(base)[at + j] = x[i];
    else if (type == FBFFTCONV_BFLOAT16) static_cast<__nv_bfloat16*>(base)[at + j] = from_float<__nv_bfloat16>(x[i]);
    else static_cast<__half*>(base)[at + j] = from_float<__half>(x[i]);
  }
}

__device__ __forceinline__ float2 decode2(uint32_t codes) {
  return __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)codes, __NV_E4M3)));
}

template <bool kVectors>
__device__ __forceinline__ void load_codes(const uint8_t* base, long long at, int left, float scale, float (&x)[8]) {
  const int lane = threadIdx.x & 31;
  if (kVectors) {
    const uint2 q = *reinterpret_cast<const uint2*>(base + at + 8 * lane);
    const uint32_t u[2] = {q.x, q.y};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = decode2(u[i >> 1] >> (16 * (i & 1)) & 0xffffu);
      x[2 * i] = f.x * scale, x[2 * i + 1] = f.y * scale;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int j = lane + 32 * i;
      x[i] = j < left ? decode2(base[at + j]).x * scale : 0.f;
    }
  }
}

// Four codes, the lowest bytes of c, with the signs of x.
__device__ __forceinline__ uint32_t pack_codes(const uint32_t* c) {
  return __byte_perm(__byte_perm(c[0], c[1], 0x0040), __byte_perm(c[2], c[3], 0x0040), 0x5410);
}
__device__ __forceinline__ uint32_t pack_codes(const uint32_t* c, const float* x) {
  const uint32_t a = __byte_perm(__float_as_uint(x[0]), __float_as_uint(x[1]), 0x0073);
  const uint32_t b = __byte_perm(__float_as_uint(x[2]), __float_as_uint(x[3]), 0x0073);
  return pack_codes(c) | (__byte_perm(a, b, 0x5410) & 0x80808080u);
}

// The codes of both moments, the first's with the signs of m.
template <bool kVectors>
__device__ __forceinline__ void store_codes(uint8_t* first, uint8_t* second, long long at, int left, const uint32_t (&c1)[8],
                                            const float (&m)[8], const uint32_t (&c2)[8]) {
  const int lane = threadIdx.x & 31;
  if (kVectors) {
    *reinterpret_cast<uint2*>(first + at + 8 * lane) = make_uint2(pack_codes(c1, m), pack_codes(c1 + 4, m + 4));
    *reinterpret_cast<uint2*>(second + at + 8 * lane) = make_uint2(pack_codes(c2), pack_codes(c2 + 4));
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int j = lane + 32 * i;
      if (j >= left) continue;
      first[at + j] = (uint8_t)((c1[i] & 0x7Fu) | (__float_as_uint(m[i]) >> 24 & 0x80u));
      second[at + j] = (uint8_t)c2[i];
    }
  }
}

// A random number in [0, 1) from 16 bits: behind the exponent of 128 they are its last places.
__device__ __forceinline__ float uniform_low(uint32_t h) { return __uint_as_float(__byte_perm(h, 0x43000000u, 0x7610)) - 128.f; }
__device__ __forceinline__ float uniform_high(uint32_t h) { return __uint_as_float(__byte_perm(h, 0x43000000u, 0x7632)) - 128.f; }

// The e4m3 code of size >= 0 without its sign, in the lowest byte: size is cut to a multiple of its binade's step (at
// least the subnormals' 2^-9) after `uniform` in [0, 1) steps were added, and is at least `least` steps.  The steps n, at
// most 16, are the last places of the sum rounded down at 2^23; with 8 codes to a binade the code is 8 (binade -
// lowest) + n, and the lowest binade's 8 * 121 is 256 * 4 less the 56 that the sum gets besides.  The largest size,
// 448 (1 + 2^-22) = 14.000004 steps, and the largest uniform, 1 - 2^-16, do not reach 15.
__device__ __forceinline__ uint32_t round8(float size, float uniform, float least) {
  const uint32_t top = max(__float_as_uint(size) & 0x7f800000u, 121u << 23);
  const float steps = fmaxf(fmaf(size, __uint_as_float((257u << 23) - top), uniform), least);
  uint32_t code;
  asm("mad.hi.u32 %0, %1, 4096, %2;" : "=r"(code) : "r"(top), "r"(__float_as_uint(__fadd_rd(steps, 8388608.f + 56.f))));
  return code;
}

// The largest magnitude of a block; NaN if it holds one, which so reaches all of it.
__device__ __forceinline__ float magnitude(const float (&x)[8]) {
  float top = fabsf(x[0]);
#pragma unroll
  for (int i = 1; i < 8; ++i) asm("max.NaN.f32 %0, %0, %1;" : "+f"(top) : "f"(fabsf(x[i])));
  return __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top)));  // NaN's bits are above infinity's
}

// Flushed, what is below the smallest normal number counts as zero: a root that is then below 2^-63 is nothing beside eps,
// unless eps is nearly as small (`small_eps`): a kernel of its own takes the others then, which are some instructions more
// (134M elements in one tensor with masters and 8-bit moments 434 us and 459; 32-bit moments take as long).
template <bool kFlush> __device__ __forceinline__ float sqrt_fast(float v) {
  float s;
  if (kFlush) asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(s) : "f"(v));
  else asm("sqrt.approx.f32 %0, %1;" : "=f"(s) : "f"(v));
  return s;
}

// sqrt(v) after one of Newton's steps: within one place of the rounded root, and nearly always equal to it.  At zero
// and infinity the step is NaN, which the minimum drops.
template <bool kFlush> __device__ __forceinline__ float sqrt_near(float v) {
  const float s = sqrt_fast<kFlush>(v);
  float r;
  if (kFlush) asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  else asm("rsqrt.approx.f32 %0, %1;" : "=f"(r) : "f"(v));
  return s + fminf(fmaf(-s, s, v) * (0.5f * r), s);
}

__device__ __forceinline__ float reciprocal(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

struct Step {
  float decay, size, root_scale, grad_scale;  // p's factor, lr / (1 - b1^t), 1 / sqrt(1 - b2^t)
  uint32_t key;
};

// A warp's blocks of one tensor: `block`, `block + stride`, ... below `end`.
// P and G are the types of parameter and gradient where vectors are loaded; elsewhere the entry's are looked up.
template <bool kVectors, bool kPacked, bool kMaster, bool kFlush, typename P, typename G>
__device__ __forceinline__ void update_blocks(const Entry& e, const Common& c, const Step& s, int block, int end, int stride) {
  const int lane = threadIdx.x & 31;
  using Weight = std::conditional_t<kMaster, float, P>;
  const bool has_master = kVectors ? kMaster : e.master != nullptr;
  void* const param = e.param;
  void* const weights = has_master ? e.master : param;
  const int param_type = e.param_type, grad_type = e.grad_type, weight_type = has_master ? FBFFTCONV_FLOAT32 : param_type;
  const void* const grad = e.grad;
  void* const moment1 = e.moment1;
  void* const moment2 = e.moment2;
  float* const scale1 = e.scale1;
  float* const scale2 = e.scale2;
  const uint32_t tensor_key = kPacked ? mix(s.key + e.index) : 0;
  for (; block < end; block += stride) {
    const long long base = (long long)block * kBlock;
    const int left = kVectors ? kBlock : (int)min((long long)kBlock, e.count - base);
    const long long mine = base + 8 * lane;
    float p[8], g[8], m[8], v[8];
    if (kVectors) {
      load8<G>(grad, mine, g);
      load8<Weight>(weights, mine, p);
    } else {
      load_each(grad, base, left, grad_type, g);
      load_each(weights, base, left, weight_type, p);
    }
    if (kPacked) {
      load_codes<kVectors>(static_cast<const uint8_t*>(moment1), base, left, scale1[block], m);
      load_codes<kVectors>(static_cast<const uint8_t*>(moment2), base, left, scale2[block], v);
    } else if (kVectors) {
      load8<float>(moment1, mine, m);
      load8<float>(moment2, mine, v);
    } else {
      load_each(moment1, base, left, FBFFTCONV_FLOAT32, m);
      load_each(moment2, base, left, FBFFTCONV_FLOAT32, v);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      // one rounding to an operation, nothing contracted: whoever follows the formulas in fp32 gets the same codes
      g[i] = __fmul_rn(g[i], s.grad_scale);
      m[i] = __fadd_rn(__fmul_rn(m[i], c.beta1), __fmul_rn(g[i], c.rest1));
      if (kPacked) v[i] = __fmul_rn(v[i], v[i]);
      v[i] = __fadd_rn(__fmul_rn(v[i], c.beta2), __fmul_rn(__fmul_rn(g[i], g[i]), c.rest2));
      const float root = kPacked ? sqrt_near<kFlush>(v[i]) : sqrt_fast<kFlush>(v[i]);
      p[i] = p[i] * s.decay - s.size * m[i] * reciprocal(fmaf(root, s.root_scale, c.eps));
      if (kPacked) v[i] = root;
    }
    if (kVectors) store8<Weight>(weights, mine, p);
    else store_each(weights, base, left, weight_type, p);
    if (has_master) {
      if (kVectors) store8<P>(param, mine, p);
      else store_each(param, base, left, param_type, p);
    }
    if (kPacked) {
      const float top1 = magnitude(m), top2 = magnitude(v);
      const bool none1 = top1 < kTiny, none2 = top2 < kTiny;
      const float to1 = none1 ? 0.f : 448.f * __frcp_rn(top1), to2 = none2 ? 0.f : 448.f * __frcp_rn(top2);
      const uint32_t key = tensor_key + (uint32_t)((unsigned long long)base >> 32) * 0x9E3779B9u;
      uint32_t code1[8], code2[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t element = (uint32_t)base + (kVectors ? 8 * lane + i : lane + 32 * i);
        const uint32_t h = mix(element ^ key);
        const float y = v[i] * to2;
        code1[i] = round8(fabsf(m[i] * to1), uniform_low(h), 0.f);
        code2[i] = round8(y, uniform_high(h), fminf(y * 0x1p+126f, 1.f));  // what is not zero has a step at least
      }
      if (!(top1 <= FLT_MAX && top2 <= FLT_MAX)) {  // NaN where a scaled value is none, zero elsewhere
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          code1[i] = isnan(m[i] * to1) ? 0x7Fu : top1 <= FLT_MAX ? code1[i] : 0u;
          code2[i] = isnan(v[i] * to2) ? 0x7Fu : top2 <= FLT_MAX ? code2[i] : 0u;
        }
      }
      store_codes<kVectors>(static_cast<uint8_t*>(moment1), static_cast<uint8_t*>(moment2), base, left, code1, m, code2);
      if (lane == 0) {
        scale1[block] = none1 ? 0.f : top1 * (1.f / 448);
        scale2[block] = none2 ? 0.f : top2 * (1.f / 448);
      }
    } else if (kVectors) {
      store8<float>(moment1, mine, m);
      store8<float>(moment2, mine, v);
    } else {
      store_each(moment1, base, left, FBFFTCONV_FLOAT32, m);
      store_each(moment2, base, left, FBFFTCONV_FLOAT32, v);
    }
  }
}

template <bool kPacked, bool kMaster, bool kFlush, typename P, typename G>
__device__ __forceinline__ void update_whole(const Entry& e, const Common& c, const Step& s, int block, int end, int stride) {
  update_blocks<true, kPacked, kMaster, kFlush, P, G>(e, c, s, block, end, stride);
}

template <bool kPacked, bool kMaster, bool kFlush, typename P>
__device__ __forceinline__ void update_whole(const Entry& e, const Common& c, const Step& s, int block, int end, int stride) {
  if (e.grad_type == FBFFTCONV_FLOAT32) update_whole<kPacked, kMaster, kFlush, P, float>(e, c, s, block, end, stride);
  else if (e.grad_type == FBFFTCONV_BFLOAT16) update_whole<kPacked, kMaster, kFlush, P, __nv_bfloat16>(e, c, s, block, end, stride);
  else update_whole<kPacked, kMaster, kFlush, P, __half>(e, c, s, block, end, stride);
}

template <bool kPacked, bool kFlush>
__device__ __forceinline__ void update_tensor(const Entry& e, const Common& c, const Step& s, int block, int end, int stride) {
  // whole blocks by vectors where all of the tensor's pointers allow that; the last block may be cut
  const int whole = e.vectors ? (int)min((long long)end, e.count / kBlock) : 0;
  if (block < whole) {
    if (e.param_type == FBFFTCONV_FLOAT32) update_whole<kPacked, false, kFlush, float>(e, c, s, block, whole, stride);
    else if (e.param_type == FBFFTCONV_BFLOAT16 && e.master) update_whole<kPacked, true, kFlush, __nv_bfloat16>(e, c, s, block, whole, stride);
    else if (e.param_type == FBFFTCONV_BFLOAT16) update_whole<kPacked, false, kFlush, __nv_bfloat16>(e, c, s, block, whole, stride);
    else if (e.master) update_whole<kPacked, true, kFlush, __half>(e, c, s, block, whole, stride);
    else update_whole<kPacked, false, kFlush, __half>(e, c, s, block, whole, stride);
    block += (whole - block + stride - 1) / stride * stride;
  }
  if (block < end) update_blocks<false, kPacked, false, kFlush, float, float>(e, c, s, block, end, stride);
}

template <int N, bool kFlush>
__global__ void __launch_bounds__(kThreads) adamw_kernel(const __grid_constant__ Table<N> t) {
  __shared__ Step shared;
  const Common& c = t.c;
  grid_dependency_wait();
  if (threadIdx.x == 0) {
    const long long step = *reinterpret_cast<volatile long long*>(c.steps) + 1;
    const float lr = c.scalars ? c.scalars[0] : c.lr;
    shared.grad_scale = c.scalars ? c.scalars[1] : c.grad_scale;
    shared.decay = fmaf(-lr, c.weight_decay, 1.f);
    // 1 - b^t = -(exp(t log b) - 1), whose error is the logarithm's, 2^-24 of it, at every t
    shared.size = lr / -expm1f((float)step * c.log_beta1);
    shared.root_scale = 1.f / sqrtf(-expm1f((float)step * c.log_beta2));
    shared.key = mix(c.seed + (uint32_t)step * 0x9E3779B9u);
  }
  __syncthreads();
  const Step s = shared;
  const int warps = gridDim.x * kWarps, warp = blockIdx.x * kWarps + (threadIdx.x >> 5);
  const int stride = c.run ? 1 : warps;
  const int last = c.run ? min(c.blocks, (warp + 1) * c.run) : c.blocks;
  int k = 0;
  for (int b = c.run ? warp * c.run : warp; b < last;) {
    int lo = k, hi = c.tensors;  // the tensor that block b belongs to
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (t.entry[mid].first <= b) lo = mid;
      else hi = mid;
    }
    k = lo;
    const Entry& e = t.entry[k];
    const int end = min(last, k + 1 < c.tensors ? t.entry[k + 1].first : c.blocks);
    if (e.scale1) update_tensor<true, kFlush>(e, c, s, b - e.first, end - e.first, stride);
    else update_tensor<false, kFlush>(e, c, s, b - e.first, end - e.first, stride);
    b += (end - b + stride - 1) / stride * stride;
  }
  if (!c.advance) return;
  // the step's last launch counts it, once every block has read the count
  if (threadIdx.x == 0) {
    unsigned long long* arrived = reinterpret_cast<unsigned long long*>(c.steps) + 1;
    if (atomicAdd(arrived, 1ull) == gridDim.x - 1) {
      c.steps[0] += 1;
      *arrived = 0;
    }
  }
}

// Whether a root that is flushed, one of v < 2^-126, can be more than 2^-20 of eps: it is divided by sqrt(1 - b2^t), at the
// first step sqrt(1 - b2).
bool small_eps(const fbfftconv_adamw_options& o) { return o.eps * sqrt(1 - o.beta2) < 0x1p-43; }

int blocks_of(long long count) { return (int)((count + kBlock - 1) / kBlock); }

template <int N, bool kFlush>
cudaError_t launch(const fbfftconv_adamw* h, const int* tensors, int count, const Common& common, cudaStream_t stream) {
  Table<N> table;
  table.c = common;
  long long blocks = 0, packed_blocks = 0;
  for (int i = 0; i < count; ++i) {
    const fbfftconv_adamw_tensor& t = h->tensors[tensors[i]];
    const bool packed = t.scale1 != nullptr;
    Entry& e = table.entry[i];
    e = Entry{t.param, t.master, t.grad, t.moment1, t.moment2, t.scale1, t.scale2, t.count, (int)blocks,
              (uint8_t)t.param_type, (uint8_t)t.grad_type, 0, 0, (uint32_t)tensors[i]};
    e.vectors = aligned_to(t.param, 16) && aligned_to(t.master, 16) && aligned_to(t.grad, 16) &&
                aligned_to(t.moment1, packed ? 8 : 16) && aligned_to(t.moment2, packed ? 8 : 16);
    blocks += blocks_of(t.count);
    if (packed) packed_blocks += blocks_of(t.count);
  }
  table.c.tensors = count;
  table.c.blocks = (int)blocks;
  static std::atomic<int> known{0};  // the same on every device of this architecture
  int resident = known.load(std::memory_order_relaxed);
  if (resident == 0) {
    const cudaError_t e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&resident, adamw_kernel<N, kFlush>, kThreads, 0);
    if (e != cudaSuccess) return e;
    known.store(resident, std::memory_order_relaxed);
  }
  // 32-bit moments: many short-lived blocks, which keep the warps within one stretch of each tensor (134M elements in
  // 560 us at 16 rounds of blocks, 591 at 4, 677 at 1).  8-bit moments are bound by the instructions, a warp's start in a
  // tensor among them: one round, and a warp's blocks in a row (134M elements in 40 tensors 459 us, every so many-th at 4
  // rounds 490; 11M in 60 tensors 37 and 47; in one tensor, which has few starts, 134M take 425 and 414).
  const int rounds = 2 * packed_blocks > blocks ? 1 : 16;
  const long long most = (long long)sm_count() * resident * rounds, need = (blocks + kWarps - 1) / kWarps;
  const int grid = (int)(need < 1 ? 1 : need < most ? need : most);
  if (rounds == 1) table.c.run = (int)((blocks + (long long)grid * kWarps - 1) / ((long long)grid * kWarps));
  count_launch();
  return launch_dependent(adamw_kernel<N, kFlush>, dim3(grid), kThreads, 0, stream, table);
}

template <int N>
cudaError_t launch(const fbfftconv_adamw* h, const int* tensors, int count, const Common& common, cudaStream_t stream) {
  return small_eps(h->options) ? launch<N, false>(h, tensors, count, common, stream)
                               : launch<N, true>(h, tensors, count, common, stream);
}

int check_tensor(const fbfftconv_adamw_tensor& t, int i) {
  if (t.count < 0) return op_fail(FBFFTCONV_ERR_INVALID_ARGUMENT, "tensor %d: negative element count", i);
  if (t.count > kMostElements) return op_fail(FBFFTCONV_ERR_UNSUPPORTED_SIZE, "tensor %d: more than 2^38 elements", i);
  if (!known_type(t.param_type) || !known_type(t.grad_type))
    return op_fail(FBFFTCONV_ERR_INVALID_ARGUMENT, "tensor %d: unknown element type", i);
  if (!t.scale1 != !t.scale2)
    return op_fail(FBFFTCONV_ERR_INVALID_ARGUMENT, "tensor %d: both moments are held in 8 bits or none is", i);
  if (t.master && t.param_type == FBFFTCONV_FLOAT32)
    return op_fail(FBFFTCONV_ERR_INVALID_ARGUMENT, "tensor %d: fp32 parameters have no fp32 master", i);
  if (t.count == 0) return FBFFTCONV_OK;
  if (!t.param || !t.grad || !t.moment1 || !t.moment2)
    return op_fail(FBFFTCONV_ERR_INVALID_ARGUMENT, "tensor %d: null pointer", i);
  const int moment_bytes = t.scale1 ? 1 : 4;
  if (!aligned_to(t.param, type_bytes(t.param_type)) || !aligned_to(t.grad, type_bytes(t.grad_type)) ||
      !aligned_to(t.master, 4) || !aligned_to(t.moment1, moment_bytes) || !aligned_to(t.moment2, moment_bytes) ||
      !aligned_to(t.scale1, 4) || !aligned_to(t.scale2, 4))
    return op_fail(FBFFTCONV_ERR_INVALID_ARGUMENT, "tensor %d: a pointer is not aligned to its element", i);
  return FBFFTCONV_OK;
}

int check_pointers(const fbfftconv_adamw_tensor& t, int device) {
  if (t.count == 0) return FBFFTCONV_OK;
  const struct { const void* p; const char* name; } all[] = {
      {t.param, "a parameter"}, {t.master, "a master weight"}, {t.grad, "a gradient"}, {t.moment1, "a first moment"},
      {t.moment2, "a second moment"}, {t.scale1, "a scale"}, {t.scale2, "a scale"}};
  for (const auto& a : all) OP_TRY(validate_device_pointer(device, a.p, a.name));
  return FBFFTCONV_OK;
}

// What a step writes must not be written twice, nor read as a gradient: a parameter that is listed twice would be updated
// by two warps at once, and a gradient that lies in one be read before or after its update.
int check_overlap(const fbfftconv_adamw_tensor* tensors, int count, const fbfftconv_adamw_options& options) {
  std::vector<std::pair<uintptr_t, uintptr_t>> written;
  const auto add = [&](const void* p, long long bytes) {
    if (p && bytes) written.emplace_back((uintptr_t)p, (uintptr_t)p + (uintptr_t)bytes);
  };
  for (int i = 0; i < count; ++i) {
    const fbfftconv_adamw_tensor& t = tensors[i];
    const int moment_bytes = t.scale1 ? 1 : 4;
    add(t.param, t.count * type_bytes(t.param_type));
    add(t.master, t.count * 4);
    add(t.moment1, t.count * moment_bytes);
    add(t.moment2, t.count * moment_bytes);
    add(t.scale1, 4ll * blocks_of(t.count));
    add(t.scale2, 4ll * blocks_of(t.count));
  }
  add(options.steps, 2 * sizeof(int64_t));
  std::sort(written.begin(), written.end());
  for (size_t i = 1; i < written.size(); ++i)
    if (written[i].first < written[i - 1].second)
      return op_fail(FBFFTCONV_ERR_INVALID_ARGUMENT, "parameters, masters, moments and steps must not share memory");
  for (int i = 0; i < count; ++i) {
    const uintptr_t begin = (uintptr_t)tensors[i].grad;
    const uintptr_t end = begin + (uintptr_t)(tensors[i].count * type_bytes(tensors[i].grad_type));
    if (begin == end) continue;
    const auto next = std::lower_bound(written.begin(), written.end(), std::make_pair(end, (uintptr_t)0));
    if (next != written.begin() && (next - 1)->second > begin)  // the last one that begins before the gradient's end
      return op_fail(FBFFTCONV_ERR_INVALID_ARGUMENT, "gradient %d must not share memory with what a step writes", i);
  }
  return FBFFTCONV_OK;
}

int create(const fbfftconv_adamw_tensor* tensors, int count, const fbfftconv_adamw_options* options, fbfftconv_adamw** out) {
  if (!out) return op_fail(FBFFTCONV_ERR_INVALID_ARGUMENT, "null argument");
  *out = nullptr;
  if (!options || count < 0 || (count && !tensors)) return op_fail(FBFFTCONV_ERR_INVALID_ARGUMENT, "null argument");
  const fbfftconv_adamw_options& o = *options;
  if (!(o.beta1 >= 0 && o.beta1 < 1) || !(o.beta2 >= 0 && o.beta2 < 1))
    return op_fail(FBFFTCONV_ERR_INVALID_ARGUMENT, "the betas must be in [0, 1)");
  if (!(o.eps >= 0) || !isfinite(o.eps))
    return op_fail(FBFFTCONV_ERR_INVALID_ARGUMENT, "eps must be finite and not negative");
  if (!(o.weight_decay >= 0) || !isfinite(o.weight_decay))
    return op_fail(FBFFTCONV_ERR_INVALID_ARGUMENT, "the weight decay must be finite and not negative");
  if (!o.steps || !aligned_to(o.steps, 8))
    return op_fail(FBFFTCONV_ERR_INVALID_ARGUMENT, "steps must name two 8-byte integers");
  for (int i = 0; i < count; ++i) OP_TRY(check_tensor(tensors[i], i));
  OP_TRY(check_overlap(tensors, count, o));
  std::unique_ptr<fbfftconv_adamw> h(new fbfftconv_adamw);
  h->tensors.assign(tensors, tensors + count);
  h->options = o;
  OP_TRY(resolve_device(o.device, &h->device));
  OP_TRY(validate_device_pointer(h->device, o.steps, "steps"));
  for (const auto& t : h->tensors) OP_TRY(check_pointers(t, h->device));
  *out = h.release();
  return FBFFTCONV_OK;
}

int set_gradients(fbfftconv_adamw* h, const void* const* grads, int count) {
  if (!h || count != (int)h->tensors.size() || (count && !grads))
    return op_fail(FBFFTCONV_ERR_INVALID_ARGUMENT, "one gradient for each tensor");
  std::vector<fbfftconv_adamw_tensor> tensors = h->tensors;
  for (int i = 0; i < count; ++i) {
    if (tensors[i].count == 0) continue;
    if (!grads[i] || !aligned_to(grads[i], type_bytes(tensors[i].grad_type)))
      return op_fail(FBFFTCONV_ERR_INVALID_ARGUMENT, "gradient %d is null or not aligned to its element", i);
    OP_TRY(validate_device_pointer(h->device, grads[i], "a gradient"));
    tensors[i].grad = grads[i];
  }
  OP_TRY(check_overlap(tensors.data(), count, h->options));
  h->tensors.swap(tensors);
  return FBFFTCONV_OK;
}

int step(fbfftconv_adamw* h, double lr, float grad_scale, const float* scalars, cudaStream_t stream) {
  if (!h) return op_fail(FBFFTCONV_ERR_INVALID_ARGUMENT, "null handle");
  if (!scalars && !(isfinite(lr) && isfinite(grad_scale)))
    return op_fail(FBFFTCONV_ERR_INVALID_ARGUMENT, "the learning rate and the gradient scale must be finite");
  if (!aligned_to(scalars, 4)) return op_fail(FBFFTCONV_ERR_INVALID_ARGUMENT, "scalars are not aligned");
  OP_TRY(validate_device_pointer(h->device, scalars, "scalars"));
  const OnDevice on(h->device);
  if (on.error() != cudaSuccess) return op_cuda_fail(on.error(), "cudaSetDevice");
  const fbfftconv_adamw_options& o = h->options;
  Common c{};
  c.beta1 = (float)o.beta1, c.beta2 = (float)o.beta2, c.rest1 = (float)(1 - o.beta1), c.rest2 = (float)(1 - o.beta2);
  c.log_beta1 = (float)log(o.beta1), c.log_beta2 = (float)log(o.beta2), c.eps = (float)o.eps;
  c.lr = (float)lr, c.weight_decay = (float)o.weight_decay, c.grad_scale = grad_scale, c.scalars = scalars;
  c.steps = reinterpret_cast<long long*>(o.steps), c.seed = o.seed;
  int chosen[kMany], n = 0;
  long long blocks = 0;
  const int total = (int)h->tensors.size();
  for (int i = 0; i <= total; ++i) {
    const long long more = i < total ? blocks_of(h->tensors[i].count) : 0;
    if (i == total || n == kMany || blocks + more > kMostBlocks) {
      c.advance = i == total;
      const cudaError_t e = n <= kFew    ? launch<kFew>(h, chosen, n, c, stream)
                            : n <= kSome ? launch<kSome>(h, chosen, n, c, stream)
                                         : launch<kMany>(h, chosen, n, c, stream);
      if (e != cudaSuccess) return op_cuda_fail(e, "adamw");
      n = 0, blocks = 0;
    }
    if (more) chosen[n++] = i, blocks += more;
  }
  return FBFFTCONV_OK;
}

}  // namespace
}  // namespace fbfft

using namespace fbfft;

extern "C" {

int fbfftconv_adamw_create(const fbfftconv_adamw_tensor* tensors, int count, const fbfftconv_adamw_options* options,
                           fbfftconv_adamw** out) {
  try {
    return create(tensors, count, options, out);
  } catch (const std::bad_alloc&) {
    return op_fail(FBFFTCONV_ERR_NOMEM, "out of host memory");
  }
}

int fbfftconv_adamw_destroy(fbfftconv_adamw* h) {
  delete h;
  return FBFFTCONV_OK;
}

int fbfftconv_adamw_set_gradients(fbfftconv_adamw* h, const void* const* grads, int count) {
  try {
    return set_gradients(h, grads, count);
  } catch (const std::bad_alloc&) {
    return op_fail(FBFFTCONV_ERR_NOMEM, "out of host memory");
  }
}

int fbfftconv_adamw_step(fbfftconv_adamw* h, double lr, float grad_scale, const float* scalars, fbfftconv_stream stream) {
  return step(h, lr, grad_scale, scalars, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
