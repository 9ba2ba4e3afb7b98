// wide_deep_amd/csrc/adamw.hip -- one AdamW step over many tensors, moments in 32 or in 8 bits.
//
// Elementwise over every parameter, so HBM bounds it: 28 bytes a parameter with 32-bit moments (p, m, v in and out, g in), 16 with 8-bit
// ones and fp32 gradients.  One launch walks a table of 2048-element chunks of all tensors; clipping adds one pass over the gradients.
#include "common.h"

namespace {

using namespace wd;

constexpr int TH = 256, U = WD_ADAMW_CHUNK / (4 * TH);      // a chunk = 256 lanes x U vectors of 4 elements
static_assert(TH * U * 4 == WD_ADAMW_CHUNK, "chunk");
constexpr int kTickets = 32, kTicketStride = 32;      // counters a cache line apart, and the one they meet in
static_assert((1 + kTickets) * kTicketStride == WD_ADAMW_TICKETS, "tickets");
constexpr int kGroup = WD_ADAMW_BLOCK / 4;          // lanes that share a scale

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ f32x4 unpack4(u32x2 w, int dtype) {
  if (dtype == WD_T_BF16) return {__uint_as_float(w[0] << 16), __uint_as_float(w[0] & 0xffff0000u), __uint_as_float(w[1] << 16), __uint_as_float(w[1] & 0xffff0000u)};
  const uint32_t lo = w[0], hi = w[1];      // a bit cast of the vector's element itself reads element 0
  const f32x2 a = __builtin_convertvector(__builtin_bit_cast(f16x2, lo), f32x2), b = __builtin_convertvector(__builtin_bit_cast(f16x2, hi), f32x2);
  return {a[0], a[1], b[0], b[1]};
}
__device__ __forceinline__ u32x2 pack4(f32x4 x, int dtype) {
  const f32x2 a = {x[0], x[1]}, b = {x[2], x[3]};
  if (dtype == WD_T_BF16)
    return {__builtin_bit_cast(uint32_t, __builtin_convertvector(a, bf16x2)), __builtin_bit_cast(uint32_t, __builtin_convertvector(b, bf16x2))};
  return {__builtin_bit_cast(uint32_t, __builtin_convertvector(a, f16x2)), __builtin_bit_cast(uint32_t, __builtin_convertvector(b, f16x2))};
}

// tensors' pointers come out of a table: said to be global memory, or every access would be a flat one that waits for LDS too
template <typename T> using Global = __attribute__((address_space(1))) T;
template <typename T> __device__ __forceinline__ Global<T> *global(const void *p) { return (Global<T> *)(uintptr_t)p; }
template <typename T> __device__ __forceinline__ T load_nt(const void *p) { return __builtin_nontemporal_load(global<T>(p)); }
template <typename T> __device__ __forceinline__ void store_nt(void *p, T v) { __builtin_nontemporal_store(v, global<T>(p)); }

// elements l .. l + 3 of a chunk; vec: in one access of 16 or 8 bytes, nontemporal (no stream of a step is read twice)
template <int T> __device__ __forceinline__ f32x4 load4(const void *p, int l, int left, bool vec) {
  if (vec) {
    if (T == WD_T_F32) return load_nt<f32x4>((const float *)p + l);
    return unpack4(load_nt<u32x2>((const uint16_t *)p + l), T);
  }
  f32x4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (l + k < left) {
      if (T == WD_T_F32) x[k] = global<float>(p)[l + k];
      else if (T == WD_T_BF16) x[k] = __uint_as_float((uint32_t)global<uint16_t>(p)[l + k] << 16);
      else x[k] = (float)global<_Float16>(p)[l + k];
    }
  return x;
}

// chunk c: where its elements are, and how many
struct Chunk {
  float *p;
  const char *g;
  uint16_t *copy;
  int64_t flat;      // in the moment buffers
  float decay;
  int left;          // elements, at most WD_ADAMW_CHUNK
};
template <int GT> __device__ __forceinline__ Chunk chunk_of(const wd_adamw_tensor_t *__restrict__ tensors, const int32_t *__restrict__ chunks, int64_t c) {
  const wd_adamw_tensor_t t = tensors[chunks[2 * c]];
  const int64_t e = (int64_t)chunks[2 * c + 1] * WD_ADAMW_CHUNK;
  Chunk x;
  x.p = t.p + e;
  x.g = (const char *)t.g + e * (GT == WD_T_F32 ? 4 : 2);
  x.copy = t.copy ? (uint16_t *)t.copy + e : nullptr;
  x.flat = t.start + e;
  x.decay = t.decay;
  x.left = (int)min(t.n - e, (int64_t)WD_ADAMW_CHUNK);
  return x;
}
// a full chunk, everything aligned for vectors
__device__ __forceinline__ bool whole(const Chunk &x) {
  return x.left == WD_ADAMW_CHUNK && (((uintptr_t)x.p | (uintptr_t)x.g | (uintptr_t)x.copy) & 15) == 0;
}

// largest of the 16 lanes of a block, in all of them: four rotations within the row of lanes
__device__ __forceinline__ uint32_t group_max(uint32_t v) {
  static_assert(kGroup == 16, "a block is a row of lanes");
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x128, 0xf, 0xf, false));
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x124, 0xf, 0xf, false));
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x122, 0xf, 0xf, false));
  return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x121, 0xf, 0xf, false));
}

// ---- 8-bit numbers: 4 exponent bits, M mantissa bits.  y = |x| 2^(142 - s) puts the block's largest value into [2^15, 2^16); scaled
// down by 2^127 the code is the exponent and the top M mantissa bits of an IEEE number -- its subnormals are the code's --, so
// rounding is an integer addition below the cut and one shift.
template <int M> __device__ __forceinline__ uint32_t encode(float x, int32_t s, uint32_t dither) {      // dither: 23 - M bits
  const uint32_t c = (__float_as_uint(ldexpf(fabsf(x), 15 - s)) + dither) >> (23 - M);                // 142 - 127
  return min(c, (16u << M) - 1u);
}
// byte k of w; `nan`: the block's nan_bits
__device__ __forceinline__ float decode_m(uint32_t w, int k, int32_t s, uint32_t nan) {
  const uint32_t t = w << (24 - 8 * k);      // sign and code on top
  return __uint_as_float(__float_as_uint(ldexpf(__uint_as_float((t & 0x80000000u) | ((t >> 4) & 0x07f00000u)), s - 15)) | nan);
}
__device__ __forceinline__ float decode_r(uint32_t w, int k, int32_t s, uint32_t nan) {
  return __uint_as_float(__float_as_uint(ldexpf(__uint_as_float(((w >> (8 * k)) & 255u) << 19), s - 15)) | nan);
}
// The root that a step goes on from: code 0 counts as code 1.  A root far below its block's largest may be stored as 0 while m keeps a code;
// m / eps would be the next update (one element in 64 with gradients 10^6 times its neighbours': steps of 10^5 lr).  Code 1 is 2^-18 to 2^-19
// of the block's largest, and m's code 1 is of that size of its own: a few lr at most (4.5 there).  In a block of zeros code 1 squared is 0.
// 200 M parameters 534.5 -> 537 us, 3 M 10.67 -> 10.73.
__device__ __forceinline__ float decode_root(uint32_t w, int k, int32_t s, uint32_t nan) {
  return __uint_as_float(__float_as_uint(ldexpf(__uint_as_float(max((w >> (8 * k)) & 255u, 1u) << 19), s - 15)) | nan);
}
__device__ __forceinline__ uint32_t nan_bits(int32_t s) { return s == 255 ? 0x7fc00000u : 0u; }
// scale byte of a block from the bits of its lanes' largest |x| (integers order as the numbers do, NaN above all)
__device__ __forceinline__ int32_t scale_of(uint32_t top) { return min(max((int32_t)(group_max(top) >> 23), 27), 255); }
__device__ __forceinline__ uint32_t top4(f32x4 x) {
  uint32_t t = 0;
#pragma unroll
  for (int k = 0; k < 4; ++k) t = max(t, __float_as_uint(x[k]) & 0x7fffffffu);
  return t;
}

// sqrt(v) to half a step and a bit: the reciprocal root and one Newton step, a third of the instructions of the correctly rounded one
// (below 2^-126, where the square of a gradient is not a normal number any more, it falls faster than the root; 0 stays 0)
__device__ __forceinline__ float root_of(float v) {
  const float y = __builtin_amdgcn_rsqf(fmaxf(v, 1.17549435e-38f)), r = v * y;
  return v == v ? fmaf(fmaf(-r, r, v), 0.5f * y, r) : v;
}

// 32 random bits of ((index ^ seed) + step 0x9E3779B1 + high word 0xBB67AE85): two multiply-xorshift rounds; the multipliers are the leading
// 32 bits of the fractions of (sqrt(5) - 1) / 2, sqrt(3) and sqrt(2), all odd
__device__ __forceinline__ uint32_t hash32(uint32_t h) {
  h = (h ^ (h >> 16)) * 0xBB67AE85u;
  h = (h ^ (h >> 15)) * 0x6A09E667u;
  return h ^ (h >> 16);
}

__device__ __forceinline__ double block_sum(double v, double *lds) {
#pragma unroll
  for (int o = 1; o < kWave; o <<= 1) v += __shfl_xor(v, o);
  if ((threadIdx.x & (kWave - 1)) == 0) lds[threadIdx.x / kWave] = v;
  __syncthreads();
  double t = lds[0];
#pragma unroll
  for (int w = 1; w < TH / kWave; ++w) t += lds[w];
  return t;
}

// partials[b] = sum of squares of workgroup b's chunks.  A chunk is 4 or 8 KB and a chain of three loads, so several are under way, and the
// next ones' places with them: fp32 480 MB 84 us = 5.7 TB/s
template <int GT> __global__ void __launch_bounds__(TH)
k_grad_square(const wd_adamw_tensor_t *__restrict__ tensors, const int32_t *__restrict__ chunks, int64_t nchunks, double *__restrict__ partials) {
  constexpr int L = GT == WD_T_F32 ? 4 : 8, N = WD_ADAMW_CHUNK / TH / L, C = 4 / N;      // N loads of 16 bytes a chunk, C chunks
  __shared__ double lds[TH / kWave];
  double total = 0.0;
  const int64_t last = nchunks - 1;
  Chunk x[C], y[C];
#pragma unroll
  for (int c = 0; c < C; ++c) x[c] = chunk_of<GT>(tensors, chunks, min(blockIdx.x + (int64_t)c * gridDim.x, last));
  for (int64_t c0 = blockIdx.x; c0 <= last; c0 += (int64_t)gridDim.x * C) {
    f32x4 w[C][N];
    bool full[C];
#pragma unroll
    for (int c = 0; c < C; ++c) {
      full[c] = c0 + (int64_t)c * gridDim.x <= last && ((uintptr_t)x[c].g & 15) == 0 && x[c].left == WD_ADAMW_CHUNK;
#pragma unroll
      for (int u = 0; u < N; ++u) {
        w[c][u] = {0.f, 0.f, 0.f, 0.f};
        if (full[c]) w[c][u] = global<f32x4>(x[c].g)[u * TH + threadIdx.x];
      }
    }
#pragma unroll
    for (int c = 0; c < C; ++c) y[c] = chunk_of<GT>(tensors, chunks, min(c0 + (int64_t)(C + c) * gridDim.x, last));
#pragma unroll
    for (int c = 0; c < C; ++c) {
      float s = 0.f;      // 8 squares in fp32 (finite up to sqrt(2^128 / 8) = 6.5e18 each), then 64 bits
#pragma unroll
      for (int u = 0; u < N; ++u)
#pragma unroll
        for (int h = 0; h < L / 4; ++h) {
          f32x4 g = w[c][u];
          if (GT != WD_T_F32) {
            const float lo = w[c][u][2 * h], hi = w[c][u][(2 * h + 1) & 3];
            const u32x2 half = {__float_as_uint(lo), __float_as_uint(hi)};
            g = unpack4(half, GT);
          }
#pragma unroll
          for (int k = 0; k < 4; ++k) s = fmaf(g[k], g[k], s);
        }
      if (!full[c] && c0 + (int64_t)c * gridDim.x <= last)      // a tensor's end, or one that starts anywhere
#pragma unroll 1
        for (int u = 0; u < U; ++u) {
          const f32x4 g = load4<GT>(x[c].g, (u * TH + threadIdx.x) * 4, x[c].left, false);
#pragma unroll
          for (int k = 0; k < 4; ++k) s = fmaf(g[k], g[k], s);
        }
      total += s;
      x[c] = y[c];
    }
  }
  total = block_sum(total, lds);
  if (threadIdx.x == 0) partials[blockIdx.x] = total;
}

// what a lane holds of a chunk, and the step's numbers
struct Piece {
  f32x4 p, g, m, v;
  uint32_t mc, rc;
  int32_t ms, rs;
};
struct Hyper {
  float lr, c1, c2, b1, n1, b2, n2, eps, coef;
  uint32_t step;
};

// WHOLE: no lane of the chunk has an element missing
template <int GT, int BITS, bool WHOLE> __device__ __forceinline__ void load_piece(Piece &x, const wd_adamw_t &o, const Chunk &t, int l) {
  x.p = load4<WD_T_F32>(t.p, l, t.left, WHOLE);
  x.g = load4<GT>(t.g, l, t.left, WHOLE);
  x.m = x.v = {0.f, 0.f, 0.f, 0.f};
  x.mc = x.rc = 0;
  x.ms = x.rs = 27;
  if (!WHOLE && l >= t.left) return;           // the flat moment buffers are padded to whole blocks
  if (BITS == 32) {
    x.m = load_nt<f32x4>((const float *)o.m + t.flat + l);
    x.v = load_nt<f32x4>((const float *)o.v + t.flat + l);
  } else {
    x.mc = load_nt<uint32_t>((const uint8_t *)o.m + t.flat + l);
    x.rc = load_nt<uint32_t>((const uint8_t *)o.v + t.flat + l);
    x.ms = o.m_scale[t.flat / WD_ADAMW_BLOCK + l / WD_ADAMW_BLOCK];
    x.rs = o.r_scale[t.flat / WD_ADAMW_BLOCK + l / WD_ADAMW_BLOCK];
  }
}
template <int BITS, bool WHOLE> __device__ __forceinline__ void update_piece(Piece &x, const wd_adamw_t &o, const Hyper &h, const Chunk &t, int l) {
  f32x4 r;
  const uint32_t nm = BITS == 8 ? nan_bits(x.ms) : 0, nr = BITS == 8 ? nan_bits(x.rs) : 0;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float gk = x.g[k] * h.coef;
    if (BITS == 32) {
      x.m[k] = fmaf(h.b1, x.m[k], h.n1 * gk);
      x.v[k] = fmaf(h.b2, x.v[k], h.n2 * (gk * gk));
      x.p[k] -= h.lr * (x.m[k] * h.c1 / (sqrtf(x.v[k]) * h.c2 + h.eps) + t.decay * x.p[k]);
    } else {           // instructions count here: roots and reciprocals to one unit of the last place; rk * rk is exact (5 bits)
      const float rk = decode_root(x.rc, k, x.rs, nr);
      x.m[k] = fmaf(h.b1, decode_m(x.mc, k, x.ms, nm), h.n1 * gk);
      r[k] = root_of(fmaf(h.b2, rk * rk, h.n2 * gk * gk));
      x.p[k] -= h.lr * (x.m[k] * h.c1 * __builtin_amdgcn_rcpf(r[k] * h.c2 + h.eps) + t.decay * x.p[k]);
    }
  }
  if (BITS == 8) {           // every lane: the scale is a maximum over 16 lanes
    if (!WHOLE) {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (l + k >= t.left) x.m[k] = r[k] = 0.f;
    }
    const int32_t sm = scale_of(top4(x.m)), sr = scale_of(top4(r));
    const int64_t f = t.flat + l;
    const uint32_t lo = (uint32_t)f ^ o.seed, hi = h.step + (uint32_t)(f >> 32) * 0xBB67AE85u;
    uint32_t a = 0, b = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t d = hash32((lo ^ k) + hi);      // f is a multiple of 4
      a |= (encode<3>(x.m[k], sm, (d >> 12) & 0xffff0u) | ((__float_as_uint(x.m[k]) >> 24) & 128u)) << (8 * k);
      b |= encode<4>(r[k], sr, (d & 0xffffu) << 3) << (8 * k);
    }
    if (WHOLE || l < t.left) {
      store_nt<uint32_t>((uint8_t *)o.m + t.flat + l, a);
      store_nt<uint32_t>((uint8_t *)o.v + t.flat + l, b);
      if ((threadIdx.x & (kGroup - 1)) == 0) {
        o.m_scale[t.flat / WD_ADAMW_BLOCK + l / WD_ADAMW_BLOCK] = (uint8_t)sm;
        o.r_scale[t.flat / WD_ADAMW_BLOCK + l / WD_ADAMW_BLOCK] = (uint8_t)sr;
      }
    }
  } else if (WHOLE || l < t.left) {
    store_nt<f32x4>((float *)o.m + t.flat + l, x.m);
    store_nt<f32x4>((float *)o.v + t.flat + l, x.v);
  }
  if (WHOLE) store_nt<f32x4>(t.p + l, x.p);
  else
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (l + k < t.left) global<float>(t.p)[l + k] = x.p[k];
  if (t.copy) {
    const u32x2 w = pack4(x.p, o.copy_dtype);
    if (WHOLE) store_nt<u32x2>(t.copy + l, w);
    else
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (l + k < t.left) global<uint16_t>(t.copy)[l + k] = (uint16_t)(w[k >> 1] >> (16 * (k & 1)));
  }
}
template <int GT, int BITS, bool WHOLE> __device__ __forceinline__ void load_chunk(Piece (&x)[U], const wd_adamw_t &o, const Chunk &t) {
#pragma unroll
  for (int u = 0; u < U; ++u) load_piece<GT, BITS, WHOLE>(x[u], o, t, (u * TH + threadIdx.x) * 4);
}
template <int BITS, bool WHOLE> __device__ __forceinline__ void update_chunk(Piece (&x)[U], const wd_adamw_t &o, const Hyper &h, const Chunk &t) {
#pragma unroll
  for (int u = 0; u < U; ++u) update_piece<BITS, WHOLE>(x[u], o, h, t, (u * TH + threadIdx.x) * 4);
}

template <int GT, int BITS> __global__ void __launch_bounds__(TH)
k_adamw(wd_adamw_t o, const wd_adamw_tensor_t *__restrict__ tensors, const int32_t *__restrict__ chunks, int32_t npart) {
  __shared__ double lds[TH / kWave];
  Hyper h;
  h.lr = o.lr_dev ? *o.lr_dev : o.lr;
  h.c1 = o.state->corr1;
  h.c2 = o.state->corr2;
  h.step = (uint32_t)(o.state->step + 1) * 0x9E3779B1u;
  h.b1 = (float)o.beta1, h.n1 = (float)(1.0 - o.beta1), h.b2 = (float)o.beta2, h.n2 = (float)(1.0 - o.beta2);   // 1 - 0.999f is 5e-5 off
  h.eps = o.eps;
  h.coef = 1.f;
  float norm = 0.f;
  bool skip = false;
  if (npart) {
    double s = 0.0;
    for (int i = threadIdx.x; i < npart; i += TH) s += o.partials[i];
    const double G = sqrt(block_sum(s, lds));
    norm = (float)G;
    skip = !(G < (double)INFINITY);
    h.coef = G > (double)o.max_norm ? (float)((double)o.max_norm / G) : 1.f;      // max_norm may be infinite: the norm is told, nothing clipped
  }
  // backwards: the norm's pass has left the ends of the gradients in the last cache
  int64_t c = o.nchunks - 1 - blockIdx.x;
  Chunk next = chunk_of<GT>(tensors, chunks, c);
  while (c >= 0 && !skip) {
    const Chunk t = next;
    Piece x[U];
    if (whole(t)) load_chunk<GT, BITS, true>(x, o, t);
    else load_chunk<GT, BITS, false>(x, o, t);
    c -= gridDim.x;
    next = chunk_of<GT>(tensors, chunks, max(c, (int64_t)0));
    if (whole(t)) update_chunk<BITS, true>(x, o, h, t);
    else update_chunk<BITS, false>(x, o, h, t);
  }
  // The last workgroup to get here moves the step: every other one has read the state.  Arrivals at one address queue up at about 10 ns
  // each (1465 workgroups on one counter: 23 us instead of 17 for 3 million parameters), so they meet in 32 counters first.
  __syncthreads();
  if (threadIdx.x) return;
  auto arrive = [](int32_t *p) { return __hip_atomic_fetch_add(p, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); };
  const int k = blockIdx.x % kTickets, groups = min((int)gridDim.x, kTickets);
  int32_t *mine = o.tickets + (1 + k) * kTicketStride;
  if (arrive(mine) != ((int)gridDim.x - k + kTickets - 1) / kTickets - 1) return;
  *mine = 0;
  if (arrive(o.tickets) != groups - 1) return;
  *o.tickets = 0;
  o.state->norm = norm;
  if (skip) {
    o.state->skipped += 1;
    return;
  }
  o.state->step += 1;
  const double p1 = o.state->pow1 *= o.beta1, p2 = o.state->pow2 *= o.beta2;
  o.state->corr1 = (float)(1.0 / (1.0 - p1));
  o.state->corr2 = (float)(1.0 / sqrt(1.0 - p2));
}

__global__ void k_adamw_set_step(wd_adamw_state_t *s, int32_t *tickets, int64_t step, double beta1, double beta2) {
  for (int i = threadIdx.x; i < WD_ADAMW_TICKETS; i += blockDim.x) tickets[i] = 0;
  if (threadIdx.x) return;
  const double t = (double)step + 1.0;
  s->step = step;
  s->skipped = 0;
  s->pow1 = pow(beta1, t);
  s->pow2 = pow(beta2, t);
  s->corr1 = (float)(1.0 / (1.0 - s->pow1));
  s->corr2 = (float)(1.0 / sqrt(1.0 - s->pow2));
  s->norm = 0.f;
}

// eight values a lane: 16-byte stores of bf16
template <int OT> __device__ __forceinline__ void put8(void *out, int64_t i, f32x4 x, f32x4 y) {
  if (OT == WD_T_F32) {
    store_nt<f32x4>((float *)out + i, x);
    store_nt<f32x4>((float *)out + i + 4, y);
  } else {
    const u32x2 a = pack4(x, OT), b = pack4(y, OT);
    const u32x4 w = {a[0], a[1], b[0], b[1]};
    store_nt<u32x4>((uint16_t *)out + i, w);
  }
}
template <int OT> __global__ void __launch_bounds__(TH)
k_adamw_unpack(const uint8_t *__restrict__ m, const uint8_t *__restrict__ m_scale, const uint8_t *__restrict__ r,
               const uint8_t *__restrict__ r_scale, int64_t n, void *__restrict__ out_m, void *__restrict__ out_r) {
  for (int64_t i = ((int64_t)blockIdx.x * TH + threadIdx.x) * 8; i < n; i += (int64_t)gridDim.x * TH * 8) {
    const u32x2 a = load_nt<u32x2>(m + i), b = load_nt<u32x2>(r + i);
    const int32_t sm = m_scale[i / WD_ADAMW_BLOCK], sr = r_scale[i / WD_ADAMW_BLOCK];
    f32x4 x[2], y[2];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      x[k / 4][k & 3] = decode_m(a[k / 4], k & 3, sm, nan_bits(sm));
      y[k / 4][k & 3] = decode_r(b[k / 4], k & 3, sr, nan_bits(sr));
    }
    put8<OT>(out_m, i, x[0], x[1]);
    put8<OT>(out_r, i, y[0], y[1]);
  }
}
__global__ void __launch_bounds__(TH)
k_adamw_pack(const float *__restrict__ in_m, const float *__restrict__ in_r, int64_t n, uint8_t *__restrict__ m,
             uint8_t *__restrict__ m_scale, uint8_t *__restrict__ r, uint8_t *__restrict__ r_scale) {
  const int64_t i = ((int64_t)blockIdx.x * TH + threadIdx.x) * 4;
  const f32x4 zero = {0.f, 0.f, 0.f, 0.f}, x = i < n ? *(const f32x4 *)(in_m + i) : zero, y = i < n ? *(const f32x4 *)(in_r + i) : zero;
  const int32_t sm = scale_of(top4(x)), sr = scale_of(top4(y));
  uint32_t a = 0, b = 0;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    a |= (encode<3>(x[k], sm, 0x80000u) | (__float_as_uint(x[k]) >> 31 << 7)) << (8 * k);
    b |= encode<4>(y[k], sr, 0x40000u) << (8 * k);
  }
  if (i >= n) return;
  *(uint32_t *)(m + i) = a;
  *(uint32_t *)(r + i) = b;
  if ((threadIdx.x & (kGroup - 1)) == 0) {
    m_scale[i / WD_ADAMW_BLOCK] = (uint8_t)sm;
    r_scale[i / WD_ADAMW_BLOCK] = (uint8_t)sr;
  }
}

template <int GT> void launch_adamw(const wd_adamw_t &o, hipStream_t st) {
  int npart = 0;
  if (o.max_norm > 0.f) {
    npart = (int)(o.nchunks < WD_ADAMW_PARTIALS ? o.nchunks : WD_ADAMW_PARTIALS);
    k_grad_square<GT><<<npart, TH, 0, st>>>(o.tensors, o.chunks, o.nchunks, o.partials);
  }
  // Workgroups: few parameters are a matter of latency and want all of the chip; many are a matter of how well HBM pages are used, and
  // fewer streams in flight read and write them better.  us a step, 1 / 2 / 4 workgroups on a CU, 32 bits: 1 M parameters 10.4 / 9.0 / 8.4,
  // 8 M 42.3 / 41.3 / 42.5, 64 M 302 / 329 / 338; 8 bits: 9.9 / 8.4 / 7.8, 39.6 / 27.9 / 27.0, 281 / 193 / 211
  const int64_t most = (o.nchunks <= 8192 ? 4 : o.bits == 32 ? 1 : 2) * kCUs;
  const int grid = (int)(o.nchunks < most ? o.nchunks : most);
  if (o.bits == 32) k_adamw<GT, 32><<<grid, TH, 0, st>>>(o, o.tensors, o.chunks, npart);
  else k_adamw<GT, 8><<<grid, TH, 0, st>>>(o, o.tensors, o.chunks, npart);
}

}  // namespace

extern "C" int wd_adamw_step(const wd_adamw_t *opts, wd_stream_t stream) {
  WD_REQUIRE(opts, "null argument");
  const wd_adamw_t o = *opts;
  WD_REQUIRE(o.tensors && o.chunks && o.m && o.v && o.state && o.tickets && o.nchunks > 0, "null pointer or no chunks");
  WD_REQUIRE(o.bits == 32 || o.bits == 8, "moments are kept in 32 or in 8 bits");
  WD_REQUIRE((((uintptr_t)o.m | (uintptr_t)o.v) & 15) == 0, "moments not aligned to 16 bytes");
  WD_REQUIRE(o.bits == 32 || (o.m_scale && o.r_scale), "8-bit moments need their scales");
  WD_REQUIRE(o.grad_dtype == WD_T_F32 || o.grad_dtype == WD_T_F16 || o.grad_dtype == WD_T_BF16, "bad gradient type");
  WD_REQUIRE(o.copy_dtype == WD_T_F16 || o.copy_dtype == WD_T_BF16, "the copy is fp16 or bf16");
  WD_REQUIRE(o.beta1 >= 0. && o.beta1 < 1. && o.beta2 >= 0. && o.beta2 < 1. && o.eps >= 0.f, "betas must be in [0, 1), eps >= 0");
  WD_REQUIRE(!(o.max_norm > 0.f) || o.partials, "clipping needs the partials buffer");
  hipStream_t st = as_stream(stream);
  if (o.grad_dtype == WD_T_F32) launch_adamw<WD_T_F32>(o, st);
  else if (o.grad_dtype == WD_T_F16) launch_adamw<WD_T_F16>(o, st);
  else launch_adamw<WD_T_BF16>(o, st);
  return check_launch(__func__);
}

extern "C" int wd_adamw_set_step(wd_adamw_state_t *state, int32_t *tickets, int64_t step, double beta1, double beta2, wd_stream_t stream) {
  WD_REQUIRE(state && tickets && step >= 0, "null pointer or negative step");
  WD_REQUIRE(beta1 >= 0. && beta1 < 1. && beta2 >= 0. && beta2 < 1., "betas must be in [0, 1)");
  k_adamw_set_step<<<1, 64, 0, as_stream(stream)>>>(state, tickets, step, beta1, beta2);
  return check_launch(__func__);
}

extern "C" int wd_adamw_unpack(const uint8_t *m, const uint8_t *m_scale, const uint8_t *r, const uint8_t *r_scale, int64_t n, void *out_m,
                               void *out_r, int32_t out_dtype, wd_stream_t stream) {
  WD_REQUIRE(m && m_scale && r && r_scale && out_m && out_r, "null pointer");
  WD_REQUIRE(n > 0 && n % WD_ADAMW_BLOCK == 0, "n must be a positive multiple of the block");
  WD_REQUIRE((((uintptr_t)m | (uintptr_t)r | (uintptr_t)out_m | (uintptr_t)out_r) & 15) == 0, "buffers not aligned to 16 bytes");
  WD_REQUIRE(out_dtype == WD_T_F32 || out_dtype == WD_T_BF16, "numbers come as bf16 or fp32");
  const int64_t blocks = ceil_div(n, TH * 8);
  const int grid = (int)(blocks < 8 * kCUs ? blocks : 8 * kCUs);
  if (out_dtype == WD_T_F32) k_adamw_unpack<WD_T_F32><<<grid, TH, 0, as_stream(stream)>>>(m, m_scale, r, r_scale, n, out_m, out_r);
  else k_adamw_unpack<WD_T_BF16><<<grid, TH, 0, as_stream(stream)>>>(m, m_scale, r, r_scale, n, out_m, out_r);
  return check_launch(__func__);
}

extern "C" int wd_adamw_pack(const float *in_m, const float *in_r, int64_t n, uint8_t *m, uint8_t *m_scale, uint8_t *r, uint8_t *r_scale,
                             wd_stream_t stream) {
  WD_REQUIRE(in_m && in_r && m && m_scale && r && r_scale, "null pointer");
  WD_REQUIRE(n > 0 && n % WD_ADAMW_BLOCK == 0, "n must be a positive multiple of the block");
  WD_REQUIRE((((uintptr_t)m | (uintptr_t)r | (uintptr_t)in_m | (uintptr_t)in_r) & 15) == 0, "buffers not aligned to 16 bytes");
  WD_REQUIRE(ceil_div(n, TH * 4) * TH < ((int64_t)1 << 32), "more than 2^34 values in one call");
  k_adamw_pack<<<(unsigned)ceil_div(n, TH * 4), TH, 0, as_stream(stream)>>>(in_m, in_r, n, m, m_scale, r, r_scale);
  return check_launch(__func__);
}
