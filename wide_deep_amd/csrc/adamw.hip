// wide_deep_amd/csrc/adamw.hip -- one AdamW step over many tensors, moments in 32 or in 8 bits.
//
// Elementwise over every parameter, so HBM bounds it: 28 bytes a parameter with 32-bit moments (p, m, v in and out, g in), 16 with 8-bit
// ones and fp32 gradients.  One launch walks a table of 4096-element chunks of all tensors; clipping adds one pass over the gradients.
#include "common.h"

namespace {

using namespace wd;

constexpr int TH = 256, U = 4;                      // a chunk = 256 lanes x 4 vectors of 4 elements
static_assert(TH * U * 4 == WD_ADAMW_CHUNK, "chunk");
constexpr int kGroup = WD_ADAMW_BLOCK / 4;          // lanes that share a scale

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
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

// four elements from i on, zeros from n on; `vec`: the tensor's pointers allow vectors
template <int GT> __device__ __forceinline__ f32x4 load4(const void *p, int64_t i, int64_t n, bool vec) {
  if (vec && i + 4 <= n) {
    if (GT == WD_T_F32) return *(const f32x4 *)((const float *)p + i);
    return unpack4(*(const u32x2 *)((const uint16_t *)p + i), GT);
  }
  f32x4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (i + k < n) {
      if (GT == WD_T_F32) x[k] = ((const float *)p)[i + k];
      else if (GT == WD_T_BF16) x[k] = __uint_as_float((uint32_t)((const uint16_t *)p)[i + k] << 16);
      else x[k] = (float)((const _Float16 *)p)[i + k];
    }
  return x;
}

template <typename T> __device__ __forceinline__ T group_max(T v) {      // over the 16 lanes of a block
#pragma unroll
  for (int o = 1; o < kGroup; o <<= 1) v = max(v, __shfl_xor(v, o));
  return v;
}

// ---- 8-bit numbers: 4 exponent bits, M mantissa bits.  y = |x| 2^(142 - s) puts the block's largest value into [2^15, 2^16); scaled
// down by 2^127 the code is the exponent and the top M mantissa bits of an IEEE number -- its subnormals are the code's --, so
// rounding is an integer addition below the cut and one shift.
template <int M> __device__ __forceinline__ uint32_t encode(float x, int32_t s, uint32_t dither16) {
  const uint32_t b = __float_as_uint(ldexpf(fabsf(x), 15 - s));          // 142 - 127
  const uint32_t c = (b + (dither16 << (23 - M - 16))) >> (23 - M);
  return min(c, (16u << M) - 1u);
}
template <int M> __device__ __forceinline__ float decode(uint32_t code, int32_t s) {
  return s == 255 ? __uint_as_float(0x7fc00000u) : ldexpf(__uint_as_float(code << (23 - M)), s - 15);
}
// scale byte of a block from the bits of its lanes' largest |x| (integers order as the numbers do, NaN above all)
__device__ __forceinline__ int32_t scale_of(uint32_t top) { return min(max((int32_t)(group_max(top) >> 23), 27), 255); }
__device__ __forceinline__ uint32_t top4(f32x4 x) {
  uint32_t t = 0;
#pragma unroll
  for (int k = 0; k < 4; ++k) t = max(t, __float_as_uint(x[k]) & 0x7fffffffu);
  return t;
}

// 32 random bits of (index, step, seed): two multiply-xorshift rounds; the multipliers are the leading 32 bits of the fractions of
// (sqrt(5) - 1) / 2, sqrt(3) and sqrt(2), all odd
__device__ __forceinline__ uint32_t hash32(int64_t i, uint32_t step, uint32_t seed) {
  uint32_t h = ((uint32_t)i ^ seed) + step * 0x9E3779B1u + (uint32_t)(i >> 32) * 0xBB67AE85u;
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

// partials[b] = sum of squares of workgroup b's chunks
template <int GT> __global__ void __launch_bounds__(TH) k_grad_square(wd_adamw_t o) {
  __shared__ double lds[TH / kWave];
  double total = 0.0;
  for (int64_t c = blockIdx.x; c < o.nchunks; c += gridDim.x) {
    const wd_adamw_tensor_t t = o.tensors[o.chunks[2 * c]];
    const int64_t e0 = (int64_t)o.chunks[2 * c + 1] * WD_ADAMW_CHUNK + threadIdx.x * 4;
    const bool vec = ((uintptr_t)t.g & (GT == WD_T_F32 ? 15 : 7)) == 0;
    float s = 0.f;
    f32x4 g[U];
#pragma unroll
    for (int u = 0; u < U; ++u) g[u] = load4<GT>(t.g, e0 + u * TH * 4, t.n, vec);
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int k = 0; k < 4; ++k) s = fmaf(g[u][k], g[u][k], s);
    total += s;      // 16 squares in fp32, then 64 bits
  }
  total = block_sum(total, lds);
  if (threadIdx.x == 0) o.partials[blockIdx.x] = total;
}

template <int GT, int BITS> __global__ void __launch_bounds__(TH) k_adamw(wd_adamw_t o, int32_t npart) {
  __shared__ double lds[TH / kWave];
  const float lr = o.lr_dev ? *o.lr_dev : o.lr;
  const float c1 = o.state->corr1, c2 = o.state->corr2;
  const uint32_t step = (uint32_t)(o.state->step + 1);
  const float b1 = (float)o.beta1, n1 = (float)(1.0 - o.beta1), b2 = (float)o.beta2, n2 = (float)(1.0 - o.beta2);   // 1 - 0.999f is 5e-5 off
  float coef = 1.f, norm = 0.f;
  bool skip = false;
  if (npart) {
    double s = 0.0;
    for (int i = threadIdx.x; i < npart; i += TH) s += o.partials[i];
    const double G = sqrt(block_sum(s, lds));
    norm = (float)G;
    skip = !(G < (double)INFINITY);
    coef = (float)((double)o.max_norm / fmax(G, (double)o.max_norm));
  }
  if (!skip)
    for (int64_t c = blockIdx.x; c < o.nchunks; c += gridDim.x) {
      const wd_adamw_tensor_t t = o.tensors[o.chunks[2 * c]];
      const int64_t e0 = (int64_t)o.chunks[2 * c + 1] * WD_ADAMW_CHUNK + threadIdx.x * 4;
      const bool vp = ((uintptr_t)t.p & 15) == 0, vg = ((uintptr_t)t.g & (GT == WD_T_F32 ? 15 : 7)) == 0;
      f32x4 p[U], g[U], m[U], v[U];
      uint32_t mc[U], rc[U];
      int32_t ms[U], rs[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int64_t e = e0 + u * TH * 4, f = t.start + e;
        p[u] = load4<WD_T_F32>(t.p, e, t.n, vp);
        g[u] = load4<GT>(t.g, e, t.n, vg);
        if (e < t.n) {           // the flat moment buffers are padded to whole blocks
          if (BITS == 32) {
            m[u] = *(const f32x4 *)((const float *)o.m + f);
            v[u] = *(const f32x4 *)((const float *)o.v + f);
          } else {
            mc[u] = *(const uint32_t *)((const uint8_t *)o.m + f);
            rc[u] = *(const uint32_t *)((const uint8_t *)o.v + f);
            ms[u] = o.m_scale[f / WD_ADAMW_BLOCK];
            rs[u] = o.r_scale[f / WD_ADAMW_BLOCK];
          }
        } else {
          m[u] = v[u] = {0.f, 0.f, 0.f, 0.f};
          mc[u] = rc[u] = 0;
          ms[u] = rs[u] = 27;
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int64_t e = e0 + u * TH * 4, f = t.start + e;
        f32x4 r;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          float mk, vk;
          if (BITS == 32) {
            mk = m[u][k];
            vk = v[u][k];
          } else {
            const uint32_t a = (mc[u] >> (8 * k)) & 255u, b = (rc[u] >> (8 * k)) & 255u;
            mk = copysignf(decode<3>(a & 127u, ms[u]), a & 128u ? -1.f : 1.f);
            const float rk = decode<4>(b, rs[u]);
            vk = rk * rk;
          }
          const float gk = g[u][k] * coef;
          mk = b1 * mk + n1 * gk;
          vk = b2 * vk + n2 * (gk * gk);
          const float root = sqrtf(vk);
          p[u][k] -= lr * (mk * c1 / (root * c2 + o.eps) + t.decay * p[u][k]);
          m[u][k] = mk;
          v[u][k] = vk;
          r[k] = root;
        }
        if (BITS == 8) {           // every lane: the scale is a maximum over 16 lanes
          if (e + 4 > t.n) {
#pragma unroll
            for (int k = 0; k < 4; ++k)
              if (e + k >= t.n) m[u][k] = r[k] = 0.f;
          }
          const int32_t sm = scale_of(top4(m[u])), sr = scale_of(top4(r));
          uint32_t a = 0, b = 0;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint32_t h = hash32(f + k, step, o.seed);
            a |= (encode<3>(m[u][k], sm, h >> 16) | (__float_as_uint(m[u][k]) >> 31 << 7)) << (8 * k);
            b |= encode<4>(r[k], sr, h & 0xffffu) << (8 * k);
          }
          if (e < t.n) {
            *(uint32_t *)((uint8_t *)o.m + f) = a;
            *(uint32_t *)((uint8_t *)o.v + f) = b;
            if ((threadIdx.x & (kGroup - 1)) == 0) {
              o.m_scale[f / WD_ADAMW_BLOCK] = (uint8_t)sm;
              o.r_scale[f / WD_ADAMW_BLOCK] = (uint8_t)sr;
            }
          }
        } else if (e < t.n) {
          *(f32x4 *)((float *)o.m + f) = m[u];
          *(f32x4 *)((float *)o.v + f) = v[u];
        }
        if (vp && e + 4 <= t.n) *(f32x4 *)(t.p + e) = p[u];
        else
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (e + k < t.n) t.p[e + k] = p[u][k];
        if (t.copy) {
          const u32x2 h = pack4(p[u], o.copy_dtype);
          if (((uintptr_t)t.copy & 7) == 0 && e + 4 <= t.n) *(u32x2 *)((uint16_t *)t.copy + e) = h;
          else
#pragma unroll
            for (int k = 0; k < 4; ++k)
              if (e + k < t.n) ((uint16_t *)t.copy)[e + k] = (uint16_t)(h[k >> 1] >> (16 * (k & 1)));
        }
      }
    }
  // the last workgroup to get here moves the step: every other one has read the state
  __syncthreads();
  if (threadIdx.x == 0 && __hip_atomic_fetch_add(&o.state->ticket, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (int32_t)gridDim.x - 1) {
    o.state->ticket = 0;
    o.state->norm = norm;
    if (skip) o.state->skipped += 1;
    else {
      const double t = (double)(o.state->step += 1) + 1.0;
      o.state->corr1 = (float)(1.0 / (1.0 - pow(o.beta1, t)));
      o.state->corr2 = (float)(1.0 / sqrt(1.0 - pow(o.beta2, t)));
    }
  }
}

__global__ void k_adamw_set_step(wd_adamw_state_t *s, int64_t step, double beta1, double beta2) {
  const double t = (double)step + 1.0;
  s->step = step;
  s->skipped = s->ticket = 0;
  s->corr1 = (float)(1.0 / (1.0 - pow(beta1, t)));
  s->corr2 = (float)(1.0 / sqrt(1.0 - pow(beta2, t)));
  s->norm = 0.f;
}

template <int OT> __device__ __forceinline__ void put4(void *out, int64_t i, f32x4 x) {
  if (OT == WD_T_F32) *(f32x4 *)((float *)out + i) = x;
  else *(u32x2 *)((uint16_t *)out + i) = pack4(x, OT);
}
template <int OT> __global__ void __launch_bounds__(TH)
k_adamw_unpack(const uint8_t *__restrict__ m, const uint8_t *__restrict__ m_scale, const uint8_t *__restrict__ r,
               const uint8_t *__restrict__ r_scale, int64_t n, void *__restrict__ out_m, void *__restrict__ out_r) {
  for (int64_t i = ((int64_t)blockIdx.x * TH + threadIdx.x) * 4; i < n; i += (int64_t)gridDim.x * TH * 4) {
    const uint32_t a = *(const uint32_t *)(m + i), b = *(const uint32_t *)(r + i);
    const int32_t sm = m_scale[i / WD_ADAMW_BLOCK], sr = r_scale[i / WD_ADAMW_BLOCK];
    f32x4 x, y;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t c = (a >> (8 * k)) & 255u;
      x[k] = copysignf(decode<3>(c & 127u, sm), c & 128u ? -1.f : 1.f);
      y[k] = decode<4>((b >> (8 * k)) & 255u, sr);
    }
    put4<OT>(out_m, i, x);
    put4<OT>(out_r, i, y);
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
    a |= (encode<3>(x[k], sm, 0x8000u) | (__float_as_uint(x[k]) >> 31 << 7)) << (8 * k);
    b |= encode<4>(y[k], sr, 0x8000u) << (8 * k);
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
    k_grad_square<GT><<<npart, TH, 0, st>>>(o);
  }
  const int grid = (int)(o.nchunks < 8 * kCUs ? o.nchunks : 8 * kCUs);
  if (o.bits == 32) k_adamw<GT, 32><<<grid, TH, 0, st>>>(o, npart);
  else k_adamw<GT, 8><<<grid, TH, 0, st>>>(o, npart);
}

}  // namespace

extern "C" int wd_adamw_step(const wd_adamw_t *opts, wd_stream_t stream) {
  WD_REQUIRE(opts, "null argument");
  const wd_adamw_t o = *opts;
  WD_REQUIRE(o.tensors && o.chunks && o.m && o.v && o.state && o.nchunks > 0, "null pointer or no chunks");
  WD_REQUIRE(o.bits == 32 || o.bits == 8, "moments are kept in 32 or in 8 bits");
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

extern "C" int wd_adamw_set_step(wd_adamw_state_t *state, int64_t step, double beta1, double beta2, wd_stream_t stream) {
  WD_REQUIRE(state && step >= 0, "null state or negative step");
  WD_REQUIRE(beta1 >= 0. && beta1 < 1. && beta2 >= 0. && beta2 < 1., "betas must be in [0, 1)");
  k_adamw_set_step<<<1, 1, 0, as_stream(stream)>>>(state, step, beta1, beta2);
  return check_launch(__func__);
}

extern "C" int wd_adamw_unpack(const uint8_t *m, const uint8_t *m_scale, const uint8_t *r, const uint8_t *r_scale, int64_t n, void *out_m,
                               void *out_r, int32_t out_dtype, wd_stream_t stream) {
  WD_REQUIRE(m && m_scale && r && r_scale && out_m && out_r, "null pointer");
  WD_REQUIRE(n > 0 && n % WD_ADAMW_BLOCK == 0, "n must be a positive multiple of the block");
  WD_REQUIRE(out_dtype == WD_T_F32 || out_dtype == WD_T_BF16, "numbers come as bf16 or fp32");
  const int64_t blocks = ceil_div(n, TH * 4);
  const int grid = (int)(blocks < 16 * kCUs ? blocks : 16 * kCUs);
  if (out_dtype == WD_T_F32) k_adamw_unpack<WD_T_F32><<<grid, TH, 0, as_stream(stream)>>>(m, m_scale, r, r_scale, n, out_m, out_r);
  else k_adamw_unpack<WD_T_BF16><<<grid, TH, 0, as_stream(stream)>>>(m, m_scale, r, r_scale, n, out_m, out_r);
  return check_launch(__func__);
}

extern "C" int wd_adamw_pack(const float *in_m, const float *in_r, int64_t n, uint8_t *m, uint8_t *m_scale, uint8_t *r, uint8_t *r_scale,
                             wd_stream_t stream) {
  WD_REQUIRE(in_m && in_r && m && m_scale && r && r_scale, "null pointer");
  WD_REQUIRE(n > 0 && n % WD_ADAMW_BLOCK == 0, "n must be a positive multiple of the block");
  WD_REQUIRE(ceil_div(n, TH * 4) * TH < ((int64_t)1 << 32), "more than 2^34 values in one call");
  k_adamw_pack<<<(unsigned)ceil_div(n, TH * 4), TH, 0, as_stream(stream)>>>(in_m, in_r, n, m, m_scale, r, r_scale);
  return check_launch(__func__);
}
