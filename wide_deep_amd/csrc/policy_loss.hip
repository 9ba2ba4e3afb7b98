// wide_deep_amd/csrc/policy_loss.hip -- heads of a policy over items: log-probabilities of the chosen items of ragged sequences,
// a preference loss over pairs of sequences and a clipped policy loss with a KL term, each with the gradient of the logits.
//
// Mathematics (rows r of logits z[r, 0..V), chosen item t[r], sequences = CSR over rows):
//   m = max_v z_v,  s = sum_v e^(z_v - m)                 one pass, running maximum and sum
//   lp = (z_t - m) - ln s                                 (not z_t - lse: the difference keeps its low bits where |m| is large)
//   dlp/dz_v = [v = t] - e^(z_v - m) / s,  dz_v = c * dlp/dz_v   with c = dloss/dlp of the row
// Everything a row needs from other rows is a handful of numbers, so the kernels are passes over rows and HBM bounds them.
#include <type_traits>

#include "common.h"

namespace {

using namespace wd;

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

constexpr float kLog2e = 1.44269504088896340736f;
// batches whose rows find their pair, weight or advantage themselves instead of in a launch of its own
constexpr int64_t kSelfRows = 256, kSelfSeqs = 256, kPairRows = 2048, kPairSeqs = 64, kWeightRows = 1024;
static_assert(kWeightRows <= kWave * kWave, "a lane for 64 rows");
constexpr int64_t kCountSeqs = 1024;      // up to as many sequences every wavefront adds the counts up itself
constexpr float kLowest = -3.402823466e38f;

// ---- element types: one 16-byte word <-> floats.  Sums and statistics are fp32; gradients are rounded once, to nearest even.
template <int DT> struct Elem;
template <> struct Elem<WD_T_F32> {
  typedef float type;
  static constexpr int W = 4;
  static __device__ __forceinline__ void unpack(const u32x4 &w, float *x) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = __uint_as_float(w[i]);
  }
  static __device__ __forceinline__ u32x4 pack(const float *x) {
    u32x4 w;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = __float_as_uint(x[i]);
    return w;
  }
  static __device__ __forceinline__ float to_float(float v) { return v; }
  static __device__ __forceinline__ float from_float(float v) { return v; }
};
template <> struct Elem<WD_T_BF16> {
  typedef uint16_t type;
  static constexpr int W = 8;
  static __device__ __forceinline__ void unpack(const u32x4 &w, float *x) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ u32x4 pack(const float *x) {
    u32x4 w;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const f32x2 p = {x[2 * i], x[2 * i + 1]};
      w[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(p, bf16x2));
    }
    return w;
  }
  static __device__ __forceinline__ float to_float(uint16_t v) { return __uint_as_float((uint32_t)v << 16); }
  static __device__ __forceinline__ uint16_t from_float(float v) { return __builtin_bit_cast(uint16_t, (__bf16)v); }
};
template <> struct Elem<WD_T_F16> {
  typedef uint16_t type;
  static constexpr int W = 8;
  static __device__ __forceinline__ void unpack(const u32x4 &w, float *x) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t v = w[i];      // a bit cast of the vector's element itself reads element 0
      const f32x2 p = __builtin_convertvector(__builtin_bit_cast(f16x2, v), f32x2);
      x[2 * i] = p[0];
      x[2 * i + 1] = p[1];
    }
  }
  static __device__ __forceinline__ u32x4 pack(const float *x) {
    u32x4 w;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const f32x2 p = {x[2 * i], x[2 * i + 1]};
      w[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(p, f16x2));
    }
    return w;
  }
  static __device__ __forceinline__ float to_float(uint16_t v) { return (float)__builtin_bit_cast(_Float16, v); }
  static __device__ __forceinline__ uint16_t from_float(float v) { return __builtin_bit_cast(uint16_t, (_Float16)v); }
};

// A row of odd length or stride starts anywhere: `head` elements up to the first 16-byte boundary, `nb` whole words, the rest.  The
// at most 2 (W - 1) elements outside the words are dealt one to a lane (`edge`), so nothing outside the row is ever touched.
template <int DT> struct Row {
  typedef typename Elem<DT>::type type;
  static constexpr int W = Elem<DT>::W;
  const type *p;
  int V, head, nb, rest;
  __device__ __forceinline__ Row(const void *base, int64_t ld, int64_t r, int vocab) {
    p = (const type *)base + r * ld;
    V = vocab;
    const int mis = (int)(((uintptr_t)p & 15) / sizeof(type));
    head = min((W - mis) & (W - 1), V);
    nb = (V - head) / W;
    rest = V - head - nb * W;
  }
  template <bool NT = false> __device__ __forceinline__ u32x4 word(int j) const {
    const u32x4 *q = (const u32x4 *)(p + head + j * W);
    return NT ? __builtin_nontemporal_load(q) : *q;
  }
  // the element outside the words that lane i takes, -1: none
  __device__ __forceinline__ int edge(int i) const { return i < head ? i : i < head + rest ? i + nb * W : -1; }
};
// a word of -inf
template <int DT> __device__ __forceinline__ u32x4 no_word() {
  constexpr uint32_t v = DT == WD_T_F32 ? 0xff800000u : DT == WD_T_BF16 ? 0xff80ff80u : 0xfc00fc00u;
  return {v, v, v, v};
}
// all loads before the first use, and what was unpacked for one pass over the words is not kept in registers for the next
template <int N> __device__ __forceinline__ void hold(u32x4 (&w)[N]) {
#pragma unroll
  for (int u = 0; u < N; ++u) asm volatile("" : "+v"(w[u]));
}
template <int DT> __device__ __forceinline__ void store_word(typename Elem<DT>::type *g, bool aligned, const float *x) {
  if (aligned) {      // the gradient is not read here: it need not push the logits out of the last cache (policy loss of 988 x 50021 fp16: 48 -> 36 us)
    __builtin_nontemporal_store(Elem<DT>::pack(x), (u32x4 *)g);
    return;
  }
#pragma unroll
  for (int i = 0; i < Elem<DT>::W; ++i) g[i] = Elem<DT>::from_float(x[i]);
}

__device__ __forceinline__ float exp_rel(float x, float m) { return __builtin_amdgcn_exp2f((x - m) * kLog2e); }

// (m, s) of two parts of a row.  m is at least the lowest finite number, so a part of nothing but -inf is (lowest, 0).
__device__ __forceinline__ void join(float &m, float &s, float m2, float s2) {
  const float M = fmaxf(m, m2);
  s = s * exp_rel(m, M) + s2 * exp_rel(m2, M);
  m = M;
}

// Reductions of a wavefront, the same value in every lane.  Neighbours meet inside their row of 16 lanes (each quad holds one value after the
// first two steps, so a mirrored row is an exchange), rows by the swaps of rows and halves: no trip through LDS, 6 steps of a few cycles each (policy loss of 988 x 50021 fp16 35.5 -> 34.3 us).
template <typename T, typename F> __device__ __forceinline__ T by_words(T v, F f) {
  static_assert(sizeof(T) == 4 || sizeof(T) == 8, "words");
  if constexpr (sizeof(T) == 4) return __builtin_bit_cast(T, f(__builtin_bit_cast(uint32_t, v)));
  else {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    return __builtin_bit_cast(T, (uint64_t)f((uint32_t)(b >> 32)) << 32 | f((uint32_t)b));
  }
}
template <int LANES> __device__ __forceinline__ auto swap_rows(uint32_t w) {
  if constexpr (LANES == 16) return __builtin_amdgcn_permlane16_swap(w, w, false, false);
  else return __builtin_amdgcn_permlane32_swap(w, w, false, false);
}
template <int CTRL, typename T> __device__ __forceinline__ T lane_move(T v) {
  return by_words(v, [](uint32_t w) { return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)w, CTRL, 0xf, 0xf, false); });
}
// f of the values of lanes i and i ^ LANES, the lower one's first, in both
template <int LANES, typename T, typename F> __device__ __forceinline__ T lane_halves(T v, F f) {
  const auto low = by_words(v, [](uint32_t w) { return swap_rows<LANES>(w)[0]; });
  const auto high = by_words(v, [](uint32_t w) { return swap_rows<LANES>(w)[1]; });
  return f(low, high);
}
template <typename T, typename F> __device__ __forceinline__ T wave_reduce(T v, F f) {
  v = f(v, lane_move<0xb1>(v));       // lanes 1 0 3 2 of each quad
  v = f(v, lane_move<0x4e>(v));       // 2 3 0 1
  v = f(v, lane_move<0x141>(v));      // half a row mirrored
  v = f(v, lane_move<0x140>(v));      // a row mirrored
  v = lane_halves<16>(v, f);
  return lane_halves<32>(v, f);
}
__device__ __forceinline__ float wave_max(float v) {
  return wave_reduce(v, [](float a, float b) { return fmaxf(a, b); });
}
template <typename T> __device__ __forceinline__ T wave_sum(T v) {
  return wave_reduce(v, [](T a, T b) { return a + b; });
}
__device__ __forceinline__ void wave_join(float &m, float &s) {
  const float M = wave_max(m);
  s = wave_sum(s * exp_rel(m, M));
  m = M;
}
// sum over the workgroup in a fixed order, the same value in every lane; `lds`: one T per wavefront, reusable after the call
template <int TH, typename T> __device__ __forceinline__ T block_sum(T v, T *lds) {
  v = wave_sum(v);
  if (TH == kWave) return v;
  __syncthreads();
  if ((threadIdx.x & (kWave - 1)) == 0) lds[threadIdx.x / kWave] = v;
  __syncthreads();
  T t = lds[0];
#pragma unroll
  for (int w = 1; w < TH / kWave; ++w) t += lds[w];
  return t;
}
template <int TH> __device__ __forceinline__ float block_max(float v, float *lds) {
  v = wave_max(v);
  if (TH == kWave) return v;
  __syncthreads();
  if ((threadIdx.x & (kWave - 1)) == 0) lds[threadIdx.x / kWave] = v;
  __syncthreads();
  float t = lds[0];
#pragma unroll
  for (int w = 1; w < TH / kWave; ++w) t = fmaxf(t, lds[w]);
  return t;
}

// sequence n as a range of rows that exist
__device__ __forceinline__ void seq_range(const wd_seq_rows_t &q, int64_t n, int64_t &a, int64_t &b) {
  a = min((int64_t)max(q.seq_offs[n], 0), q.rows);
  b = max(a, min((int64_t)q.seq_offs[n + 1], q.rows));
}
// rows in front of the first and behind the last sequence
__device__ __forceinline__ int64_t first_row(const wd_seq_rows_t &q) { return min((int64_t)max(q.seq_offs[0], 0), q.rows); }
__device__ __forceinline__ int64_t last_row(const wd_seq_rows_t &q) { return min((int64_t)max(q.seq_offs[q.nseq], 0), q.rows); }
__device__ __forceinline__ bool outside(const wd_seq_rows_t &q, int64_t r) { return r < first_row(q) || r >= last_row(q); }
// workgroup (part, row): parts of a row are neighbours in x, rows fill y and z (a grid dimension holds 2^32 lanes)
__device__ __forceinline__ int64_t block_row() { return (int64_t)blockIdx.z * gridDim.y + blockIdx.y; }
__device__ __forceinline__ bool is_action(const wd_seq_rows_t &q, int32_t t) { return t >= 0 && t < q.vocab; }

__device__ __forceinline__ float logp(float xt, float m, float s) { return (xt - m) - logf(s); }

// N words into the running maximum and sum
template <int DT, int N, int U> __device__ __forceinline__ void take_words(u32x4 (&w)[U], float &m, float &s) {
  constexpr int W = Elem<DT>::W;
  float x[N * W], M = m;
#pragma unroll
  for (int u = 0; u < N; ++u) Elem<DT>::unpack(w[u], x + u * W);
#pragma unroll
  for (int i = 0; i < N * W; ++i) M = fmaxf(M, x[i]);
  s *= exp_rel(m, M);
  m = M;
#pragma unroll
  for (int i = 0; i < N * W; ++i) s += exp_rel(x[i], m);
}
// four words of a wavefront, of which it has `left` (at least one): two that no lane has cost nothing (scores of 35 rows of 1000 bf16, replayed 7.0 -> 5.3 us)
template <int DT> __device__ __forceinline__ void take_four(u32x4 (&w)[4], int left, float &m, float &s) {
  hold(w);
  if (left > 2) take_words<DT, 4>(w, m, s);
  else take_words<DT, 2>(w, m, s);
}

// ---- (m, s) of every part of every row: LANES = 256, a workgroup a part; 64, a wavefront a (short) row.  A row in one part is done here,
// its log-probability too.  NT: logits that the last cache cannot keep for a later pass anyway are read past it (0.39 GB: 87 -> 82 us)
template <int DT, int LANES, bool NT>
__global__ void __launch_bounds__(256)
k_row_stats(wd_seq_rows_t q, int32_t nsplit, float2 *__restrict__ part, float *__restrict__ pick, float2 *__restrict__ stat,
            float *__restrict__ token) {
  constexpr int U = 4, ROWS = 256 / LANES;
  __shared__ float lm[256 / kWave], ls[256 / kWave];
  const int64_t r = block_row() * ROWS + threadIdx.x / LANES;
  const int z = (int)blockIdx.x, lane = threadIdx.x & (LANES - 1);
  if (r >= q.rows) return;
  const int32_t t = q.targets[r];
  if (outside(q, r) || !is_action(q, t)) {
    if (z == 0 && lane == 0) token[r] = 0.f;
    return;
  }
  const Row<DT> row(q.logits, q.ld, r, (int)q.vocab);
  const int per = (row.nb + nsplit - 1) / nsplit;
  const int j1 = min(row.nb, (z + 1) * per);
  const float xt = Elem<DT>::to_float(row.p[t]);
  float m = kLowest, s = 0.f;
  if (z == 0) {
    const int e = row.edge(lane);
    if (e >= 0) {
      const float x = Elem<DT>::to_float(row.p[e]);
      m = fmaxf(m, x);
      s = exp_rel(x, m);
    }
  }
  for (int j = z * per + lane; j < j1; j += LANES * U) {
    u32x4 w[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      w[u] = no_word<DT>();
      if (j + u * LANES < j1) w[u] = row.template word<NT>(j + u * LANES);
    }
    take_four<DT>(w, (j1 - __builtin_amdgcn_readfirstlane(j) + LANES - 1) / LANES, m, s);
  }
  wave_join(m, s);
  if (LANES > kWave) {
    if ((lane & (kWave - 1)) == 0) {
      lm[lane / kWave] = m;
      ls[lane / kWave] = s;
    }
    __syncthreads();
#pragma unroll
    for (int w = 1; w < LANES / kWave; ++w) join(m, s, lm[w], ls[w]);      // lane 0 holds its own wavefront's
  }
  if (lane == 0) {
    if (nsplit == 1) {
      stat[r] = make_float2(m, s);
      token[r] = logp(xt, m, s);
    } else {
      part[r * nsplit + z] = make_float2(m, s);
      if (z == 0) pick[r] = xt;      // whoever joins the parts may run while the gradient overwrites the logits
    }
  }
}

// What k_row_stats leaves of rows in parts (a power of two, at most 64): (m, s) of each part and the target's logit
struct Parts {
  const float2 *ms;
  const float *pick;
  int32_t n;
};
// the parts of row r joined by as many lanes, part z in lane z of them; the first one stores (m, s) and the target's log-probability where
// it is told to, and returns it
__device__ __forceinline__ float row_join(const Parts &p, int64_t r, int z, float2 *stat, float *token) {
  float2 ms = p.ms[r * p.n + z];
  const float xt = p.pick[r];
  for (int o = 1; o < p.n; o <<= 1) join(ms.x, ms.y, __shfl_xor(ms.x, o), __shfl_xor(ms.y, o));
  const float lp = logp(xt, ms.x, ms.y);
  if (z == 0) {
    if (stat) stat[r] = ms;
    if (token) token[r] = lp;
  }
  return lp;
}

// sum and number of the actions of rows [a, b)
template <int TH>
__device__ __forceinline__ void seq_logp(const wd_seq_rows_t &q, int64_t a, int64_t b, const Parts &p, float2 *stat, float *token,
                                         double &sum, int32_t &count, double *ld, int32_t *li) {
  double v = 0.0;      // long sums in 64 bits: a sequence of a thousand items sums to thousands, its pair's difference to units
  int32_t c = 0;
  if (p.n == 1) {
    for (int64_t r = a + threadIdx.x; r < b; r += TH) {
      v += token[r];      // 0 where the row is no action
      c += is_action(q, q.targets[r]);
    }
  } else {
    const int z = threadIdx.x & (p.n - 1);
    for (int64_t r = a + threadIdx.x / p.n; r < b; r += TH / p.n) {      // the lanes of a row leave together
      if (!is_action(q, q.targets[r])) continue;
      const float lp = row_join(p, r, z, stat, token);
      if (z == 0) {
        v += lp;
        ++c;
      }
    }
  }
  sum = block_sum<TH>(v, ld);
  count = block_sum<TH>(c, li);
}

// ---- scores: workgroup n = sequence n
__global__ void __launch_bounds__(256)
k_seq_logp(wd_seq_rows_t q, Parts p, int32_t length_norm, float2 *__restrict__ stat, float *__restrict__ token, float *__restrict__ seq) {
  constexpr int TH = 256;
  __shared__ double ld[TH / kWave];
  __shared__ int32_t li[TH / kWave];
  const int64_t n = block_row();
  if (n >= q.nseq) return;
  int64_t a, b;
  seq_range(q, n, a, b);
  double sum;
  int32_t count;
  seq_logp<TH>(q, a, b, p, stat, token, sum, count, ld, li);
  if (threadIdx.x == 0) seq[n] = (float)(length_norm ? sum / max(count, 1) : sum);
}

// log sigma(h) without overflow on either side
__device__ __forceinline__ double log_sigmoid(double h) { return fmin(h, 0.0) - log1p(exp(-fabs(h))); }

// ---- pairs.  The scalars of a pair are computed in 64 bits: there are a few of them, and the coefficient multiplies whole rows.
struct PairInput {
  float chosen, rejected, weight;      // of the reference, of the loss
};
__device__ __forceinline__ PairInput pair_input(const wd_pref_t &o, int64_t i) {
  return {o.ref_logp ? o.ref_logp[2 * i] : 0.f, o.ref_logp ? o.ref_logp[2 * i + 1] : 0.f, o.weights ? o.weights[i] : 1.f};
}
__device__ __forceinline__ double pair_difference(const PairInput &p, double chosen, double rejected) {
  return chosen - rejected - ((double)p.chosen - (double)p.rejected);
}
__device__ __forceinline__ double pair_loss_of(const wd_pref_t &o, double d) {
  if (o.kind == WD_PREF_SQUARE) {
    const double h = d - 0.5 / (double)o.beta;
    return h * h;
  }
  const double h = (double)o.beta * d - (double)o.margin, eps = (double)o.label_smoothing;
  const double loss = -(1.0 - eps) * log_sigmoid(h);
  return eps > 0.0 ? loss - eps * log_sigmoid(-h) : loss;      // a pair that is settled for good, h = inf: 0 x inf is no loss
}
// what a pair adds to the sum of the batch's loss
__device__ __forceinline__ double weighted(double loss, double weight) { return weight == 0.0 ? 0.0 : loss * weight; }
// grad_scale times dloss/dd of the batch's loss
__device__ __forceinline__ double pair_slope(const wd_pref_t &o, const PairInput &p, double d) {
  if (p.weight == 0.f) return 0.0;      // a pair that is left out adds nothing, an infinite d of its own too
  const double w = (double)o.scale * (double)p.weight * (double)o.grad_scale;
  if (o.kind == WD_PREF_SQUARE) return 2.0 * (d - 0.5 / (double)o.beta) * w;
  // sigma(h) - (1 - eps) as eps sigma(h) - (1 - eps) sigma(-h): no cancellation where the pair is settled
  const double h = (double)o.beta * d - (double)o.margin, eps = (double)o.label_smoothing;
  const double e = exp(-fabs(h)), big = 1.0 / (1.0 + e), small = e * big;
  return (double)o.beta * w * (eps * (h >= 0 ? big : small) - (1.0 - eps) * (h >= 0 ? small : big));
}
__device__ __forceinline__ void store_pair(const wd_pref_t &o, int64_t i, double d, double loss, const double *lp) {
  o.pair_loss[i] = (float)loss;
  o.difference[i] = (float)d;
  o.seq_logp[2 * i] = (float)lp[0];
  o.seq_logp[2 * i + 1] = (float)lp[1];
}

// workgroup i = pair i; leaves dloss/dlp of every row
__global__ void __launch_bounds__(256)
k_pref_pairs(wd_seq_rows_t q, wd_pref_t o, Parts p, float2 *__restrict__ stat, float *__restrict__ coef) {
  constexpr int TH = 256;
  __shared__ double ld[TH / kWave];
  __shared__ int32_t li[TH / kWave];
  const int64_t i = block_row();
  if (i >= q.nseq / 2) return;
  int64_t a[2], b[2];
  double lp[2];
  int32_t n[2];
  for (int k = 0; k < 2; ++k) {
    seq_range(q, 2 * i + k, a[k], b[k]);
    seq_logp<TH>(q, a[k], b[k], p, stat, o.token_logp, lp[k], n[k], ld, li);
    n[k] = o.length_norm ? max(n[k], 1) : 1;
    lp[k] /= n[k];
  }
  const PairInput in = pair_input(o, i);
  const double d = pair_difference(in, lp[0], lp[1]), slope = pair_slope(o, in, d);
  if (threadIdx.x == 0) store_pair(o, i, d, pair_loss_of(o, d), lp);
  for (int k = 0; k < 2; ++k) {
    const float c = (float)((k ? -slope : slope) / n[k]);
    for (int64_t r = a[k] + threadIdx.x; r < b[k]; r += TH) coef[r] = c;
  }
}

// ---- gradient of the logits from (m, s, coefficient) of each row: workgroup (row, part); the last one adds the loss up
template <int TH> __device__ __forceinline__ void weighted_sum(const float *v, const float *w, int64_t n, double scale, float *out, double *ld) {
  constexpr int U = 8;
  double t = 0.0;
  for (int64_t i = threadIdx.x; i < n; i += TH * U) {
    float x[U], y[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const bool in = i + u * TH < n;
      x[u] = in ? v[i + u * TH] : 0.f;
      y[u] = in && w ? w[i + u * TH] : 1.f;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) t += weighted((double)x[u], (double)y[u]);
  }
  t = block_sum<TH>(t, ld);
  if (threadIdx.x == 0) *out = (float)(t * scale);
}

struct RowScalars {
  float m, s, c;
};
// part z of a row's gradient; zeros for a row that is no action (its logits are not read).  scalars() is asked for (m, s, c) when the first
// words are on their way.
template <int DT, int TH, bool NT, typename F>
__device__ __forceinline__ void grad_part(const Row<DT> &row, typename Elem<DT>::type *g, int z, int nsplit, bool action, int32_t t, F scalars) {
  constexpr int W = Elem<DT>::W, U = 4;
  const int lane = threadIdx.x & (TH - 1);      // TH lanes: a workgroup or a wavefront of it
  const int per = (row.nb + nsplit - 1) / nsplit;
  const int j0 = z * per, j1 = min(row.nb, (z + 1) * per), jt = t < row.head ? -1 : (t - row.head) / W;
  typename Elem<DT>::type *gb = g + row.head;
  const bool aligned = ((uintptr_t)gb & 15) == 0;
  const int e = z == 0 ? row.edge(lane) : -1;
  float x[W];
  if (!action) {
    if (e >= 0) g[e] = 0;
#pragma unroll
    for (int i = 0; i < W; ++i) x[i] = 0.f;
    for (int j = j0 + lane; j < j1; j += TH) store_word<DT>(gb + j * W, aligned, x);
    return;
  }
  RowScalars k;
  for (int jw = j0; jw < j1 || jw == j0; jw += TH * U) {      // once at least: a short row may be all edge
    const int j = jw + lane;
    u32x4 w[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      w[u] = no_word<DT>();
      if (j + u * TH < j1) w[u] = row.template word<NT>(j + u * TH);
    }
    if (jw == j0) {
      const float xe = e >= 0 ? Elem<DT>::to_float(row.p[e]) : 0.f;
      k = scalars();
      k.s = -k.c / k.s;
      if (e >= 0) g[e] = Elem<DT>::from_float(k.s * exp_rel(xe, k.m) + (e == t ? k.c : 0.f));
    }
    hold(w);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int ju = j + u * TH;
      if (ju >= j1) break;
      Elem<DT>::unpack(w[u], x);
#pragma unroll
      for (int i = 0; i < W; ++i) x[i] = k.s * exp_rel(x[i], k.m);
      if (ju == jt) {
#pragma unroll
        for (int i = 0; i < W; ++i) x[i] += row.head + ju * W + i == t ? k.c : 0.f;
      }
      store_word<DT>(gb + ju * W, aligned, x);
    }
  }
}

template <int DT, int LANES, bool NT>
__global__ void __launch_bounds__(256)
k_logits_grad(wd_seq_rows_t q, void *dlogits, int64_t ldg, int32_t zero_tail, int32_t nsplit, const float2 *__restrict__ stat,
              const float *__restrict__ coef, const float *__restrict__ pair_loss, const float *__restrict__ weights, double scale,
              float *__restrict__ loss) {
  constexpr int ROWS = 256 / LANES;
  __shared__ double ld[256 / kWave];
  const int z = (int)blockIdx.x;
  if (loss && z == 0 && block_row() == (q.rows + ROWS - 1) / ROWS) weighted_sum<256>(pair_loss, weights, q.nseq / 2, scale, loss, ld);
  const int64_t r = block_row() * ROWS + threadIdx.x / LANES;
  if (r >= q.rows) return;
  const bool tail = outside(q, r);
  if (tail && !zero_tail) return;
  const int32_t t = q.targets[r];
  const bool action = !tail && is_action(q, t);
  const Row<DT> row(q.logits, q.ld, r, (int)q.vocab);
  grad_part<DT, LANES, NT>(row, (typename Elem<DT>::type *)dlogits + r * ldg, z, nsplit, action, t, [&] {
    const float2 ms = stat[r];
    return RowScalars{ms.x, ms.y, coef[r]};
  });
}

// sequence of row r, by a wavefront: the number of sequences that end in front of it
__device__ __forceinline__ int64_t wave_sequence(const wd_seq_rows_t &q, int64_t r) {
  const int lane = threadIdx.x & (kWave - 1);
  int64_t s = 0;
  for (int64_t k = lane; k - lane < q.nseq; k += kWave) s += __popcll(__ballot(k < q.nseq && q.seq_offs[k + 1] <= r));
  return s;
}

// Pairs and gradient in one launch, up to kPairRows rows and kPairSeqs sequences (self_pairs()).  Every wavefront adds its row's pair up for itself, a lane per row or
// per part of one, behind the row's first loads; the workgroup behind the last row does the pairs' outputs and the loss.
__device__ __forceinline__ void wave_pair(const wd_seq_rows_t &q, const wd_pref_t &o, int64_t i, const Parts &p, double *lp, int32_t *n) {
  const int lane = threadIdx.x & (kWave - 1), z = lane & (p.n - 1);
  int64_t a[2], b[2];
  for (int k = 0; k < 2; ++k) seq_range(q, 2 * i + k, a[k], b[k]);
  for (int k = 0; k < 2; ++k) {
    double v = 0.0;
    int32_t c = 0;
    if (p.n == 1) {
      const int first = (int)a[k] + lane, last = (int)b[k];
      if (o.length_norm) {
#pragma unroll 4
        for (int r = first; r < last; r += kWave) {
          v += o.token_logp[r];      // 0 where the row is no action
          c += is_action(q, q.targets[r]);
        }
      } else {
#pragma unroll 4
        for (int r = first; r < last; r += kWave) v += o.token_logp[r];
      }
    } else {
      for (int64_t r = a[k] + lane / p.n; r < b[k]; r += kWave / p.n) {      // the lanes of a row leave together
        if (!is_action(q, q.targets[r])) continue;
        const float x = row_join(p, r, z, nullptr, nullptr);
        if (z) continue;
        v += x;
        ++c;
      }
    }
    n[k] = 1;
    if (o.length_norm) n[k] = max(wave_sum(c), 1);
    lp[k] = wave_sum(v) / n[k];
  }
}
struct PairSums {
  double lp[kPairSeqs];
  float token[kPairRows];
  int32_t offs[kPairSeqs + 1];
  uint8_t action[kPairRows];
};
// one workgroup: token_logp of split rows, the pairs' outputs and the loss.  All rows through LDS once, a wavefront per sequence, a lane per pair
template <int TH> __device__ __forceinline__ void all_pairs(const wd_seq_rows_t &q, const wd_pref_t &o, const Parts &p, PairSums &x, double *ld) {
  const int rows = (int)q.rows, seqs = (int)q.nseq, lane = threadIdx.x & (kWave - 1);
  for (int n = threadIdx.x; n <= seqs; n += TH) x.offs[n] = min(max(q.seq_offs[n], 0), rows);
  const int z = threadIdx.x & (p.n - 1);
#pragma unroll 4
  for (int r = threadIdx.x / p.n; r < rows; r += TH / p.n) {      // the lanes of a row leave together
    const bool action = !outside(q, r) && is_action(q, q.targets[r]);
    float lp = 0.f;
    if (p.n == 1) lp = o.token_logp[r];
    else if (action) lp = row_join(p, r, z, nullptr, o.token_logp);
    if (z) continue;
    x.token[r] = lp;
    x.action[r] = action;
  }
  __syncthreads();
  for (int n = threadIdx.x / kWave; n < seqs; n += TH / kWave) {
    double v = 0.0;
    int32_t c = 0;
    for (int r = x.offs[n] + lane; r < x.offs[n + 1]; r += kWave) {
      v += x.token[r];
      c += x.action[r];
    }
    v = wave_sum(v);
    if (o.length_norm) v /= max(wave_sum(c), 1);
    if (lane == 0) x.lp[n] = v;
  }
  __syncthreads();
  double total = 0.0;
  for (int i = threadIdx.x; i < seqs / 2; i += TH) {
    const PairInput in = pair_input(o, i);
    const double d = pair_difference(in, x.lp[2 * i], x.lp[2 * i + 1]), loss = pair_loss_of(o, d);
    store_pair(o, i, d, loss, x.lp + 2 * i);
    total += weighted(loss, (double)in.weight);
  }
  total = block_sum<TH>(total, ld);
  if (threadIdx.x == 0) *o.loss = (float)(total * (double)o.scale);
}
template <int DT>
__global__ void __launch_bounds__(256)
k_pref_grad(wd_seq_rows_t q, wd_pref_t o, int32_t nsplit, Parts p, const float2 *__restrict__ stat) {
  constexpr int TH = 256;
  __shared__ double ld[TH / kWave];
  __shared__ PairSums sums;
  const int64_t r = block_row();
  const int z = (int)blockIdx.x, lane = threadIdx.x & (kWave - 1);
  double lp[2];
  int32_t n[2];
  if (r == q.rows && z == 0) all_pairs<TH>(q, o, p, sums, ld);
  if (r >= q.rows || !o.dlogits) return;
  const bool tail = outside(q, r);
  if (tail && !o.zero_tail) return;
  const int32_t t = q.targets[r];
  const bool action = !tail && is_action(q, t);
  const Row<DT> row(q.logits, q.ld, r, (int)q.vocab);
  grad_part<DT, TH, false>(row, (typename Elem<DT>::type *)o.dlogits + r * o.ld_dlogits, z, nsplit, action, t, [&] {
    float2 ms;
    if (p.n == 1) {
      ms = stat[r];
    } else {
      ms = p.ms[r * p.n + (lane & (p.n - 1))];
      for (int k = 1; k < p.n; k <<= 1) join(ms.x, ms.y, __shfl_xor(ms.x, k), __shfl_xor(ms.y, k));
      ms.x = __shfl(ms.x, 0);      // the sides of a join round differently
      ms.y = __shfl(ms.y, 0);
    }
    const int64_t s = wave_sequence(q, r);
    const PairInput in = pair_input(o, s / 2);
    wave_pair(q, o, s / 2, p, lp, n);
    const double slope = pair_slope(o, in, pair_difference(in, lp[0], lp[1]));
    return RowScalars{ms.x, ms.y, (float)(s & 1 ? -slope / n[1] : slope / n[0])};
  });
}

// ---- clipped policy loss
// workgroup n = sequence n: its number of actions, and by row the part of the weight that is the sequence's own and the advantage
template <int TH>
__global__ void __launch_bounds__(TH)
k_policy_rows(wd_seq_rows_t q, wd_policy_t o, float *__restrict__ w, float *__restrict__ adv, int32_t *__restrict__ cnt) {
  __shared__ int32_t li[TH / kWave];
  const int64_t n = block_row();
  if (n >= q.nseq) return;
  int64_t a, b;
  seq_range(q, n, a, b);
  int32_t c = 0;
  for (int64_t r = a + threadIdx.x; r < b; r += TH) c += is_action(q, q.targets[r]);
  c = block_sum<TH>(c, li);
  const float inv = o.reduction == WD_POLICY_SEQUENCE_MEAN ? 1.0f / (float)max(c, 1) : 1.0f;
  const float av = o.adv_per_row ? 0.f : o.advantages[n];
  for (int64_t r = a + threadIdx.x; r < b; r += TH) {
    w[r] = inv;
    adv[r] = o.adv_per_row ? o.advantages[r] : av;
  }
  if (threadIdx.x == 0) cnt[n] = c;
}
// the rest of every weight, the same in all rows: 1, 1 / actions, or 1 / sequences with an action; `lane` of `step` lanes adds
__device__ __forceinline__ int32_t policy_count(const wd_seq_rows_t &q, const wd_policy_t &o, const int32_t *cnt, int lane, int step) {
  int32_t d = 0;
  if (o.reduction != WD_POLICY_SUM)
    for (int64_t n = lane; n < q.nseq; n += step) d += o.reduction == WD_POLICY_TOKEN_MEAN ? cnt[n] : cnt[n] > 0;
  return d;
}
__global__ void __launch_bounds__(1024) k_policy_total(wd_seq_rows_t q, wd_policy_t o, int32_t *__restrict__ cnt) {
  __shared__ int32_t li[1024 / kWave];
  const int32_t d = block_sum<1024>(policy_count(q, o, cnt, threadIdx.x, 1024), li);
  if (threadIdx.x == 0) cnt[q.nseq] = d;
}
// by a wavefront; many sequences: k_policy_total has done it
__device__ __forceinline__ float policy_factor(const wd_seq_rows_t &q, const wd_policy_t &o, const int32_t *cnt) {
  if (o.reduction == WD_POLICY_SUM) return 1.f;
  const int32_t d = q.nseq > kCountSeqs ? cnt[q.nseq] : wave_sum(policy_count(q, o, cnt, threadIdx.x & (kWave - 1), kWave));
  return 1.0f / (float)max(d, 1);
}

struct PolicyRow {
  float loss, kl, clipped, slope;
};
// rho = e^(lp - old); the surrogate takes the smaller of rho A and clip(rho) A and has no slope where that is the clipped one;
// k = e^(ref - lp) - (ref - lp) - 1 >= 0 estimates KL(policy || reference) from the sampled item (expm1: small differences keep bits)
__device__ __forceinline__ PolicyRow policy_row(const wd_policy_t &o, float lp, float old, float adv, float ref) {
  PolicyRow p;
  const float rho = expf(lp - old);
  const float a = adv == 0.f && rho == INFINITY ? 0.f : rho * adv;      // no advantage: no loss and no slope, also where the ratio is beyond fp32
  const float b = fminf(fmaxf(rho, 1.0f - o.clip_low), 1.0f + o.clip_high) * adv;
  const bool out = a > b;
  p.loss = -(out ? b : a);
  p.slope = out ? 0.f : -a;
  p.clipped = out ? 1.f : 0.f;
  p.kl = 0.f;
  if (o.ref_logp) {
    const float d = ref - lp, e = expm1f(d);
    p.kl = e == INFINITY ? e : e - d;      // lp = -inf: d is infinite too, e^d the larger
    if (o.kl_coef != 0.f) {      // told of only: an infinite k leaves the loss alone
      p.loss += o.kl_coef * p.kl;
      p.slope -= o.kl_coef * e;
    }
  }
  return p;
}

// the weight of an action of sequence n, by a wavefront, for at most kWeightRows rows (any number, reduction SUM): a bit for each action
__device__ __forceinline__ float self_weight(const wd_seq_rows_t &q, const wd_policy_t &o, int64_t n) {
  if (o.reduction == WD_POLICY_SUM) return 1.f;
  const int lane = threadIdx.x & (kWave - 1), rows = (int)q.rows, first = (int)first_row(q), last = (int)last_row(q);
  uint32_t low = 0, high = 0;      // lane k: rows 64 k ..
  int32_t actions = 0;
#pragma unroll 4
  for (int k = 0; k < rows; k += kWave) {
    const int r = k + lane;
    const uint64_t bits = __ballot(r >= first && r < last && is_action(q, q.targets[min(r, rows - 1)]));
    if (lane == k / kWave) {
      low = (uint32_t)bits;
      high = (uint32_t)(bits >> 32);
    }
    actions += __popcll(bits);
  }
  if (o.reduction == WD_POLICY_TOKEN_MEAN) return 1.0f / (float)actions;
  auto count = [&](int64_t s) {
    int64_t a, b;
    seq_range(q, s, a, b);
    int32_t c = 0;
    for (int k = 0; k < rows; k += kWave) {
      const uint64_t bits = (uint64_t)(uint32_t)__builtin_amdgcn_readlane(high, k / kWave) << 32 | (uint32_t)__builtin_amdgcn_readlane(low, k / kWave);
      const int lo = min(max((int)a - k, 0), kWave), hi = min(max((int)b - k, 0), kWave);
      const uint64_t below = hi == kWave ? ~0ull : (1ull << hi) - 1, under = lo == kWave ? ~0ull : (1ull << lo) - 1;
      c += __popcll(bits & below & ~under);
    }
    return c;
  };
  int32_t seqs = 0;
  for (int64_t s = lane; s - lane < q.nseq; s += kWave) seqs += __popcll(__ballot(s < q.nseq && count(min(s, q.nseq - 1)) > 0));
  return (1.0f / (float)count(n)) * (1.0f / (float)seqs);
}
// weight and advantage of row r, an action, by a wavefront
__device__ __forceinline__ void self_row(const wd_seq_rows_t &q, const wd_policy_t &o, int64_t r, float &w, float &adv) {
  const int64_t n = o.adv_per_row && o.reduction != WD_POLICY_SEQUENCE_MEAN ? 0 : wave_sequence(q, r);
  adv = o.advantages[o.adv_per_row ? r : n];
  w = self_weight(q, o, n);
}

// The whole row in registers between its statistics and its gradient: one read and one write of the logits, workgroup = row.
// w == nullptr: no launch has made weights and advantages; each wavefront finds them.
template <int DT, int TH, int NV>
__global__ void __launch_bounds__(TH, TH == 512 ? 4 : 1)
k_policy_resident(wd_seq_rows_t q, wd_policy_t o, const float *__restrict__ w, const float *__restrict__ adv,
                  const int32_t *__restrict__ cnt, float *__restrict__ rows3) {
  constexpr int W = Elem<DT>::W;
  typedef typename Elem<DT>::type type;
  __shared__ float lf[TH / kWave], lg[TH / kWave];
  const int64_t r = block_row();
  if (r >= q.rows) return;
  const bool tail = outside(q, r);
  if (tail && threadIdx.x == 0) {
    o.token_logp[r] = 0.f;
    rows3[r] = rows3[q.rows + r] = rows3[2 * q.rows + r] = 0.f;
  }
  if (tail && !o.zero_tail) return;
  const int32_t t = q.targets[r];
  const Row<DT> row(q.logits, q.ld, r, (int)q.vocab);
  type *g = (type *)o.dlogits + r * o.ld_dlogits;
  if (tail || !is_action(q, t)) {
    if (threadIdx.x == 0 && !tail) {
      o.token_logp[r] = 0.f;
      rows3[r] = rows3[q.rows + r] = rows3[2 * q.rows + r] = 0.f;
    }
    if (o.dlogits) grad_part<DT, TH, false>(row, g, 0, 1, false, -1, [] { return RowScalars{0.f, 1.f, 0.f}; });
    return;
  }
  u32x4 v[NV];
#pragma unroll
  for (int u = 0; u < NV; ++u) {
    v[u] = no_word<DT>();
    if ((int)threadIdx.x + u * TH < row.nb) v[u] = row.word(threadIdx.x + u * TH);
  }
  const int e = row.edge(threadIdx.x);
  const float xe = e >= 0 ? Elem<DT>::to_float(row.p[e]) : -INFINITY;
  const float xt = Elem<DT>::to_float(row.p[t]);
  const float old = o.old_logp[r], ref = o.ref_logp ? o.ref_logp[r] : 0.f;
  float wr = 1.f, ar;
  if (w) {
    wr = w[r] * policy_factor(q, o, cnt);
    ar = adv[r];
  } else {
    self_row(q, o, r, wr, ar);
  }
  hold(v);
  float x[W], m = fmaxf(kLowest, xe);
#pragma unroll
  for (int u = 0; u < NV; ++u) {
    Elem<DT>::unpack(v[u], x);
#pragma unroll
    for (int i = 0; i < W; ++i) m = fmaxf(m, x[i]);
  }
  m = block_max<TH>(m, lf);
  hold(v);
  float s = exp_rel(xe, m);
#pragma unroll
  for (int u = 0; u < NV; ++u) {
    Elem<DT>::unpack(v[u], x);
#pragma unroll
    for (int i = 0; i < W; ++i) s += exp_rel(x[i], m);
  }
  s = block_sum<TH>(s, lg);
  const float lp = logp(xt, m, s);
  const PolicyRow p = policy_row(o, lp, old, ar, ref);
  if (threadIdx.x == 0) {
    o.token_logp[r] = lp;
    rows3[r] = p.loss * wr;
    rows3[q.rows + r] = p.kl * wr;
    rows3[2 * q.rows + r] = p.clipped * wr;
  }
  if (!o.dlogits) return;
  const float c = p.slope * wr * o.grad_scale, k = -c / s;
  const int jt = t < row.head ? -1 : (t - row.head) / W;
  type *gb = g + row.head;
  const bool aligned = ((uintptr_t)gb & 15) == 0;
  if (e >= 0) g[e] = Elem<DT>::from_float(k * exp_rel(xe, m) + (e == t ? c : 0.f));
  hold(v);
#pragma unroll
  for (int u = 0; u < NV; ++u) {
    const int j = threadIdx.x + u * TH;
    if (j >= row.nb) break;
    Elem<DT>::unpack(v[u], x);
#pragma unroll
    for (int i = 0; i < W; ++i) x[i] = k * exp_rel(x[i], m);
    if (j == jt) {
#pragma unroll
      for (int i = 0; i < W; ++i) x[i] += row.head + j * W + i == t ? c : 0.f;
    }
    store_word<DT>(gb + j * W, aligned, x);
  }
}

// ---- a handful of rows (at most 64, 64 K logits): a loss in one launch.  The launches of the general way cost a caller more than its kernels:
// 25 rows of 2000 14.7 -> 12.3 us a call.  Every workgroup finds the statistics of all rows for itself, so none waits for another; they share
// the gradient, and the first one does everything else (policy, replayed from a graph: 64 rows of 1000 15.4 -> 11.9 us, 35 rows 9.5 -> 8.6).
// A gradient in the logits' place would be under the other workgroups' feet: one workgroup then.  Few rows are shared by wavefronts
// (scores of one row of 65536 fp32: 24 -> 8.6 us a call; the general way 11.6).
struct Tiny {
  static constexpr int kRows = kWave, kWaves = 1024 / kWave;
  float m[kRows], s[kRows], lp[kRows], c[kRows];
  int32_t t[kRows];      // the target, -1: no action
  int64_t begin[kRows], end[kRows];
  float pm[kWaves], ps[kWaves], pt[kWaves];      // rows in parts
};
// wavefronts that share a row in the statistics, as a power of two; a part has 256 words or more, one round of loads
__device__ __forceinline__ int tiny_parts(int64_t rows, int words) {
  int p = 0;
  while (rows << p <= Tiny::kWaves / 2 && words > 256 << p) ++p;
  return p;
}
__device__ __forceinline__ int tiny_wave() { return __builtin_amdgcn_readfirstlane(threadIdx.x / kWave); }
template <int DT, int TH> __device__ __forceinline__ void tiny_stats(const wd_seq_rows_t &q, Tiny &x, float *token) {
  constexpr int U = 4;
  const int lane = threadIdx.x & (kWave - 1), wave = tiny_wave(), shift = tiny_parts(q.rows, (int)q.vocab / Elem<DT>::W), P = 1 << shift;
  const int z = wave & (P - 1);
  if (threadIdx.x < q.nseq) seq_range(q, threadIdx.x, x.begin[threadIdx.x], x.end[threadIdx.x]);
  for (int r = wave >> shift; r < q.rows; r += Tiny::kWaves >> shift) {
    int32_t t = q.targets[r];
    if (outside(q, r) || !is_action(q, t)) t = -1;
    float m = kLowest, s = 0.f, xt = 0.f;
    if (t >= 0) {
      const Row<DT> row(q.logits, q.ld, r, (int)q.vocab);
      const int per = (row.nb + P - 1) >> shift, j1 = min(row.nb, (z + 1) * per), e = z == 0 ? row.edge(lane) : -1;
      xt = Elem<DT>::to_float(row.p[t]);
      if (e >= 0) {
        const float v = Elem<DT>::to_float(row.p[e]);
        m = fmaxf(m, v);
        s = exp_rel(v, m);
      }
      for (int j = z * per + lane; j < j1; j += kWave * U) {
        u32x4 w[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          w[u] = no_word<DT>();
          if (j + u * kWave < j1) w[u] = row.word(j + u * kWave);
        }
        take_four<DT>(w, (j1 - __builtin_amdgcn_readfirstlane(j) + kWave - 1) / kWave, m, s);
      }
      wave_join(m, s);
    }
    if (lane == 0) {
      if (z == 0) x.t[r] = t;
      if (P > 1) {      // the rows are at most as many as there are wavefronts for
        x.pm[wave] = m;
        x.ps[wave] = s;
        x.pt[wave] = xt;
      } else {
        x.m[r] = m;
        x.s[r] = s;
        x.lp[r] = t >= 0 ? logp(xt, m, s) : 0.f;
        if (blockIdx.x == 0) token[r] = x.lp[r];
      }
    }
  }
  __syncthreads();
  if (P > 1) {
    if (threadIdx.x < q.rows) {
      const int r = threadIdx.x;
      float m = x.pm[r * P], s = x.ps[r * P];
      for (int k = 1; k < P; ++k) join(m, s, x.pm[r * P + k], x.ps[r * P + k]);
      x.m[r] = m;
      x.s[r] = s;
      x.lp[r] = x.t[r] >= 0 ? logp(x.pt[r * P], m, s) : 0.f;
      if (blockIdx.x == 0) token[r] = x.lp[r];
    }
    __syncthreads();
  }
}
// and in the gradient, up to 64 of all workgroups
__host__ __device__ __forceinline__ int tiny_grad_parts(int64_t rows, int words) {
  return rows < 1 ? 1 : words <= 256 ? 1 : (int)(Tiny::kRows / rows) < (words + 255) / 256 ? (int)(Tiny::kRows / rows) : (words + 255) / 256;
}
template <int DT, int TH>
__device__ __forceinline__ void tiny_gradient(const wd_seq_rows_t &q, const Tiny &x, void *dlogits, int64_t ldg, int32_t zero_tail) {
  __syncthreads();
  if (!dlogits) return;
  const int P = tiny_grad_parts(q.rows, (int)q.vocab / Elem<DT>::W);
  for (int i = blockIdx.x * Tiny::kWaves + tiny_wave(); i < q.rows * P; i += gridDim.x * Tiny::kWaves) {
    const int r = i / P;
    if (!zero_tail && outside(q, r)) continue;
    const Row<DT> row(q.logits, q.ld, r, (int)q.vocab);
    grad_part<DT, kWave, false>(row, (typename Elem<DT>::type *)dlogits + r * ldg, i - r * P, P, x.t[r] >= 0, x.t[r],
                                [&] { return RowScalars{x.m[r], x.s[r], x.c[r]}; });
  }
}
template <int DT>
__global__ void __launch_bounds__(1024) k_seq_tiny(wd_seq_rows_t q, int32_t length_norm, float *__restrict__ token, float *__restrict__ seq) {
  constexpr int TH = 1024;
  __shared__ Tiny x;
  tiny_stats<DT, TH>(q, x, token);
  const int lane = threadIdx.x & (kWave - 1);
  for (int n = threadIdx.x / kWave; n < q.nseq; n += TH / kWave) {      // a lane per row
    const bool in = lane >= x.begin[n] && lane < x.end[n];
    const double sum = wave_sum(in ? (double)x.lp[lane] : 0.0);
    const int32_t count = wave_sum(in && x.t[lane] >= 0 ? 1 : 0);
    if (lane == 0) seq[n] = (float)(length_norm ? sum / max(count, 1) : sum);
  }
}
template <int DT> __global__ void __launch_bounds__(1024) k_pref_tiny(wd_seq_rows_t q, wd_pref_t o) {
  constexpr int TH = 1024;
  __shared__ Tiny x;
  __shared__ double part[Tiny::kRows / 2];
  const int lane = threadIdx.x & (kWave - 1), pairs = (int)q.nseq / 2;
  PairInput next = {0.f, 0.f, 1.f};      // on its way while the rows are read
  if (threadIdx.x / kWave < pairs) next = pair_input(o, threadIdx.x / kWave);
  tiny_stats<DT, TH>(q, x, o.token_logp);
  for (int i = threadIdx.x / kWave; i < pairs; i += TH / kWave) {      // a lane per row
    const PairInput in = next;
    if (i + TH / kWave < pairs) next = pair_input(o, i + TH / kWave);
    double lp[2];
    int32_t n[2];
    for (int k = 0; k < 2; ++k) {
      const bool mine = lane >= x.begin[2 * i + k] && lane < x.end[2 * i + k];
      n[k] = o.length_norm ? max(wave_sum(mine && x.t[lane] >= 0 ? 1 : 0), 1) : 1;
      lp[k] = wave_sum(mine ? (double)x.lp[lane] : 0.0) / n[k];
    }
    const double d = pair_difference(in, lp[0], lp[1]), slope = pair_slope(o, in, d), loss = pair_loss_of(o, d);
    if (lane == 0) {
      if (blockIdx.x == 0) store_pair(o, i, d, loss, lp);
      part[i] = weighted(loss, (double)in.weight);
    }
    for (int k = 0; k < 2; ++k)
      if (lane >= x.begin[2 * i + k] && lane < x.end[2 * i + k]) x.c[lane] = (float)((k ? -slope : slope) / n[k]);
  }
  tiny_gradient<DT, TH>(q, x, o.dlogits, o.ld_dlogits, o.zero_tail);
  if (blockIdx.x == 0 && threadIdx.x < kWave) {
    const double total = wave_sum(lane < pairs ? part[lane] : 0.0);
    if (lane == 0) *o.loss = (float)(total * (double)o.scale);
  }
}
template <int DT> __global__ void __launch_bounds__(1024) k_policy_tiny(wd_seq_rows_t q, wd_policy_t o) {
  constexpr int TH = 1024;
  __shared__ Tiny x;
  float old = 0.f, ref = 0.f, adv = 0.f;      // on their way while the rows are read
  if (threadIdx.x < q.rows) {
    old = o.old_logp[threadIdx.x];
    if (o.ref_logp) ref = o.ref_logp[threadIdx.x];
  }
  if (threadIdx.x < (o.adv_per_row ? q.rows : q.nseq)) adv = o.advantages[threadIdx.x];
  tiny_stats<DT, TH>(q, x, o.token_logp);
  if (threadIdx.x < kWave) {      // a lane per row
    const int r = threadIdx.x;
    const bool action = r < q.rows && x.t[r] >= 0;
    int32_t mine = 1, total = wave_sum(action ? 1 : 0), seqs = 0, n = 0;
    for (int k = 0; k < q.nseq; ++k) {
      const bool in = r >= x.begin[k] && r < x.end[k];
      const int32_t c = __popcll(__ballot(in && action));
      if (in) {
        mine = c;
        n = k;
      }
      seqs += c > 0;
    }
    if (!o.adv_per_row) adv = __shfl(adv, n);
    float loss = 0.f, kl = 0.f, clipped = 0.f;
    if (action) {
      const float w = o.reduction == WD_POLICY_SUM ? 1.0f : o.reduction == WD_POLICY_TOKEN_MEAN ? 1.0f / (float)total : (1.0f / (float)mine) * (1.0f / (float)seqs);
      const PolicyRow p = policy_row(o, x.lp[r], old, adv, ref);
      loss = p.loss * w;
      kl = p.kl * w;
      clipped = p.clipped * w;
      x.c[r] = p.slope * w * o.grad_scale;
    }
    const double a = wave_sum((double)loss), b = wave_sum((double)kl), c = wave_sum((double)clipped);
    if (r == 0 && blockIdx.x == 0) {
      o.sums[0] = (float)a;
      o.sums[1] = (float)b;
      o.sums[2] = (float)c;
    }
  }
  tiny_gradient<DT, TH>(q, x, o.dlogits, o.ld_dlogits, o.zero_tail);
}

// rows too long for the registers: loss and coefficient of each row, a lane per part of it
__global__ void __launch_bounds__(256)
k_policy_join(wd_seq_rows_t q, wd_policy_t o, Parts ps, const float *__restrict__ w, const float *__restrict__ adv, const int32_t *__restrict__ cnt,
              float2 *__restrict__ stat, float *__restrict__ coef, float *__restrict__ rows3) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, r = i / ps.n;
  const int z = (int)(i & (ps.n - 1));
  const float factor = policy_factor(q, o, cnt);      // whole wavefronts
  if (r >= q.rows) return;
  float lp = 0.f, wr = 0.f, c = 0.f;
  PolicyRow p = {0.f, 0.f, 0.f, 0.f};
  if (!outside(q, r) && is_action(q, q.targets[r])) {
    lp = ps.n == 1 ? o.token_logp[r] : row_join(ps, r, z, stat, o.token_logp);
    wr = w[r] * factor;
    p = policy_row(o, lp, o.old_logp[r], adv[r], o.ref_logp ? o.ref_logp[r] : 0.f);
    c = p.slope * wr * o.grad_scale;
  }
  if (z) return;
  coef[r] = c;
  rows3[r] = p.loss * wr;
  rows3[q.rows + r] = p.kl * wr;
  rows3[2 * q.rows + r] = p.clipped * wr;
}

// The same in the gradient's launch, where rows find their weights themselves: every wavefront joins its row and does that behind the row's
// first loads (28 x 97327 fp32 22 -> 17 us, 250 x 140001 bf16 38 -> 34)
template <int DT, bool GRAD, bool NT>
__global__ void __launch_bounds__(256)
k_policy_grad(wd_seq_rows_t q, wd_policy_t o, int32_t nsplit, Parts p, const float2 *__restrict__ stat, float *__restrict__ rows3) {
  constexpr int TH = 256;
  const int64_t r = block_row();
  if (r >= q.rows) return;
  const int z = (int)blockIdx.x, lane = threadIdx.x & (kWave - 1);
  const bool tail = outside(q, r), writer = z == 0 && threadIdx.x == 0;
  const int32_t t = q.targets[r];
  const bool action = !tail && is_action(q, t);
  if (writer && !action) rows3[r] = rows3[q.rows + r] = rows3[2 * q.rows + r] = 0.f;
  auto scalars = [&] {
    const float old = o.old_logp[r], ref = o.ref_logp ? o.ref_logp[r] : 0.f;
    float2 ms;
    float lp, w, adv;
    if (p.n == 1) {
      ms = stat[r];
      lp = o.token_logp[r];
    } else {
      ms = p.ms[r * p.n + (lane & (p.n - 1))];
      const float xt = p.pick[r];
      for (int k = 1; k < p.n; k <<= 1) join(ms.x, ms.y, __shfl_xor(ms.x, k), __shfl_xor(ms.y, k));
      ms.x = __shfl(ms.x, 0);      // the sides of a join round differently
      ms.y = __shfl(ms.y, 0);
      lp = logp(xt, ms.x, ms.y);
      if (writer) o.token_logp[r] = lp;
    }
    self_row(q, o, r, w, adv);
    const PolicyRow x = policy_row(o, lp, old, adv, ref);
    if (writer) {
      rows3[r] = x.loss * w;
      rows3[q.rows + r] = x.kl * w;
      rows3[2 * q.rows + r] = x.clipped * w;
    }
    return RowScalars{ms.x, ms.y, x.slope * w * o.grad_scale};
  };
  if constexpr (GRAD) {
    if (tail && !o.zero_tail) return;
    const Row<DT> row(q.logits, q.ld, r, (int)q.vocab);
    grad_part<DT, TH, NT>(row, (typename Elem<DT>::type *)o.dlogits + r * o.ld_dlogits, z, nsplit, action, t, scalars);
  } else if (action) {
    scalars();
  }
}

// out[k] = sum of rows3[k][0..rows), in a fixed order
__global__ void __launch_bounds__(1024) k_policy_sums(const float *__restrict__ rows3, int64_t rows, float *__restrict__ out) {
  __shared__ double ld[1024 / kWave];
  weighted_sum<1024>(rows3 + blockIdx.x * rows, nullptr, rows, 1.0, out + blockIdx.x, ld);
}

// ---- host side
int check_rows(const char *who, const wd_seq_rows_t *q) {
  if (!q) { set_error("%s: null argument", who); return WD_ERR_INVALID; }
  if (q->rows < 0 || q->nseq < 0 || q->vocab < 1) { set_error("%s: bad sizes (rows %lld, sequences %lld, vocab %lld)", who, (long long)q->rows, (long long)q->nseq, (long long)q->vocab); return WD_ERR_INVALID; }
  if (q->dtype != WD_T_F32 && q->dtype != WD_T_F16 && q->dtype != WD_T_BF16) { set_error("%s: bad element type %d", who, q->dtype); return WD_ERR_INVALID; }
  if (q->vocab > INT32_MAX / 2 || q->rows > INT32_MAX / 2 || q->nseq > INT32_MAX / 4) { set_error("%s: more than 2^30 rows or items or 2^29 sequences", who); return WD_ERR_UNSUPPORTED; }
  if (q->ld < q->vocab) { set_error("%s: row stride %lld below the row length %lld", who, (long long)q->ld, (long long)q->vocab); return WD_ERR_INVALID; }
  if (!q->seq_offs || (q->rows > 0 && (!q->logits || !q->targets))) { set_error("%s: null pointer", who); return WD_ERR_INVALID; }
  const int size = q->dtype == WD_T_F32 ? 4 : 2;
  if ((uintptr_t)q->logits % size) { set_error("%s: logits not aligned to their element size", who); return WD_ERR_INVALID; }
  return WD_OK;
}

// whether a row of one of two matrices of `rows` rows of `w` bytes, `s` and `t` bytes apart, meets a row of the other without their being the
// same matrix.  Rows of either between the other's (s == t, a wider buffer of both) are apart.
bool meet(const void *a, int64_t s, const void *b, int64_t t, int64_t rows, int64_t w) {
  int64_t d = (int64_t)((uintptr_t)b - (uintptr_t)a);
  if (rows < 1 || (d == 0 && (s == t || rows == 1)) || d >= (rows - 1) * s + w || -d >= (rows - 1) * t + w) return false;
  if (s == t) {
    const int64_t k = d >= 0 ? d / s : -((-d + s - 1) / s), off = d - k * s;      // row i of b begins `off` behind row i + k of a
    return (k > -rows && k < rows && off < w) || (k + 1 > -rows && k + 1 < rows && s - off < w);
  }
  for (int64_t i = 0, j = 0; i < rows && j < rows;) {      // both ascend
    const int64_t x = i * s, y = d + j * t;
    if (x < y + w && y < x + w) return true;
    if (x < y) ++i;
    else ++j;
  }
  return false;
}
int check_gradient(const char *who, const wd_seq_rows_t &q, const void *dlogits, int64_t ld) {
  const int64_t size = q.dtype == WD_T_F32 ? 4 : 2;
  if (!dlogits) return WD_OK;
  if (ld < q.vocab) { set_error("%s: row stride of the gradient below the row length", who); return WD_ERR_INVALID; }
  if ((uintptr_t)dlogits % size) { set_error("%s: gradient not aligned to its element size", who); return WD_ERR_INVALID; }
  if (meet(q.logits, q.ld * size, dlogits, ld * size, q.rows, q.vocab * size)) { set_error("%s: the gradient shares memory with the logits without being in their place", who); return WD_ERR_INVALID; }
  return WD_OK;
}

int words(const wd_seq_rows_t &q) { return (int)(q.vocab / (q.dtype == WD_T_F32 ? 4 : 8)); }      // whole words of a row, at most

// parts of a row: two workgroups for every CU where there are few rows, at least 4 KB each; a power of two up to a wavefront of them
int row_split(const wd_seq_rows_t &q) {
  int n = 1;
  while (n < kWave && q.rows * n < 2 * kCUs && words(q) >= 512 * n) n *= 2;
  return n;
}
// parts of a row for the gradient pass, 16 KB each: a lane has four words in flight
int grad_split(const wd_seq_rows_t &q) { return words(q) <= 1024 ? 1 : (int)ceil_div(words(q), 1024); }

// where every part finds its row's coefficient: parts of 64 KB, which make little of that; of 16 KB where there are few rows
int self_split(const wd_seq_rows_t &q) {
  const int most = grad_split(q);
  int gs = (int)ceil_div(most, 4);
  if (q.rows > 0 && gs < ceil_div(2 * kCUs, q.rows)) gs = (int)(ceil_div(2 * kCUs, q.rows) < most ? ceil_div(2 * kCUs, q.rows) : most);
  return gs;
}

// whether the rows of a preference loss find their pair themselves: a launch less, for a sum over the pair by every wavefront.  us a call with
// and without: 1000 x 2000 in 64 sequences 13.5 / 16.4, 2000 x 30000 in 2 54 / 73, 2000 x 2000 in 4 18.2 / 15.6, 1000 x 300 in 200 24 / 16.4
bool self_pairs(const wd_seq_rows_t &q) {
  return q.nseq <= kPairSeqs && (q.rows <= kPairRows / 2 || (q.rows <= kPairRows && words(q) >= 2048));
}
// whether the rows of a policy loss find weight and advantage themselves: a launch less, for a look at every target by every wavefront.  us a call
// with and without, 16 sequences: sum, 12000 x 300 14.8 / 17.4, 3000 x 50000 106 / 108; a mean over actions, 1000 x 8000 14.8 / 17.4,
// 988 x 50021 43 / 37; over sequences, 1000 x 4000 14.8 / 17.3, 1000 x 8000 22 / 17.5, with 250 of them 1000 x 2000 18.8 / 17.4
bool self_weights(const wd_seq_rows_t &q, int reduction) {
  if (q.nseq > kSelfSeqs) return false;
  if (reduction == WD_POLICY_SUM || q.rows <= kSelfRows) return true;
  if (reduction == WD_POLICY_TOKEN_MEAN) return q.rows <= kWeightRows && q.rows * q.vocab <= 8 << 20;
  return q.rows <= kWeightRows && q.rows * q.vocab <= 4 << 20 && q.nseq <= kWave;
}

bool tiny(const wd_seq_rows_t &q) { return q.rows <= Tiny::kRows && q.nseq <= Tiny::kRows && q.rows * q.vocab <= 65536; }
unsigned tiny_grid(const wd_seq_rows_t &q, const void *dlogits, int64_t ldg) {
  const uintptr_t z = (uintptr_t)q.logits, g = (uintptr_t)dlogits;
  const int64_t size = q.dtype == WD_T_F32 ? 4 : 2, nz = ((q.rows - 1) * q.ld + q.vocab) * size, ng = ((q.rows - 1) * ldg + q.vocab) * size;
  if (!dlogits || q.rows < 1 || (z < g + ng && g < z + nz)) return 1;
  return (unsigned)ceil_div(q.rows * tiny_grad_parts(q.rows, words(q)), Tiny::kWaves);
}
// whole words of the longest row that a workgroup holds in registers: 1024 lanes x 16
constexpr int kResidentWords = 16384;

dim3 row_grid(int64_t rows, int parts) {
  const int64_t y = rows < 32768 ? rows : 32768;
  return dim3((unsigned)parts, (unsigned)y, (unsigned)ceil_div(rows, y));
}

struct Work {      // [rows * nsplit] (m, s) parts | [rows] (m, s) | [rows] picked logits, coefficients | 3 [rows] | [rows] weights, advantages | counts
  float2 *part, *stat;
  float *pick, *coef, *rows3, *w, *adv;
  int32_t *cnt;
  Work(const wd_seq_rows_t &q, float *p) {
    const int64_t T = q.rows;
    part = (float2 *)p;
    stat = part + T * row_split(q);
    pick = (float *)(stat + T);
    coef = pick + T;
    rows3 = coef + T;
    w = rows3 + 3 * T;
    adv = w + T;
    cnt = (int32_t *)(adv + T);
  }
  Parts parts(int n) const { return {part, pick, n}; }
};

template <typename F> void by_type(int32_t dtype, F f) {
  if (dtype == WD_T_F32) f(std::integral_constant<int, WD_T_F32>());
  else if (dtype == WD_T_F16) f(std::integral_constant<int, WD_T_F16>());
  else f(std::integral_constant<int, WD_T_BF16>());
}

// rows below 8 KB, which are never split: four to a workgroup, a wavefront each
bool short_rows(const wd_seq_rows_t &q) { return words(q) < 512; }
// more logits than the last cache (256 MB) holds
bool beyond_cache(const wd_seq_rows_t &q) { return q.rows * q.ld * (q.dtype == WD_T_F32 ? 4 : 2) > ((int64_t)256 << 20); }

// `again`: another pass reads the logits afterwards
void launch_stats(const wd_seq_rows_t &q, int nsplit, const Work &k, float *token, bool again, hipStream_t st) {
  if (q.rows < 1) return;
  by_type(q.dtype, [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    const dim3 grid = row_grid(q.rows, nsplit);
    if (short_rows(q)) k_row_stats<DT, kWave, false><<<row_grid(ceil_div(q.rows, 4), 1), 256, 0, st>>>(q, 1, k.part, k.pick, k.stat, token);
    else if (!again && beyond_cache(q)) k_row_stats<DT, 256, true><<<grid, 256, 0, st>>>(q, nsplit, k.part, k.pick, k.stat, token);
    else k_row_stats<DT, 256, false><<<grid, 256, 0, st>>>(q, nsplit, k.part, k.pick, k.stat, token);
  });
}
// the gradient is the last to read the logits: 1.14 GB 489 -> 448 us past the cache, 61 MB 33 -> 36 us
template <int DT>
void launch_grad(const wd_seq_rows_t &q, int64_t rows, void *dlogits, int64_t ldg, int32_t zero_tail, const Work &k, const float *pair_loss,
                 const float *weights, double scale, float *loss, hipStream_t st) {
  wd_seq_rows_t last = q;
  last.rows = rows;
  const int gs = grad_split(q);
  const dim3 grid = row_grid(rows + (loss ? 1 : 0), gs);
  if (short_rows(q))
    k_logits_grad<DT, kWave, false><<<row_grid(ceil_div(rows, 4) + (loss ? 1 : 0), 1), 256, 0, st>>>(last, dlogits, ldg, zero_tail, 1, k.stat, k.coef, pair_loss, weights, scale, loss);
  else if (beyond_cache(q))
    k_logits_grad<DT, 256, true><<<grid, 256, 0, st>>>(last, dlogits, ldg, zero_tail, gs, k.stat, k.coef, pair_loss, weights, scale, loss);
  else
    k_logits_grad<DT, 256, false><<<grid, 256, 0, st>>>(last, dlogits, ldg, zero_tail, gs, k.stat, k.coef, pair_loss, weights, scale, loss);
}

// A row in the registers of a workgroup, NV words a lane.  Two or more workgroups have to fit on a CU, so that one loads or stores while
// another adds up, and no lane should hold many words it has not got: measured on bf16 rows, 0.8 GB in and out, TB/s:
//   words 125 (0.4 GB)  64 x 2 2.84, 128 x 1 2.25, 256 x 1 1.56      250   128 x 2 3.77, 64 x 4 3.70, 256 x 1 2.78
//   1000  512 x 2 4.76, 256 x 4 4.57, 1024 x 1 3.11     2000  512 x 4 5.14, 256 x 8 4.89, 1024 x 2 4.68
//   4000  1024 x 4 5.28, 512 x 8 4.97, 256 x 16 4.89    8000  512 x 16 4.94, 256 x 32 4.79, 1024 x 8 4.15
//   12500 512 x 25 4.49 (128 registers), 4.22 (151), 1024 x 13 4.12        16375 1024 x 16 4.08, 512 x 32 3.99
template <int DT, int TH, int... NV>
bool launch_resident_of(int nw, const wd_seq_rows_t &q, const wd_policy_t &o, const Work &k, hipStream_t st) {
  bool done = false;
  ((done || nw > TH * NV ? (void)0
                         : (k_policy_resident<DT, TH, NV><<<row_grid(q.rows, 1), TH, 0, st>>>(q, o, k.w, k.adv, k.cnt, k.rows3), (void)(done = true))),
   ...);
  return done;
}
template <int DT> bool launch_resident(const wd_seq_rows_t &q, const wd_policy_t &o, const Work &k, hipStream_t st) {
  const int nw = words(q);
  if (nw <= 128) return launch_resident_of<DT, 64, 1, 2>(nw, q, o, k, st);
  if (nw <= 512) return launch_resident_of<DT, 128, 2, 3, 4>(nw, q, o, k, st);
  if (nw <= 2048) return launch_resident_of<DT, 512, 2, 3, 4>(nw, q, o, k, st);
  if (nw <= 4096) return launch_resident_of<DT, 1024, 3, 4>(nw, q, o, k, st);
  if (nw <= 12800) return launch_resident_of<DT, 512, 9, 10, 11, 12, 13, 14, 16, 18, 20, 22, 25>(nw, q, o, k, st);
  return nw <= kResidentWords && launch_resident_of<DT, 1024, 14, 16>(nw, q, o, k, st);
}

}  // namespace

extern "C" int64_t wd_policy_workspace_floats(const wd_seq_rows_t *rows) {
  const int rc = check_rows(__func__, rows);
  if (rc) return rc;
  return rows->rows * (2 * (int64_t)row_split(*rows) + 2 + 1 + 1 + 3 + 1 + 1) + rows->nseq + 1;
}

extern "C" int wd_seq_logp(const wd_seq_rows_t *rows, int32_t length_norm, float *token_logp, float *seq_logp, float *ws,
                           wd_stream_t stream) {
  if (const int rc = check_rows(__func__, rows)) return rc;
  const wd_seq_rows_t q = *rows;
  WD_REQUIRE((token_logp || !q.rows) && (seq_logp || !q.nseq) && ws, "null pointer");
  hipStream_t st = as_stream(stream);
  if (tiny(q)) {
    by_type(q.dtype, [&](auto dt) { k_seq_tiny<decltype(dt)::value><<<1, 1024, 0, st>>>(q, length_norm, token_logp, seq_logp); });
    return check_launch(__func__);
  }
  const Work k(q, ws);
  const int ns = row_split(q);
  launch_stats(q, ns, k, token_logp, false, st);
  if (q.nseq > 0) k_seq_logp<<<row_grid(q.nseq, 1), 256, 0, st>>>(q, k.parts(ns), length_norm, k.stat, token_logp, seq_logp);
  return check_launch(__func__);
}

extern "C" int wd_pref_loss_fwd_bwd(const wd_seq_rows_t *rows, const wd_pref_t *opts, float *ws, wd_stream_t stream) {
  if (const int rc = check_rows(__func__, rows)) return rc;
  WD_REQUIRE(opts && ws, "null argument");
  const wd_seq_rows_t q = *rows;
  const wd_pref_t o = *opts;
  WD_REQUIRE(q.nseq % 2 == 0, "an odd number of sequences: pair i is sequences 2i (chosen) and 2i + 1 (rejected)");
  WD_REQUIRE(o.kind == WD_PREF_LOGISTIC || o.kind == WD_PREF_SQUARE, "bad loss kind");
  WD_REQUIRE(o.beta > 0.f, "beta must be positive");
  WD_REQUIRE(o.label_smoothing >= 0.f && o.label_smoothing < 0.5f, "label_smoothing must be in [0, 0.5)");
  WD_REQUIRE(o.kind == WD_PREF_LOGISTIC || (o.label_smoothing == 0.f && o.margin == 0.f), "label_smoothing and margin belong to the logistic loss");
  WD_REQUIRE(o.loss && (q.nseq == 0 || (o.pair_loss && o.difference && o.seq_logp)) && (q.rows == 0 || o.token_logp), "null output");
  if (const int rc = check_gradient(__func__, q, o.dlogits, o.ld_dlogits)) return rc;
  hipStream_t st = as_stream(stream);
  const Work k(q, ws);
  const int ns = row_split(q);
  if (tiny(q)) {
    by_type(q.dtype, [&](auto dt) { k_pref_tiny<decltype(dt)::value><<<tiny_grid(q, o.dlogits, o.ld_dlogits), 1024, 0, st>>>(q, o); });
    return check_launch(__func__);
  }
  launch_stats(q, ns, k, o.token_logp, o.dlogits != nullptr, st);
  by_type(q.dtype, [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    if (self_pairs(q)) {
      const int gs = self_split(q);
      k_pref_grad<DT><<<row_grid(q.rows + 1, gs), 256, 0, st>>>(q, o, gs, k.parts(ns), k.stat);
      return;
    }
    if (q.nseq > 0) k_pref_pairs<<<row_grid(q.nseq / 2, 1), 256, 0, st>>>(q, o, k.parts(ns), k.stat, k.coef);
    launch_grad<DT>(q, o.dlogits ? q.rows : 0, o.dlogits, o.ld_dlogits, o.zero_tail, k, o.pair_loss, o.weights, (double)o.scale, o.loss, st);
  });
  return check_launch(__func__);
}

extern "C" int wd_policy_loss_fwd_bwd(const wd_seq_rows_t *rows, const wd_policy_t *opts, float *ws, wd_stream_t stream) {
  if (const int rc = check_rows(__func__, rows)) return rc;
  WD_REQUIRE(opts && ws, "null argument");
  const wd_seq_rows_t q = *rows;
  const wd_policy_t o = *opts;
  WD_REQUIRE(o.reduction == WD_POLICY_SUM || o.reduction == WD_POLICY_TOKEN_MEAN || o.reduction == WD_POLICY_SEQUENCE_MEAN, "bad reduction");
  WD_REQUIRE(o.clip_low >= 0.f && o.clip_low <= 1.f && o.clip_high >= 0.f, "clip range: low in [0, 1], high >= 0");
  WD_REQUIRE(o.kl_coef == 0.f || o.ref_logp || q.rows == 0, "a KL term needs the reference policy's log-probabilities");
  WD_REQUIRE(o.sums && (q.rows == 0 || (o.old_logp && o.token_logp)) && (o.advantages || (o.adv_per_row ? q.rows : q.nseq) == 0), "null pointer");
  if (const int rc = check_gradient(__func__, q, o.dlogits, o.ld_dlogits)) return rc;
  hipStream_t st = as_stream(stream);
  if (tiny(q)) {
    by_type(q.dtype, [&](auto dt) { k_policy_tiny<decltype(dt)::value><<<tiny_grid(q, o.dlogits, o.ld_dlogits), 1024, 0, st>>>(q, o); });
    return check_launch(__func__);
  }
  Work k(q, ws);
  if (self_weights(q, o.reduction)) k.w = nullptr;
  else if (q.nseq > 0) {
    if (q.rows < 256 * q.nseq) k_policy_rows<256><<<row_grid(q.nseq, 1), 256, 0, st>>>(q, o, k.w, k.adv, k.cnt);
    else k_policy_rows<1024><<<row_grid(q.nseq, 1), 1024, 0, st>>>(q, o, k.w, k.adv, k.cnt);
    if (q.nseq > kCountSeqs && o.reduction != WD_POLICY_SUM) k_policy_total<<<1, 1024, 0, st>>>(q, o, k.cnt);
  }
  if (q.rows > 0) {
    by_type(q.dtype, [&](auto dt) {
      constexpr int DT = decltype(dt)::value;
      if (!launch_resident<DT>(q, o, k, st)) {
        const int ns = row_split(q);
        launch_stats(q, ns, k, o.token_logp, o.dlogits != nullptr, st);
        if (!k.w) {
          const int gs = self_split(q);
          const dim3 grid = row_grid(q.rows, o.dlogits ? gs : 1);
          if (!o.dlogits) k_policy_grad<DT, false, false><<<grid, 256, 0, st>>>(q, o, 1, k.parts(ns), k.stat, k.rows3);
          else if (beyond_cache(q)) k_policy_grad<DT, true, true><<<grid, 256, 0, st>>>(q, o, gs, k.parts(ns), k.stat, k.rows3);
          else k_policy_grad<DT, true, false><<<grid, 256, 0, st>>>(q, o, gs, k.parts(ns), k.stat, k.rows3);
          return;
        }
        k_policy_join<<<dim3((unsigned)ceil_div(q.rows * ns, 256)), 256, 0, st>>>(q, o, k.parts(ns), k.w, k.adv, k.cnt, k.stat, k.coef, k.rows3);
        if (o.dlogits) launch_grad<DT>(q, q.rows, o.dlogits, o.ld_dlogits, o.zero_tail, k, nullptr, nullptr, 0.0, nullptr, st);
      }
    });
  }
  k_policy_sums<<<3, 1024, 0, st>>>(k.rows3, q.rows, o.sums);
  return check_launch(__func__);
}
