// Log probabilities of tokens under rows of logits, and the clipped policy loss on them, with the
// gradients to the logits (muon_token_logprobs, muon_policy_loss and their backward passes).
//
// For a row x of V logits, its token t and the temperature tau:
//   m = max x,  s = sum exp((x - m) / tau),  logp = (x_t - m) / tau - log s.
// With r = exp(logp - old), advantage A, weight w and the reference's log probability ref:
//   term = -min(r A, clip(r, 1 - lo, 1 + hi) A) + beta (exp(ref - logp) - (ref - logp) - 1)
//   loss = sum over rows of w term,  g = w d term / d logp.
// The gradient of g logp: dx_v = g / tau ([v = t] - exp((x_v - m) / tau) / s).
//
// A row with weight 0, or a negative token, is left out: nothing of it is read, logp is 0 and its
// gradient 0. A token of V or more gives NaN.
//
// Every pass is bound by memory, or nearly: 8192 rows of 128000 bf16 logits are read in 335 us,
// 6.3 TB/s, and the gradient of 4096 such rows is made in 381 us, 5.5 TB/s. The policy loss reads its
// logits once for loss and gradient: 6144 rows of 128000, a quarter of them left out, 510 us,
// 5.4 TB/s, where a copy of 2 GiB moves 5.0 and a second reading would add 190 us.
// Sums and exponentials are fp32 with the row's maximum taken off first, logp is formed in
// double, gradients are rounded once at the store.
#include <algorithm>

#include "logits.h"

namespace {

struct Rows {
  const void* x;
  int64_t stride;  // between rows, in elements
  int64_t N, V;
  const int64_t* tokens;
  float k;     // log2(e) / tau
  double tau_inv;
  float* logp;
  float* stats;  // per row m, then per row 1 / s (null: not kept)
};

// The policy loss's per-row inputs; weights null: plain log probabilities.
struct Policy {
  const float* old;
  const float* adv;
  const float* weights;
  const float* ref;  // or null
  float lo, hi, beta;
  float* terms;  // w term per row
  float* coef;   // g per row (two-pass form)
};

// A row's own inputs: the token and weight, which say whether its logits are read, and the rest,
// loaded behind the row's logits by the wave that will need it. Loaded after the row's sum, one
// is waited for behind the other (4096 rows of 50257: 189 us instead of 181), before the logits,
// they wait for it (6144 rows of 128000: 533 us instead of 511).
struct RowIn {
  int64_t tok;
  float w, old, adv, ref, xt;
  // left out: nothing of the row's logits is read
  MUON_DEVICE bool out() const { return tok < 0 || w == 0.0f; }
};
MUON_DEVICE RowIn first_of_row(const Rows& a, const Policy& p, int64_t row) {
  return {a.tokens[row], p.weights ? p.weights[row] : 1.0f, 0.0f, 0.0f, 0.0f, 0.0f};
}
template <int DT>
MUON_DEVICE void rest_of_row(RowIn& r, const Rows& a, const Policy& p, int64_t row) {
  if (p.weights) {
    r.old = p.old[row];
    r.adv = p.adv[row];
    if (p.ref) r.ref = p.ref[row];
  }
  if (r.tok < a.V) r.xt = Elem<DT>::load(a.x, row * a.stride + r.tok);
}

// A running maximum and the sum of exp((x - m) / tau) under it.
struct Sum {
  float m, s;
};
// exp2 of -inf - -inf would be NaN: against a maximum of -inf the sum is 0 whatever is added.
MUON_DEVICE float base_of(float m) { return m == -INFINITY ? 0.0f : m; }
MUON_DEVICE Sum join(Sum a, Sum b, float k) {
  Sum r;
  r.m = fmaxf(a.m, b.m);
  const float base = base_of(r.m);
  r.s = a.s * __builtin_amdgcn_exp2f((a.m - base) * k) + b.s * __builtin_amdgcn_exp2f((b.m - base) * k);
  return r;
}
template <int N>
MUON_DEVICE void add_values(Sum& a, const float (&v)[N], float k) {
  float m = a.m;
#pragma unroll
  for (int e = 0; e < N; ++e) m = fmaxf(m, v[e]);
  const float base = base_of(m);
  float s = 0.0f;
#pragma unroll
  for (int e = 0; e < N; ++e) s += __builtin_amdgcn_exp2f((v[e] - base) * k);
  a.s = a.s * __builtin_amdgcn_exp2f((a.m - base) * k) + s;
  a.m = m;
}

MUON_DEVICE Sum first_lane(Sum v) {
  return {__int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(v.m))),
          __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(v.s)))};
}

// Joined over a workgroup of NT threads in a fixed order; the result in every thread.
template <int NT>
MUON_DEVICE Sum block_join(Sum v, float k, Sum* lds) {
  auto op = [k](Sum a, Sum b) { return join(a, b, k); };
  v = group_reduce<64>(v, op);
  // the two operands' order decides the last bit: every lane takes the first one's
  if constexpr (NT == 64) return first_lane(v);
  if (threadIdx.x % 64 == 0) lds[threadIdx.x / 64] = v;
  __syncthreads();
  return first_lane(group_reduce<NT / 64>(lds[threadIdx.x % (NT / 64)], op));
}

// log s for s in 1..2^31 (s is 0, infinite or NaN where a row has no sum), to 2^-24 of one: the
// hardware's logarithm of the fraction beside the whole exponent, which a single fp32 result
// would round away.
MUON_DEVICE double log_of(float s) {
  constexpr double LN2_D = 0.69314718055994530942;
  if (!(s > 0.0f && s < INFINITY)) return s == 0.0f ? -INFINITY : s;
  return LN2_D * ((double)__builtin_amdgcn_frexp_expf(s) +
                  (double)__builtin_amdgcn_logf(__builtin_amdgcn_frexp_mantf(s)));
}
MUON_DEVICE float exp_of(double x) { return __builtin_amdgcn_exp2f((float)(x * LOG2E_D)); }

// exp(d) - d - 1, which is never negative, and its derivative, to a few roundings of their own size.
// Below |d| = 1 the exponential is nearly all of what is taken off it: there the series
// d^2 (1/2 + d (1/6 + ...)), whose first term left out, d^11 / 11!, is below 2^-23 of the sum.
struct Beyond {
  float value, slope;
};
MUON_DEVICE Beyond exp_beyond(float d) {
  if (!(fabsf(d) < 1.0f)) {
    const float e = exp_of((double)d);
    return {e - d - 1.0f, e - 1.0f};
  }
  float s = 1.0f / 3628800.0f;
  s = fmaf(s, d, 1.0f / 362880.0f);
  s = fmaf(s, d, 1.0f / 40320.0f);
  s = fmaf(s, d, 1.0f / 5040.0f);
  s = fmaf(s, d, 1.0f / 720.0f);
  s = fmaf(s, d, 1.0f / 120.0f);
  s = fmaf(s, d, 1.0f / 24.0f);
  s = fmaf(s, d, 1.0f / 6.0f);
  s = fmaf(s, d, 0.5f);
  s *= d * d;
  return {s, d + s};
}

// What a row's sum gives: logp, and for the policy loss its term and slope g. One thread, while
// its workgroup waits: the differences of log probabilities, which cancel, in double, and functions
// of what is left in fp32 (with double exponentials the loss on 128000 values a row took 8% longer).
MUON_DEVICE float finish_row(const Rows& a, const Policy& p, int64_t row, const RowIn& in, Sum t) {
  const int64_t tok = in.tok;
  double logp = __builtin_nan("");
  if (tok < a.V) logp = ((double)in.xt - (double)t.m) * a.tau_inv - log_of(t.s);
  a.logp[row] = (float)logp;
  if (a.stats) {
    a.stats[row] = t.m;
    a.stats[a.N + row] = tok < a.V ? 1.0f / t.s : __int_as_float(0x7fc00000);
  }
  if (!p.weights) return 0.0f;
  const float w = in.w, A = in.adv, r = exp_of(logp - (double)in.old);
  const float low = 1.0f - p.lo, high = 1.0f + p.hi;
  // NaN ratios stay NaN: comparisons below leave r in place
  const float clipped = r < low ? low : r > high ? high : r;
  const float plain = r * A, other = clipped * A;
  float term = -(other < plain ? other : plain);
  // the smaller one is r A where r is inside, or outside on the side that A pulls it back from
  const bool cut = A >= 0.0f ? r > high : r < low;
  float slope = cut ? 0.0f : -plain;
  if (p.ref) {
    const float ahead = (float)((double)in.ref - logp);
    const Beyond kl = exp_beyond(ahead);
    term += p.beta * kl.value;
    slope -= p.beta * kl.slope;
  }
  p.terms[row] = w * term;
  const float g = w * slope;
  if (p.coef) p.coef[row] = g;
  return g;
}

MUON_DEVICE void skip_row(const Rows& a, const Policy& p, int64_t row) {
  a.logp[row] = 0.0f;
  if (a.stats) a.stats[row] = a.stats[a.N + row] = 0.0f;
  if (p.weights) {
    p.terms[row] = 0.0f;
    if (p.coef) p.coef[row] = 0.0f;
  }
}

constexpr int SUM_UNROLL = 4;  // 16-byte loads in flight per thread

// One pass over (a slice of) a row with a running maximum and sum. Grid: slices x rows; with
// one slice a row the workgroup finishes its row, else it leaves (m, s) for logp_join_kernel.
template <int DT, int NT>
__global__ __launch_bounds__(NT) void logp_kernel(Rows a, Policy p, Sum* part) {
  constexpr int N = Vec16<DT>::N;
  __shared__ Sum lds[NT / 64];
  const int slices = gridDim.x;
  for (int64_t row = blockIdx.y; row < a.N; row += gridDim.y) {
    RowIn in = first_of_row(a, p, row);
    if (in.out()) {
      if (threadIdx.x == 0 && slices == 1) skip_row(a, p, row);
      continue;
    }
    if (threadIdx.x < 64 && slices == 1) rest_of_row<DT>(in, a, p, row);
    const int64_t at = row * a.stride;
    const int64_t vecs = a.V / N;
    const int64_t begin = vecs * blockIdx.x / slices, end = vecs * (blockIdx.x + 1) / slices;
    Sum t = {-INFINITY, 0.0f};
    int64_t i = begin + threadIdx.x;
    for (; i + (SUM_UNROLL - 1) * NT < end; i += SUM_UNROLL * NT) {
      muon_u4 w[SUM_UNROLL];
#pragma unroll
      for (int u = 0; u < SUM_UNROLL; ++u) w[u] = load_u4(elem_at<DT>(a.x, at + (i + u * NT) * N));
      float v[SUM_UNROLL * N];
#pragma unroll
      for (int u = 0; u < SUM_UNROLL; ++u) {
        float h[N];
        Vec16<DT>::unpack(w[u], h);
#pragma unroll
        for (int e = 0; e < N; ++e) v[u * N + e] = h[e];
      }
      add_values(t, v, a.k);
    }
    for (; i < end; i += NT) {
      float v[N];
      Vec16<DT>::unpack(load_u4(elem_at<DT>(a.x, at + i * N)), v);
      add_values(t, v, a.k);
    }
    if (blockIdx.x == slices - 1 && threadIdx.x < a.V - vecs * N) {
      const float v[1] = {Elem<DT>::load(a.x, at + vecs * N + threadIdx.x)};
      add_values(t, v, a.k);
    }
    t = block_join<NT>(t, a.k, lds);
    if (threadIdx.x == 0) {
      if (slices == 1) finish_row(a, p, row, in, t);
      else part[row * slices + blockIdx.x] = t;
    }
    __syncthreads();  // lds is written again for the next row
  }
}

// A wave a row: the slices' sums joined in a fixed order.
template <int DT>
__global__ __launch_bounds__(256) void logp_join_kernel(Rows a, Policy p, const Sum* part, int slices) {
  const int64_t row = (int64_t)blockIdx.x * 4 + threadIdx.x / 64;
  if (row >= a.N) return;
  const int lane = threadIdx.x % 64;
  RowIn in = first_of_row(a, p, row);
  if (in.out()) {
    if (lane == 0) skip_row(a, p, row);
    return;
  }
  rest_of_row<DT>(in, a, p, row);
  Sum t = {-INFINITY, 0.0f};
  for (int i = lane; i < slices; i += 64) t = join(t, part[row * slices + i], a.k);
  t = group_reduce<64>(t, [&](Sum x, Sum y) { return join(x, y, a.k); });
  if (lane == 0) finish_row(a, p, row, in, t);
}

// The policy loss with its gradient in one pass over the logits: a workgroup holds its whole row
// in registers (NV 16-byte pieces a thread; the 512 KB of a CU hold 163840 bf16 values beside
// the working registers), sums it, makes the slope g, and writes the gradient from the same
// registers. A CU works on one long row at a time, so what its waves compute between reading and
// writing counts: with two thirds of the instructions the launch above went from 585 to
// 505 us.
template <int DT, int NT, int NV, bool STREAM>
__global__ __launch_bounds__(NT) void policy_row_kernel(Rows a, Policy p, void* dx, int64_t row0) {
  constexpr int N = Vec16<DT>::N;
  __shared__ Sum lds[NT / 64];
  __shared__ float slope;
  const int64_t row = row0 + blockIdx.x;
  const int64_t at = row * a.stride, to = row * a.V;
  const int V = (int)a.V, vecs = V / N;
  // one address register a thread: the pieces' places are added to the scalar base
  const char* xr = elem_at<DT>(a.x, at);
  char* dr = (char*)elem_at<DT>(dx, to);
  const uint32_t off = threadIdx.x * 16;
  const int tid = threadIdx.x;
  RowIn in = first_of_row(a, p, row);
  if (in.out()) {
    if (tid == 0) skip_row(a, p, row);
#pragma unroll
    for (int u = 0; u < NV; ++u) {
      const int i = u * NT + tid;
      if (i < vecs) put<STREAM>(dr + (int64_t)u * NT * 16 + off, muon_u4{0, 0, 0, 0});
      else if (i == vecs) {
        const float z[N] = {};
        store_tail<DT>(dx, to, (int64_t)i * N, V, z);
      }
    }
    return;
  }
  muon_u4 w[NV];
#pragma unroll
  for (int u = 0; u < NV; ++u) {
    if ((u + 1) * NT <= vecs) {
      w[u] = load_u4(xr + (int64_t)u * NT * 16 + off);
    } else {  // the piece that the row's end cuts, and pieces behind it
      const int i = u * NT + tid;
      const uint32_t none = DT == MUON_DT_F32 ? 0xff800000u : 0xff80ff80u;  // -inf
      w[u] = muon_u4{none, none, none, none};
      if (i < vecs) w[u] = load_u4(xr + (int64_t)u * NT * 16 + off);
      else if (i == vecs) w[u] = load_tail<DT>(a.x, at, (int64_t)i * N, V);
    }
  }
  if (tid < 64) rest_of_row<DT>(in, a, p, row);
  Sum t = {-INFINITY, 0.0f};
  // few pieces unpacked at a time: the row itself takes most of the registers
  constexpr int STEP = NV <= 16 ? 2 : 1;
#pragma unroll
  for (int u = 0; u < NV; u += STEP) {
    float v[STEP * N];
#pragma unroll
    for (int i = 0; i < STEP; ++i) {
      float h[N];
      Vec16<DT>::unpack(w[u + i], h);
#pragma unroll
      for (int e = 0; e < N; ++e) v[i * N + e] = h[e];
    }
    add_values(t, v, a.k);
    __builtin_amdgcn_sched_barrier(0);
  }
  t = block_join<NT>(t, a.k, lds);
  if (tid == 0) slope = finish_row(a, p, row, in, t);
  __syncthreads();
  const bool known = in.tok < a.V;
  const int tok = known ? (int)in.tok : -1;
  const float g = slope * (float)a.tau_inv;
  const float pc = known ? g * (1.0f / t.s) : __int_as_float(0x7fc00000);
#pragma unroll
  for (int u = 0; u < NV; ++u) {
    const int i = u * NT + tid;
    if (u * NT > vecs) break;
    float v[N], d[N];
    // unpacked again: the compiler would else keep the first pass's floats beside the row
    asm("" : "+v"(w[u]));
    Vec16<DT>::unpack(w[u], v);
    slopes<DT>(v, t.m, a.k, pc, g, tok - i * N, d);
    if (i < vecs) put<STREAM>(dr + (int64_t)u * NT * 16 + off, Vec16<DT>::pack(d));
    else if (i == vecs) store_tail<DT>(dx, to, (int64_t)i * N, V, d);
    __builtin_amdgcn_sched_barrier(0);
  }
}

// loss = the rows' terms summed in a fixed order, in double.
__global__ __launch_bounds__(1024) void loss_kernel(const float* terms, int64_t n, float* loss) {
  __shared__ double red[16];
  double s = 0.0;
#pragma unroll 4
  for (int64_t i = threadIdx.x; i < n; i += 1024) s += terms[i];
  for (int off = 32; off; off >>= 1) s += __shfl_xor(s, off, 64);
  if (threadIdx.x % 64 == 0) red[threadIdx.x / 64] = s;
  __syncthreads();
  if (threadIdx.x) return;
  s = 0.0;
  for (int w = 0; w < 16; ++w) s += red[w];
  loss[0] = (float)s;
}

// x *= scale in place; nothing to do where the scale is one.
template <int DT>
__global__ __launch_bounds__(256) void scale_kernel(void* x, int64_t n, const float* scale) {
  constexpr int N = Vec16<DT>::N;
  const float g = scale[0];
  if (g == 1.0f) return;
  const int64_t vecs = n / N, step = (int64_t)gridDim.x * 256;
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  for (int64_t i = id; i < vecs; i += step) {
    float v[N];
    Vec16<DT>::unpack(load_u4(elem_at<DT>(x, i * N)), v);
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] *= g;
    store_u4((void*)elem_at<DT>(x, i * N), Vec16<DT>::pack(v));
  }
  for (int64_t i = vecs * N + id; i < n; i += step) Elem<DT>::store(x, i, Elem<DT>::load(x, i) * g);
}

// Slices of a row. One workgroup a row as a rule: joining slices takes a second launch. Longer
// rows than SPLIT_FROM, of which fewer than 128 come together, are cut until there are four
// workgroups per CU, into slices of at least 8192 values and at most 64 a row. One row, whole and cut (us a call): 32000 values 6.1 and 10.0, 128000 9.0 and
// 10.4, 262144 14.6 and 9.2, 524288 26.1 and 9.7; 64 rows of 262144 values 17.3 and 15.3.
constexpr int64_t SPLIT_FROM = 131072;
int slices_for(int64_t N, int64_t V) {
  if (V <= SPLIT_FROM || N >= 128 || N < 1) return 1;
  return (int)std::min<int64_t>(std::min<int64_t>(1024 / N, V / 8192), 64);
}

// Threads a row: the fewest that give 2^18 in all (four waves per SIMD), with at most 64
// 16-byte pieces each (32 above a wave). 8192 rows of bf16 with 64, 128, 256 and 512 threads:
// 2000 values 12, 14, 20, 40 us, 16000 values 45, 44, 47, 77 us; 4096 rows of 32000 values 42, 46,
// 44, 52 us; 8192 rows of 128000 values with 256 and 512: 348 and 334 us. Fewer rows than CUs take
// 1024 (200 rows of 128000 values 12 us, with 512 15).
template <int DT>
void launch_sums_dt(const Rows& a, const Policy& p, int slices, Sum* part, hipStream_t s) {
  const dim3 grid(slices, (unsigned)std::min(a.N, MAX_GRID_Y));
  const int64_t vecs = a.V / Vec16<DT>::N;
  int threads = vecs <= 64 * 64 ? 64 : vecs <= 32 * 128 ? 128 : vecs <= 32 * 256 ? 256 : 512;
  while (threads < 512 && a.N * threads < (1 << 18) && 2 * threads <= vecs) threads *= 2;
  if (threads == 512 && slices == 1 && a.N <= 256 && vecs >= 2048) threads = 1024;
  if (threads == 64) logp_kernel<DT, 64><<<grid, 64, 0, s>>>(a, p, part);
  else if (threads == 128) logp_kernel<DT, 128><<<grid, 128, 0, s>>>(a, p, part);
  else if (threads == 256) logp_kernel<DT, 256><<<grid, 256, 0, s>>>(a, p, part);
  else if (threads == 512) logp_kernel<DT, 512><<<grid, 512, 0, s>>>(a, p, part);
  else logp_kernel<DT, 1024><<<grid, 1024, 0, s>>>(a, p, part);
}

int launch_sums(const Rows& a, const Policy& p, int dtype, void* ws, hipStream_t s) {
  const int slices = slices_for(a.N, a.V);
  Sum* part = (Sum*)ws;
  if (dtype == MUON_DT_F32) launch_sums_dt<MUON_DT_F32>(a, p, slices, part, s);
  else if (dtype == MUON_DT_BF16) launch_sums_dt<MUON_DT_BF16>(a, p, slices, part, s);
  else launch_sums_dt<MUON_DT_F16>(a, p, slices, part, s);
  MUON_CHECK_LAUNCH("token_logprobs");
  if (slices == 1) return MUON_OK;
  const unsigned blocks = (unsigned)((a.N + 3) / 4);
  if (dtype == MUON_DT_F32) logp_join_kernel<MUON_DT_F32><<<blocks, 256, 0, s>>>(a, p, part, slices);
  else if (dtype == MUON_DT_BF16) logp_join_kernel<MUON_DT_BF16><<<blocks, 256, 0, s>>>(a, p, part, slices);
  else logp_join_kernel<MUON_DT_F16><<<blocks, 256, 0, s>>>(a, p, part, slices);
  MUON_CHECK_LAUNCH("token_logprobs join");
  return MUON_OK;
}

template <int DT>
int launch_policy_rows(const Rows& a, const Policy& p, void* dx, hipStream_t s) {
  const int64_t vecs = (a.V + Vec16<DT>::N - 1) / Vec16<DT>::N;
  const bool stream = a.N * a.V * (DT == MUON_DT_F32 ? 4 : 2) >= STREAM_FROM;
#define MUON_POLICY_ROWS(NT, NV)                                      \
  if (vecs <= (int64_t)NT * NV) {                                     \
    /* a launch holds fewer than 2^32 threads */                      \
    for (int64_t r = 0; r < a.N; r += 1 << 20) {                      \
      const unsigned rows = (unsigned)std::min<int64_t>(a.N - r, 1 << 20); \
      if (stream) policy_row_kernel<DT, NT, NV, true><<<rows, NT, 0, s>>>(a, p, dx, r); \
      else policy_row_kernel<DT, NT, NV, false><<<rows, NT, 0, s>>>(a, p, dx, r); \
      MUON_CHECK_LAUNCH("policy_loss");                               \
    }                                                                 \
    return MUON_OK;                                                   \
  }
  MUON_POLICY_ROWS(256, 2)
  MUON_POLICY_ROWS(256, 4)
  MUON_POLICY_ROWS(512, 4)
  MUON_POLICY_ROWS(512, 8)
  MUON_POLICY_ROWS(1024, 8)
  MUON_POLICY_ROWS(1024, 12)
  MUON_POLICY_ROWS(1024, 16)
  MUON_POLICY_ROWS(1024, 20)
#undef MUON_POLICY_ROWS
  muon_set_error("policy_loss: a row of %lld values does not fit the registers", (long long)a.V);
  return MUON_ERR_SHAPE;
}

}  // namespace

extern "C" {

int64_t muon_token_logprobs_workspace_bytes(int dtype, int64_t rows, int64_t vocab) {
  if (!io_ok(dtype) || rows < 0 || vocab < 1) return -1;
  const int slices = slices_for(rows, vocab);
  return slices == 1 ? 0 : rows * slices * (int64_t)sizeof(Sum);
}

int muon_token_logprobs(const void* logits, int dtype, int64_t row_stride, int64_t rows,
                        int64_t vocab, const int64_t* tokens, float temperature, float* logprobs,
                        float* stats, void* ws, void* stream) {
  const int rc = check("token_logprobs", dtype, rows, vocab, row_stride, temperature);
  if (rc || rows == 0) return rc;
  if (!logits || !tokens || !logprobs || (!ws && slices_for(rows, vocab) > 1)) {
    muon_set_error("token_logprobs: null tensor");
    return MUON_ERR_ARG;
  }
  const double inv = 1.0 / (double)temperature;
  const Rows a = {logits, row_stride, rows, vocab, tokens, (float)(LOG2E_D * inv), inv, logprobs, stats};
  const Policy none = {};
  return launch_sums(a, none, dtype, ws, (hipStream_t)stream);
}

int muon_token_logprobs_backward(const void* logits, int dtype, int64_t row_stride, int64_t rows,
                                 int64_t vocab, const int64_t* tokens, float temperature,
                                 const float* stats, const float* dlogprobs, const float* scale,
                                 void* dlogits, void* stream) {
  const int rc = check("token_logprobs_backward", dtype, rows, vocab, row_stride, temperature);
  if (rc || rows == 0) return rc;
  if (!logits || !tokens || !stats || !dlogprobs || !dlogits) {
    muon_set_error("token_logprobs_backward: null tensor");
    return MUON_ERR_ARG;
  }
  const double inv = 1.0 / (double)temperature;
  const Back a = {logits, row_stride, rows, vocab, tokens, stats, dlogprobs, scale,
                  (float)(LOG2E_D * inv), (float)inv, dlogits, 0};
  return launch_backward<false>("token_logprobs_backward", a, dtype, (hipStream_t)stream);
}

int muon_policy_loss_one_pass(int dtype, int64_t vocab) {
  if (dtype == MUON_DT_BF16) return vocab >= 1 && vocab <= 1024 * 20 * 8;
  return dtype == MUON_DT_F32 && vocab >= 1 && vocab <= 1024 * 20 * 4;
}

int muon_policy_loss(const void* logits, int dtype, int64_t row_stride, int64_t rows,
                     int64_t vocab, const int64_t* tokens, const float* old_logprobs,
                     const float* advantages, const float* weights, const float* ref_logprobs,
                     float clip_low, float clip_high, float kl_coef, float temperature,
                     float* loss, float* logprobs, float* terms, float* stats, float* coef,
                     void* dlogits, void* ws, void* stream) {
  const int rc = check("policy_loss", dtype, rows, vocab, row_stride, temperature);
  if (rc) return rc;
  if (!loss || (rows && (!logits || !tokens || !old_logprobs || !advantages || !weights ||
                         !logprobs || !terms || (!ws && !dlogits && slices_for(rows, vocab) > 1)))) {
    muon_set_error("policy_loss: null tensor");
    return MUON_ERR_ARG;
  }
  if (!(clip_low >= 0.0f) || !(clip_high >= 0.0f)) {
    muon_set_error("policy_loss: negative clip range");
    return MUON_ERR_ARG;
  }
  if (dlogits && !muon_policy_loss_one_pass(dtype, vocab)) {
    muon_set_error("policy_loss: no gradient in the forward pass for dtype %d, vocabulary %lld",
                   dtype, (long long)vocab);
    return MUON_ERR_ARG;
  }
  hipStream_t s = (hipStream_t)stream;
  const double inv = 1.0 / (double)temperature;
  const Rows a = {logits, row_stride, rows, vocab, tokens, (float)(LOG2E_D * inv), inv, logprobs, stats};
  const Policy p = {old_logprobs, advantages, weights, ref_logprobs, clip_low, clip_high, kl_coef,
                    terms, coef};
  if (rows) {
    const int r = !dlogits ? launch_sums(a, p, dtype, ws, s)
                  : dtype == MUON_DT_BF16 ? launch_policy_rows<MUON_DT_BF16>(a, p, dlogits, s)
                                          : launch_policy_rows<MUON_DT_F32>(a, p, dlogits, s);
    if (r) return r;
  }
  loss_kernel<<<1, 1024, 0, s>>>(terms, rows, loss);
  MUON_CHECK_LAUNCH("policy_loss sum");
  return MUON_OK;
}

int muon_scale_gradient(void* x, int dtype, int64_t n, const float* scale, void* stream) {
  if (!io_ok(dtype)) {
    muon_set_error("scale_gradient: unsupported dtype %d", dtype);
    return MUON_ERR_DTYPE;
  }
  if (n < 0 || (n && (!x || !scale))) {
    muon_set_error("scale_gradient: bad arguments");
    return MUON_ERR_ARG;
  }
  if (n == 0) return MUON_OK;
  const int grid = (int)std::min<int64_t>((n / 2048) + 1, 1024);
  hipStream_t s = (hipStream_t)stream;
  if (dtype == MUON_DT_F32) scale_kernel<MUON_DT_F32><<<grid, 256, 0, s>>>(x, n, scale);
  else if (dtype == MUON_DT_BF16) scale_kernel<MUON_DT_BF16><<<grid, 256, 0, s>>>(x, n, scale);
  else scale_kernel<MUON_DT_F16><<<grid, 256, 0, s>>>(x, n, scale);
  MUON_CHECK_LAUNCH("scale_gradient");
  return MUON_OK;
}

}  // extern "C"
