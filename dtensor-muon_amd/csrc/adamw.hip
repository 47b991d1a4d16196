// One AdamW step over many tensors (muon_adamw): for every value, with t the tensor's step,
//   m = b1 m + (1 - b1) g,  v = b2 v + (1 - b2) g^2
//   p = (1 - lr wd) p - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
// in fp32, p rounded once to its type. The moments are fp32, or fp8: e4m3 codes with one scale
// (absmax / 448) for each block of values. In fp8 the second moment is held as its root, which spans half
// the binades that v does: e4m3 has 17 of them under a block's largest. Mean and root have scales of their
// own, and a block's mean can be far below its root (a large gradient whose sign alternates, or one that
// is past), so a root can be too small for a code where its mean has one, and would leave m / eps for
// the next step: the root's code is at least 1 where the mean's is not 0.
//
// Codes are rounded to nearest while a moment moves by more than that holds back: without a gradient, a mean
// by 1 - b1 and a root by 1 - sqrt(b2), where half a step of a code is 2^-5 to 2^-4. Up to b2 = 0.95 a block's
// scale, which its largest value moves, shifts the codes enough for the roots to follow. Beyond that they
// stay (b2 = 0.99, gradients that fall from 0.5 to 0.005 beside others: roots 59 times too large), and
// from b1 = 15/16 on a mean does: codes are rounded up or down at random then, by a number made from the
// step and the value's place, with the chance that keeps the value on the average. The nearest codes of a mean
// below 8 of the least codes stay too, at any b1: without a gradient it gives up half of one more a step, or a
// row that is not met beside others in its block would be stepped for good (0.2 lr after 1000 steps).
//
// Two kinds of launches: a table of the tensors (pointers, first piece of work, and the two factors that
// depend on t, whose counters it moves on), as many as a launch's arguments hold at a time; then one
// over all values, whose workgroups find their tensor in the table. Everything that changes from step
// to step is on the device, so a captured step counts on when it is replayed.
//
// It moves bytes: 28 a value in fp32, 22 with 16-bit parameters, 10 with those and fp8 moments. 39.4
// million fp32 values in 63 tensors take 231 us (4.8 TB/s), two bf16 tensors of 64000 x 4096 with fp8
// moments 1040 to 1120 (4.7 to 5.0; 1300 to 1390 with codes at random), where a copy runs at 4.9. 129 tensors
// of 128 and 4096 values: 6.6 us after tables of 1.6 to 3.9 for 48 of them.
#include <algorithm>
#include <cmath>

#include "rowops.h"

namespace {

// A tensor in the table.
struct Entry {
  void* p;
  const void* g;
  void* m;
  void* v;
  float* m_scale;
  float* v_scale;
  int64_t n;
  float size, scale;  // lr / (1 - b1^t), 1 / sqrt(1 - b2^t)
  uint32_t seed;      // of the step's random numbers
};

constexpr int TABLE_MAX = 48;  // tensors of one table launch: 3.5 KB of arguments
struct TableArgs {
  MuonAdamTensor t[TABLE_MAX];
  int first[TABLE_MAX];  // first piece of work
  int n, at;             // at: the table's index of t[0]
  Entry* table;
  int* pieces;
  double lr, log2_b1, log2_b2;
};

// 32 bits that change with every bit of x: the odd numbers are 2^32 over the golden ratio and 2^31.5.
MUON_DEVICE uint32_t scatter(uint32_t x) {
  x = (x ^ x >> 16) * 0xb504f333u;
  x = (x ^ x >> 15) * 0x9e3779b1u;
  return x ^ x >> 16;
}

__global__ __launch_bounds__(64) void adamw_table_kernel(TableArgs a) {
  const int i = threadIdx.x;
  if (i >= a.n) return;
  const MuonAdamTensor& t = a.t[i];
  const float step = *t.step + 1.0f;
  *t.step = step;
  // b^t by a power of two; b = 0 has log2 -inf and gives 0
  const double c1 = 1.0 - exp2(step * a.log2_b1), c2 = 1.0 - exp2(step * a.log2_b2);
  a.table[a.at + i] = Entry{t.param, t.grad, t.exp_avg, t.exp_avg_sq, t.avg_scale, t.sq_scale, t.numel,
                            (float)(a.lr / c1), (float)(1.0 / sqrt(c2)), scatter(__float_as_uint(step))};
  a.pieces[a.at + i] = a.first[i];
}

struct StepArgs {
  const Entry* table;
  const int* pieces;  // first piece of each tensor, in order
  int n, runs;        // tensors; runs of THREADS * 8 values in a piece
  float b1, c1, b2, c2, eps, decay;  // c = 1 - b; c1 below 0 to maximize
};

constexpr int THREADS = 256;
constexpr int64_t MOST_TENSORS = 1 << 20;

// This workgroup's tensor: the last whose first piece is not behind it.
MUON_DEVICE int find_tensor(const StepArgs& a) {
  int count = 0;
  for (int i0 = 0; i0 < a.n; i0 += THREADS) {
    const int i = i0 + threadIdx.x;
    count += __syncthreads_count(i < a.n && a.pieces[i] <= (int)blockIdx.x);
  }
  return count - 1;
}

// Eight values of a tensor from e on: those behind its end are 0 and not stored.
template <int DT>
MUON_DEVICE void load8(const void* p, int64_t e, int left, float (&x)[8]) {
  constexpr int N = Vec16<DT>::N;
  if (left >= 8) {
#pragma unroll
    for (int h = 0; h < 8 / N; ++h) {
      float part[N];
      Vec16<DT>::unpack(load_u4(elem_at<DT>(p, e + h * N)), part);
#pragma unroll
      for (int j = 0; j < N; ++j) x[h * N + j] = part[j];
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = j < left ? Elem<DT>::load(p, e + j) : 0.0f;
  }
}
template <int DT>
MUON_DEVICE void store8(void* p, int64_t e, int left, const float (&x)[8]) {
  constexpr int N = Vec16<DT>::N;
  if (left >= 8) {
#pragma unroll
    for (int h = 0; h < 8 / N; ++h) {
      float part[N];
#pragma unroll
      for (int j = 0; j < N; ++j) part[j] = x[h * N + j];
      store_u4((void*)elem_at<DT>(p, e + h * N), Vec16<DT>::pack(part));
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < left) Elem<DT>::store(p, e + j, x[j]);
  }
}

// The step of one value; m and v are the new moments, root = sqrt(v).
MUON_DEVICE void step_value(const StepArgs& a, const Entry& t, float g, float& p, float& m, float& v,
                            float& root) {
#pragma clang fp contract(off)
  m = m * a.b1 + g * a.c1;
  v = v * a.b2 + (g * g) * a.c2;
  root = sqrtf(v);
  p = p * a.decay - t.size * (m / (root * t.scale + a.eps));
}

template <int DT>
__global__ __launch_bounds__(THREADS) void adamw_kernel(StepArgs a) {
  const int i = find_tensor(a);
  const Entry t = a.table[i];
  int64_t e = (int64_t)(blockIdx.x - a.pieces[i]) * a.runs * (THREADS * 8) + threadIdx.x * 8;
  for (int r = 0; r < a.runs && e < t.n; ++r, e += THREADS * 8) {
    const int left = (int)std::min<int64_t>(t.n - e, 8);
    float p[8], g[8], m[8], v[8];
    load8<DT>(t.g, e, left, g);
    load8<DT>(t.p, e, left, p);
    load8<MUON_DT_F32>(t.m, e, left, m);
    load8<MUON_DT_F32>(t.v, e, left, v);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      float root;
      step_value(a, t, g[j], p[j], m[j], v[j], root);
    }
    store8<DT>(t.p, e, left, p);
    store8<MUON_DT_F32>(t.m, e, left, m);
    store8<MUON_DT_F32>(t.v, e, left, v);
  }
}

MUON_DEVICE uint32_t larger_bits(uint32_t a, float x) { return std::max(a, __float_as_uint(x) & 0x7fffffffu); }

// Eight codes times a scale.
MUON_DEVICE void decode8(uint2 c, float scale, float (&x)[8]) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int w = (int)(h ? c.y : c.x);
    x[4 * h] = __builtin_amdgcn_cvt_f32_fp8(w, 0) * scale;
    x[4 * h + 1] = __builtin_amdgcn_cvt_f32_fp8(w, 1) * scale;
    x[4 * h + 2] = __builtin_amdgcn_cvt_f32_fp8(w, 2) * scale;
    x[4 * h + 3] = __builtin_amdgcn_cvt_f32_fp8(w, 3) * scale;
  }
}
// The quotient x / scale, correctly rounded: inv = 1 / scale gives it up to an ulp, and the exact remainder
// of that moves it to the rounded one (P. Markstein, IBM J. Res. Dev. 34(1), 1990). A finite scale is 2^-49
// to 2^120, and only quotients from 2^-10 on have a code, so what such a value goes through is normal. Of an
// infinite or NaN scale, whose values are all NaN, the product with its inverse has the quotient's code.
struct Quotient {
  float inv, neg, back;
  MUON_DEVICE explicit Quotient(float scale) : inv(1.0f / scale) {
    const bool finite = scale <= 3.40282347e38f;
    neg = finite ? -scale : 0.0f;
    back = finite ? inv : 0.0f;
  }
  MUON_DEVICE float operator()(float x) const {
#pragma clang fp contract(off)
    const float q = x * inv;
    return __builtin_fmaf(__builtin_fmaf(neg, q, x), back, q);
  }
};
MUON_DEVICE uint2 encode8(const float (&x)[8], const Quotient& by) {
  uint32_t w[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    int c = __builtin_amdgcn_cvt_pk_fp8_f32(by(x[4 * h]), by(x[4 * h + 1]), 0, false);
    w[h] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(by(x[4 * h + 2]), by(x[4 * h + 3]), c, true);
  }
  return make_uint2(w[0], w[1]);
}
// A quotient as one of the two values of a code around it, up if random bits carry: a code has 3 bits of a
// float's 23, and below 2^-6 steps of 2^-9, which 2^-6 more makes the same. 16 of the 20 bits behind a code's
// are random and the last ones their middle: a move of a 2^-11th of a step (b2 = 0.9999) is off by 2% at most.
MUON_DEVICE float to_code(float y, uint32_t random16) {
  const float a = fabsf(y), more = a >= 0x1p-6f ? 0.0f : 0x1p-6f;
  const float c = __uint_as_float((__float_as_uint(a + more) + (random16 << 4 | 8)) & 0xfff00000u) - more;
  return copysignf(c > 448.0f ? 448.0f : c, y);
}
// The codes of eight means and roots at random, by a number for each place.
MUON_DEVICE void encode8_random(const float (&m)[8], const Quotient& by_m, const float (&v)[8], const Quotient& by_v,
                                uint32_t seed, uint2& cm, uint2& cv) {
  uint32_t wm[2], wv[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float x[4], y[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t r = scatter(seed + (4 * h + j) * 0x9e3779b1u);
      x[j] = to_code(by_m(m[4 * h + j]), r & 0xffffu);
      y[j] = to_code(by_v(v[4 * h + j]), r >> 16);
    }
    int c = __builtin_amdgcn_cvt_pk_fp8_f32(x[0], x[1], 0, false);
    wm[h] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x[2], x[3], c, true);
    c = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
    wv[h] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], c, true);
  }
  cm = make_uint2(wm[0], wm[1]);
  cv = make_uint2(wv[0], wv[1]);
}

// The codes v of roots, the least one in place of 0 where the mean's code in m is not 0.
MUON_DEVICE uint32_t least_root(uint32_t v, uint32_t m) {
  constexpr uint32_t low = 0x7f7f7f7fu, top = 0x80808080u;  // a byte of 7 bits and low: top set if it is not 0
  return v | (((m & low) + low) & ~((v & low) + low) & top) >> 7;
}
// Without a gradient, means below 8 of the least code, whose decay by up to 1/16 is less than half a code, give up
// half of one before it.
MUON_DEVICE void rest8(const float (&g)[8], float scale, float (&m)[8]) {
  float least = fabsf(g[0]);
#pragma unroll
  for (int j = 1; j < 8; ++j) least = fminf(least, fabsf(g[j]));
  if (least != 0.0f) return;
  const float half = scale * 0x1p-10f;
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (g[j] == 0.0f && fabsf(m[j]) < 16.0f * half) m[j] -= __builtin_amdgcn_fmed3f(m[j], -half, half);
}
// absmax / 448 of a block; bits are compared as integers, so that a NaN is the largest
MUON_DEVICE float block_scale(uint32_t bits) {
  const float top = __uint_as_float(bits);
  return (top < 1e-12f ? 1e-12f : top) / 448.0f;
}

// fp8 moments: a wave holds RUNS runs of 512 values, a block is G lanes of one run (G = 64: of all of
// them). Tensors are whole blocks, so the lanes of a block are all in or all out.
template <int DT, int G, int RUNS, bool RANDOM>
__global__ __launch_bounds__(THREADS) void adamw_fp8_kernel(StepArgs a) {
  const int i = find_tensor(a);
  const Entry t = a.table[i];
  constexpr int BLOCK = G * 8 * RUNS;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int64_t e0 = (int64_t)(blockIdx.x - a.pieces[i]) * a.runs * (THREADS * 8) + wave * (512 * RUNS) + lane * 8;
  for (int r = 0; r < a.runs; r += RUNS, e0 += THREADS * 8 * RUNS) {
    if (e0 >= t.n) return;
    const int64_t block = e0 / BLOCK;
    const float ms = t.m_scale[block], vs = t.v_scale[block];
    float m[RUNS][8], root[RUNS][8];
    uint32_t mt = 0, vt = 0;
#pragma unroll
    for (int q = 0; q < RUNS; ++q) {
      const int64_t e = e0 + q * 512;
      float p[8], g[8];
      load8<DT>(t.g, e, 8, g);
      load8<DT>(t.p, e, 8, p);
      uint2 cm, cv;
      __builtin_memcpy(&cm, (const uint8_t*)t.m + e, 8);
      __builtin_memcpy(&cv, (const uint8_t*)t.v + e, 8);
      decode8(cm, ms, m[q]);
      decode8(cv, vs, root[q]);
      if constexpr (!RANDOM) rest8(g, ms, m[q]);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        float v = root[q][j] * root[q][j];
        step_value(a, t, g[j], p[j], m[q][j], v, root[q][j]);
        mt = larger_bits(mt, m[q][j]);
        vt = std::max(vt, __float_as_uint(root[q][j]));  // at least 0, or a NaN of either sign
      }
      store8<DT>(t.p, e, 8, p);
    }
    const auto larger = [](uint32_t x, uint32_t y) { return std::max(x, y); };
    const float mn = block_scale(group_reduce<G>(mt, larger)), vn = block_scale(group_reduce<G>(vt, larger));
    const Quotient by_m(mn), by_v(vn);
#pragma unroll
    for (int q = 0; q < RUNS; ++q) {
      const int64_t e = e0 + q * 512;
      uint2 cm, cr;
      if constexpr (RANDOM) {
        const uint32_t seed = t.seed + (uint32_t)e * 0x9e3779b1u + (uint32_t)(e >> 32) * 0xb504f333u;
        encode8_random(m[q], by_m, root[q], by_v, seed, cm, cr);
      } else {
        cm = encode8(m[q], by_m);
        cr = encode8(root[q], by_v);
      }
      const uint2 cv = make_uint2(least_root(cr.x, cm.x), least_root(cr.y, cm.y));
      __builtin_memcpy((uint8_t*)t.m + e, &cm, 8);
      __builtin_memcpy((uint8_t*)t.v + e, &cv, 8);
    }
    if ((lane & (G - 1)) == 0) {
      t.m_scale[block] = mn;
      t.v_scale[block] = vn;
    }
  }
}

// Runs of 2048 values in a workgroup's piece: 2 where that leaves the card few pieces, else 8, so that
// finding the tensor is little beside the values; no fewer than four waves' blocks take.
int piece_runs(int64_t total, int64_t block) {
  return std::max<int>(total < (1 << 24) ? 2 : 8, (int)(block / 512));
}

}  // namespace

extern "C" int64_t muon_adamw_workspace_bytes(int64_t ntensors) {
  return ntensors < 0 || ntensors > MOST_TENSORS ? -1 : round_up(ntensors * (int64_t)sizeof(Entry), 256) + ntensors * 4;
}

extern "C" int muon_adamw(int64_t ntensors, const MuonAdamTensor* tensors, int dtype, int64_t block,
                          double lr, double beta1, double beta2, double eps, double weight_decay,
                          int maximize, void* ws, void* stream) {
  if (dtype != MUON_DT_F32 && dtype != MUON_DT_BF16 && dtype != MUON_DT_F16) {
    muon_set_error("muon_adamw: unsupported dtype %d", dtype);
    return MUON_ERR_DTYPE;
  }
  if (ntensors < 0 || ntensors > MOST_TENSORS || (block && (block < 64 || block > 2048 || (block & (block - 1))))) {
    muon_set_error("muon_adamw: %lld tensors, blocks of %lld: to 2^20, powers of two from 64 to 2048",
                   (long long)ntensors, (long long)block);
    return MUON_ERR_SHAPE;
  }
  if (ntensors && (!tensors || !ws)) {
    muon_set_error("muon_adamw: null pointer");
    return MUON_ERR_ARG;
  }
  int64_t total = 0;
  for (int64_t i = 0; i < ntensors; ++i) {
    const MuonAdamTensor& t = tensors[i];
    if (t.numel < 0 || t.numel > ((int64_t)1 << 42) || (block && t.numel % block)) {
      muon_set_error("muon_adamw: tensor %lld has %lld values in blocks of %lld", (long long)i,
                     (long long)t.numel, (long long)block);
      return MUON_ERR_SHAPE;
    }
    if (!t.step || (t.numel && (!t.param || !t.grad || !t.exp_avg || !t.exp_avg_sq ||
                                (block && (!t.avg_scale || !t.sq_scale))))) {
      muon_set_error("muon_adamw: null pointer in tensor %lld", (long long)i);
      return MUON_ERR_ARG;
    }
    total += t.numel;
  }
  if (!ntensors) return MUON_OK;
  const int runs = piece_runs(total, block);
  hipStream_t s = (hipStream_t)stream;
  Entry* table = (Entry*)ws;
  int* pieces = (int*)((char*)ws + round_up(ntensors * (int64_t)sizeof(Entry), 256));
  int64_t work = 0;
  for (const MuonAdamTensor* t = tensors; t < tensors + ntensors; ++t)
    work += (t->numel + runs * THREADS * 8 - 1) / (runs * THREADS * 8);
  if (work >= (1ll << 32) / THREADS) {  // a grid has to stay below 2^32 threads
    muon_set_error("muon_adamw: %lld values in one call", (long long)total);
    return MUON_ERR_SHAPE;
  }
  int64_t piece = 0;
  for (int64_t at = 0; at < ntensors; at += TABLE_MAX) {
    TableArgs a{};
    a.n = (int)std::min<int64_t>(ntensors - at, TABLE_MAX);
    a.at = (int)at;
    a.table = table;
    a.pieces = pieces;
    a.lr = lr;
    a.log2_b1 = std::log2(beta1);
    a.log2_b2 = std::log2(beta2);
    for (int i = 0; i < a.n; ++i) {
      a.t[i] = tensors[at + i];
      a.first[i] = (int)piece;
      piece += (tensors[at + i].numel + runs * THREADS * 8 - 1) / (runs * THREADS * 8);
    }
    adamw_table_kernel<<<1, 64, 0, s>>>(a);
    MUON_CHECK_LAUNCH("muon_adamw: table");
  }
  if (!piece) return MUON_OK;
  const float c1 = (float)(1.0 - beta1);
  const StepArgs a{table, pieces, (int)ntensors, runs, (float)beta1, maximize ? -c1 : c1, (float)beta2,
                   (float)(1.0 - beta2), (float)eps, (float)(1.0 - lr * weight_decay)};
  const bool random = beta1 >= 0.9375 || beta2 > 0.95;
  const unsigned grid = (unsigned)piece;
#define STEP(KERNEL)                                                                       \
  switch (dtype) {                                                                         \
    case MUON_DT_F32: { constexpr int DT = MUON_DT_F32; KERNEL<<<grid, THREADS, 0, s>>>(a); break; }   \
    case MUON_DT_BF16: { constexpr int DT = MUON_DT_BF16; KERNEL<<<grid, THREADS, 0, s>>>(a); break; } \
    default: { constexpr int DT = MUON_DT_F16; KERNEL<<<grid, THREADS, 0, s>>>(a); }                   \
  }
#define STEP_FP8(G, RUNS)                                \
  if (random) {                                          \
    STEP((adamw_fp8_kernel<DT, G, RUNS, true>))          \
  } else {                                               \
    STEP((adamw_fp8_kernel<DT, G, RUNS, false>))         \
  }                                                      \
  break;
  switch (block) {
    case 0: STEP((adamw_kernel<DT>)) break;
    case 64: STEP_FP8(8, 1)
    case 128: STEP_FP8(16, 1)
    case 256: STEP_FP8(32, 1)
    case 512: STEP_FP8(64, 1)
    case 1024: STEP_FP8(64, 2)
    default: STEP_FP8(64, 4)
  }
#undef STEP_FP8
#undef STEP
  MUON_CHECK_LAUNCH("muon_adamw");
  return MUON_OK;
}
