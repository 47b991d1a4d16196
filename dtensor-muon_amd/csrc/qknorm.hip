// Per-head RMS norm of queries and keys and their position rotation in one pass, with the
// backward pass (muon_qk_norm_rope, muon_qk_norm_rope_backward).
//
// One row is one head of one token: x of D values, s = sum x^2, r = 1 / sqrt(s / D + eps),
//   n_i = x_i r w_i,   (y_a, y_b) = (n_a c - n_b s, n_b c + n_a s)   over the R rotated values,
// whose pairs (a, b) are (i, i + R/2), or (2i, 2i + 1) when interleaved; the rest passes.
// Backward, with u the gradient turned back by the same angle (the rotation's transpose):
//   dw_i = sum over rows of u_i x_i r,   dx_i = r u_i w_i - x_i r^3 / D * sum_j u_j w_j x_j.
// r is recomputed from x, which the backward pass reads anyway: nothing is kept between them.
#include <algorithm>

#include "rowops.h"

namespace {

struct Side {  // queries or keys
  const void* x;
  const void* w;   // D values, or null: all ones
  const void* dy;  // backward
  void* out;       // y, or dx: contiguous (tokens, heads, D)
  void* dw;        // backward, or null
  int64_t sb, st, sh;     // strides of x in elements: batch, token, head
  int64_t gb, gt, gh;     // strides of dy
  int heads;
  int hchunks;            // groups of HC heads
};

struct Args {
  Side s[2];
  const float* cosv;
  const float* sinv;
  int64_t table_len;
  const void* pos;      // or null: token t is at position t
  int pos64;
  int64_t pos_sb;       // stride of a batch's positions (0: shared)
  int64_t tokens;       // batch * T
  int64_t T;
  int D, R, inter;
  int wdt;
  float eps;
  int64_t units[2];     // tokens * hchunks
  int blocks[2];        // workgroups of a side
  float* part;          // backward: [side][block][D] partial weight gradients
};

// Heads of a token that one group of lanes takes: their loads are in flight together, and the
// token's angles and the weights are read once for all of them.
constexpr int HC = 4;
constexpr int NTHREADS = 256;
constexpr int MAX_BWD_BLOCKS = 1024;
constexpr int64_t MAX_FWD_BLOCKS = 1 << 22;

MUON_DEVICE void store_w(void* w, int wdt, int64_t i, float v) {
  if (wdt == MUON_DT_F32) Elem<MUON_DT_F32>::store(w, i, v);
  else if (wdt == MUON_DT_BF16) Elem<MUON_DT_BF16>::store(w, i, v);
  else Elem<MUON_DT_F16>::store(w, i, v);
}

// The position of token t of batch b; -1 outside the table (its rows become NaN: a wrong index
// shows, and nothing outside the table is read).
MUON_DEVICE int64_t position(const Args& a, int64_t b, int64_t t) {
  int64_t p = t;
  if (a.pos) {
    const int64_t i = b * a.pos_sb + t;
    p = a.pos64 ? ((const int64_t*)a.pos)[i] : (int64_t)((const int*)a.pos)[i];
  }
  return p >= 0 && p < a.table_len ? p : -1;
}

// A lane's share of a row. Vec: 16 values in two runs of 8, which hold both partners of each
// rotated pair, so the rotation needs no exchange: the runs at 8u and R/2 + 8u (halves) or one
// run of 16 (interleaved, and behind R, where nothing turns). Needs D and R in 16s.
// Otherwise NP pairs of single values, G apart: for any D and any even R.
template <int DT, int G, int NP, bool VEC>
struct Lane {
  static constexpr int N = VEC ? 16 : 2 * NP;
  int lo, hi;             // VEC: the first elements of the two runs
  int at[VEC ? 1 : N];    // otherwise the element of each value, -1: none
  int ang[VEC ? 1 : NP];  // index of a pair's angle, -1: not turned
  bool on;    // VEC: this lane has values

  MUON_DEVICE void init(const Args& a, int lane) {
    const int R = a.R, D = a.D;
    if constexpr (VEC) {
      on = lane < D / 16;
      const bool turned = lane < R / 16;
      ang[0] = turned ? 8 * lane : -1;
      lo = turned && !a.inter ? 8 * lane : 16 * lane;
      hi = turned && !a.inter ? R / 2 + 8 * lane : 16 * lane + 8;
      if (!on) lo = hi = 0;
    } else {
      on = true;
      const int turned = R / 2, rest = D - R;
#pragma unroll
      for (int j = 0; j < NP; ++j) {
        const int u = lane + j * G;
        if (u < turned) {
          ang[j] = u;
          at[2 * j] = a.inter ? 2 * u : u;
          at[2 * j + 1] = a.inter ? 2 * u + 1 : u + turned;
        } else {
          const int v = 2 * (u - turned);
          ang[j] = -1;
          at[2 * j] = v < rest ? R + v : -1;
          at[2 * j + 1] = v + 1 < rest ? R + v + 1 : -1;
        }
      }
    }
  }

  MUON_DEVICE int element(int j) const {
    if constexpr (VEC) return j < 8 ? lo + j : hi + j - 8;
    else return at[j];
  }

  MUON_DEVICE void load(const void* p, int64_t base, float (&v)[N]) const {
    if constexpr (VEC) {
      float h[8];
      Vec8<DT>::load(p, base + lo, h);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = h[e];
      Vec8<DT>::load(p, base + hi, h);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[8 + e] = h[e];
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j) v[j] = at[j] >= 0 ? Elem<DT>::load(p, base + at[j]) : 0.0f;
    }
  }

  MUON_DEVICE void store(void* p, int64_t base, const float (&v)[N]) const {
    if constexpr (VEC) {
      if (!on) return;
      float h[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) h[e] = v[e];
      Vec8<DT>::store(p, base + lo, h);
#pragma unroll
      for (int e = 0; e < 8; ++e) h[e] = v[8 + e];
      Vec8<DT>::store(p, base + hi, h);
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (at[j] >= 0) Elem<DT>::store(p, base + at[j], v[j]);
    }
  }

  MUON_DEVICE void weights(const void* w, int wdt, float (&v)[N]) const {
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = 1.0f;
    if (!w) return;
    if (wdt == MUON_DT_F32) weights_of<MUON_DT_F32>(w, v);
    else if (wdt == MUON_DT_BF16) weights_of<MUON_DT_BF16>(w, v);
    else weights_of<MUON_DT_F16>(w, v);
  }
  template <int WT>
  MUON_DEVICE void weights_of(const void* w, float (&v)[N]) const {
    if constexpr (VEC) {
      float h[8];
      Vec8<WT>::load(w, lo, h);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = h[e];
      Vec8<WT>::load(w, hi, h);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[8 + e] = h[e];
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j) v[j] = at[j] >= 0 ? Elem<WT>::load(w, at[j]) : 0.0f;
    }
  }

  // Cosine and sine of this lane's pairs at position p (p < 0: NaN; no angle: 1, 0).
  MUON_DEVICE void angles(const Args& a, int64_t p, float (&c)[N / 2], float (&s)[N / 2]) const {
    const float nan = __int_as_float(0x7fc00000);
    const int half = a.R / 2;
    const bool gone = a.R && p < 0;
    const int64_t row = p < 0 ? 0 : p * half;  // read only where the table holds something
    if constexpr (VEC) {
      if (a.R && a.table_len) {
        const int i = ang[0] < 0 ? 0 : ang[0];
        Vec8<MUON_DT_F32>::load(a.cosv, row + i, c);
        Vec8<MUON_DT_F32>::load(a.sinv, row + i, s);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        c[e] = gone ? nan : ang[0] < 0 ? 1.0f : c[e];
        s[e] = gone ? nan : ang[0] < 0 ? 0.0f : s[e];
      }
    } else {
#pragma unroll
      for (int j = 0; j < NP; ++j) {
        const bool turned = ang[j] >= 0 && !gone;
        c[j] = turned ? a.cosv[row + ang[j]] : gone ? nan : 1.0f;
        s[j] = turned ? a.sinv[row + ang[j]] : gone ? nan : 0.0f;
      }
    }
  }

  // The pairs of v turned by (c, s), or back (the transpose).
  template <bool BACK>
  MUON_DEVICE void turn(const Args& a, const float (&c)[N / 2], const float (&s)[N / 2],
                        float (&v)[N]) const {
    if constexpr (VEC) {
      if (ang[0] < 0) {  // nothing turns here: an infinity stays out of its neighbours
#pragma unroll
        for (int e = 0; e < N; ++e) v[e] *= c[e / 2];
      } else if (a.inter) {
#pragma unroll
        for (int e = 0; e < N / 2; ++e) pair<BACK>(c[e], s[e], v[2 * e], v[2 * e + 1]);
      } else {
#pragma unroll
        for (int e = 0; e < N / 2; ++e) pair<BACK>(c[e], s[e], v[e], v[8 + e]);
      }
    } else {
#pragma unroll
      for (int e = 0; e < N / 2; ++e) {
        float x = v[2 * e], y = v[2 * e + 1];
        pair<BACK>(c[e], s[e], x, y);
        v[2 * e] = ang[e] < 0 ? v[2 * e] * c[e] : x;
        v[2 * e + 1] = ang[e] < 0 ? v[2 * e + 1] * c[e] : y;
      }
    }
  }

  template <bool BACK>
  static MUON_DEVICE void pair(float c, float s, float& x, float& y) {
    const float p = x, q = y;
    x = BACK ? p * c + q * s : p * c - q * s;
    y = BACK ? q * c - p * s : q * c + p * s;
  }
};

// Which side, and which of its workgroups, a workgroup is.
MUON_DEVICE int side_of(const Args& a, int& block) {
  block = blockIdx.x;
  if (block < a.blocks[0]) return 0;
  block -= a.blocks[0];
  return 1;
}

template <int DT, int G, int NP, bool VEC>
__global__ __launch_bounds__(NTHREADS) void qk_forward_kernel(Args a) {
  typedef Lane<DT, G, NP, VEC> L;
  int block;
  const int which = side_of(a, block);
  const Side& sd = a.s[which];
  L l;
  l.init(a, threadIdx.x % G);
  const uint32_t stride = (uint32_t)a.blocks[which] * (NTHREADS / G);
  // whole groups leave the loop: the sums below stay inside groups
  for (uint32_t unit = (uint32_t)block * (NTHREADS / G) + threadIdx.x / G;
       unit < (uint32_t)a.units[which]; unit += stride) {
    const uint32_t token32 = unit / (uint32_t)sd.hchunks;
    const int h0 = (int)(unit - token32 * sd.hchunks) * HC;
    const uint32_t b32 = token32 / (uint32_t)a.T;
    const int64_t token = token32, b = b32, t = token32 - b32 * (uint32_t)a.T;
    const int64_t x0 = b * sd.sb + t * sd.st + h0 * sd.sh;
    const int n = min(HC, sd.heads - h0);
    float x[HC][L::N];
#pragma unroll
    for (int i = 0; i < HC; ++i) l.load(sd.x, x0 + min(i, n - 1) * sd.sh, x[i]);
    float w[L::N], c[L::N / 2], s[L::N / 2];
    l.angles(a, position(a, b, t), c, s);
    l.weights(sd.w, a.wdt, w);
    const int64_t y0 = (token * sd.heads + h0) * a.D;
#pragma unroll
    for (int i = 0; i < HC; ++i) {
      float q = 0.0f;
      if (l.on) {
#pragma unroll
        for (int e = 0; e < L::N; ++e) q += x[i][e] * x[i][e];
      }
      const float r = 1.0f / sqrtf(group_sum<G>(q) / (float)a.D + a.eps);
#pragma unroll
      for (int e = 0; e < L::N; ++e) x[i][e] = x[i][e] * r * w[e];
      l.template turn<false>(a, c, s, x[i]);
      if (i < n) l.store(sd.out, y0 + (int64_t)i * a.D, x[i]);
    }
  }
}

// Workgroups walk over a side's (token, head group) units; each lane keeps the weight gradient
// of its own values in registers, the groups of a workgroup are joined through LDS in a fixed
// order, and the workgroup writes one partial of D values.
template <int DT, int G, int NP, bool VEC>
__global__ __launch_bounds__(NTHREADS) void qk_backward_kernel(Args a) {
  typedef Lane<DT, G, NP, VEC> L;
  constexpr int GROUPS = NTHREADS / G;
  __shared__ float part[GROUPS][G * L::N + 1];
  int block;
  const int which = side_of(a, block);
  const Side& sd = a.s[which];
  const int lane = threadIdx.x % G, group = threadIdx.x / G;
  L l;
  l.init(a, lane);
  float w[L::N], dw[L::N];
  l.weights(sd.w, a.wdt, w);
#pragma unroll
  for (int e = 0; e < L::N; ++e) dw[e] = 0.0f;
  const uint32_t stride = (uint32_t)a.blocks[which] * GROUPS;  // at most 2^16
  for (uint32_t unit = (uint32_t)block * GROUPS + group; unit < (uint32_t)a.units[which]; unit += stride) {
    const uint32_t token32 = unit / (uint32_t)sd.hchunks;
    const int h0 = (int)(unit - token32 * sd.hchunks) * HC;
    const uint32_t b32 = token32 / (uint32_t)a.T;
    const int64_t token = token32, b = b32, t = token32 - b32 * (uint32_t)a.T;
    const int64_t x0 = b * sd.sb + t * sd.st + h0 * sd.sh;
    const int64_t g0 = b * sd.gb + t * sd.gt + h0 * sd.gh;
    const int64_t y0 = (token * sd.heads + h0) * a.D;
    const int n = min(HC, sd.heads - h0);
    float x[HC][L::N], u[HC][L::N], c[L::N / 2], s[L::N / 2];
#pragma unroll
    for (int i = 0; i < HC; ++i) l.load(sd.x, x0 + min(i, n - 1) * sd.sh, x[i]);
#pragma unroll
    for (int i = 0; i < HC; ++i) l.load(sd.dy, g0 + min(i, n - 1) * sd.gh, u[i]);
    l.angles(a, position(a, b, t), c, s);
#pragma unroll
    for (int i = 0; i < HC; ++i) {
      l.template turn<true>(a, c, s, u[i]);
      float q = 0.0f, dot = 0.0f;
      if (l.on) {
#pragma unroll
        for (int e = 0; e < L::N; ++e) {
          q += x[i][e] * x[i][e];
          dot += u[i][e] * w[e] * x[i][e];
        }
      }
      const float r = 1.0f / sqrtf(group_sum<G>(q) / (float)a.D + a.eps);
      // r^3 alone leaves the range for rows of very small or large values: r dot stays in it
      const float k = group_sum<G>(dot) * r / (float)a.D * r;
      if (i < n) {
#pragma unroll
        for (int e = 0; e < L::N; ++e) {
          dw[e] += u[i][e] * (x[i][e] * r);
          x[i][e] = (u[i][e] * w[e] - x[i][e] * k) * r;
        }
        l.store(sd.out, y0 + (int64_t)i * a.D, x[i]);
      }
    }
  }
  if (!sd.dw) return;  // the whole workgroup is on one side
#pragma unroll
  for (int e = 0; e < L::N; ++e) part[group][lane * L::N + e] = dw[e];
  __syncthreads();
  // one thread a value; its place in the row of D is the owner lane's
  for (int v = threadIdx.x; v < G * L::N; v += NTHREADS) {
    float sum = 0.0f;
    for (int g = 0; g < GROUPS; ++g) sum += part[g][v];
    L own;
    own.init(a, v / L::N);
    int i = -1;
#pragma unroll
    for (int j = 0; j < L::N; ++j) i = j == v % L::N && own.on ? own.element(j) : i;
    if (i >= 0)
      a.part[((int64_t)(which ? a.blocks[0] : 0) + block) * a.D + i] = sum;
  }
}

// dw = the workgroups' partials, summed in a fixed order: 16 columns a workgroup, 64 rows of
// threads over the partials (their loads are what this kernel waits for), joined through LDS.
__global__ __launch_bounds__(1024) void qk_weight_grad_kernel(Args a) {
  __shared__ float part[64][17];
  const int which = blockIdx.y;
  const Side& sd = a.s[which];
  if (!sd.dw) return;
  const int col = blockIdx.x * 16 + threadIdx.x % 16, row = threadIdx.x / 16;
  const float* p = a.part + (int64_t)(which ? a.blocks[0] : 0) * a.D;
  float sum = 0.0f;
  if (col < a.D)
    for (int b = row; b < a.blocks[which]; b += 64) sum += p[(int64_t)b * a.D + col];
  part[row][threadIdx.x % 16] = sum;
  __syncthreads();
  if (row == 0 && col < a.D) {
    float total = 0.0f;
    for (int r = 0; r < 64; ++r) total += part[r][threadIdx.x];
    store_w(sd.dw, a.wdt, col, total);
  }
}

// Lanes of a row in the vector form: D / 16, rounded up to a power of two.
int vec_lanes(int64_t D) {
  int g = 4;
  while (g * 16 < D) g *= 2;
  return g;
}

template <int DT, int G, int NP, bool VEC>
int launch(const Args& a, bool backward, hipStream_t s) {
  const int grid = a.blocks[0] + a.blocks[1];
  if (backward) qk_backward_kernel<DT, G, NP, VEC><<<grid, NTHREADS, 0, s>>>(a);
  else qk_forward_kernel<DT, G, NP, VEC><<<grid, NTHREADS, 0, s>>>(a);
  MUON_CHECK_LAUNCH("qk_norm_rope");
  return MUON_OK;
}

template <int DT>
int launch_dt(const Args& a, bool vec, int lanes, bool backward, hipStream_t s) {
  if (vec) {
    switch (lanes) {
      case 4: return launch<DT, 4, 8, true>(a, backward, s);
      case 8: return launch<DT, 8, 8, true>(a, backward, s);
      case 16: return launch<DT, 16, 8, true>(a, backward, s);
      case 32: return launch<DT, 32, 8, true>(a, backward, s);
      default: return launch<DT, 64, 8, true>(a, backward, s);
    }
  }
  switch (lanes) {
    case 1: return launch<DT, 64, 1, false>(a, backward, s);
    case 2: return launch<DT, 64, 2, false>(a, backward, s);
    case 4: return launch<DT, 64, 4, false>(a, backward, s);
    default: return launch<DT, 64, 9, false>(a, backward, s);
  }
}

bool aligned16(const void* p) { return !((uintptr_t)p & 15); }
bool io_ok(int dt) { return dt == MUON_DT_F32 || dt == MUON_DT_BF16 || dt == MUON_DT_F16; }

constexpr int64_t MAX_DIM = 1024;

// Argument checks shared by both directions. Returns a status; *empty: nothing to do.
int check(const char* what, Args& a, int dtype, int64_t batch, int64_t T, int64_t q_heads,
          int64_t k_heads, int64_t D, int64_t R, bool* empty) {
  if (!io_ok(dtype) || ((a.s[0].w || a.s[1].w) && !io_ok(a.wdt))) {
    muon_set_error("%s: unsupported dtype (%d, weights %d)", what, dtype, a.wdt);
    return MUON_ERR_DTYPE;
  }
  if (batch < 0 || T < 0 || q_heads < 0 || k_heads < 0 || q_heads > (1 << 20) ||
      k_heads > (1 << 20) || D < 1 || D > MAX_DIM || R < 0 || R > D || R % 2 || a.table_len < 0) {
    muon_set_error("%s: bad extents (batch %lld, tokens %lld, heads %lld and %lld, dim %lld in 1..%lld, "
                   "rotary %lld even and at most dim)", what, (long long)batch, (long long)T,
                   (long long)q_heads, (long long)k_heads, (long long)D, (long long)MAX_DIM,
                   (long long)R);
    return MUON_ERR_SHAPE;
  }
  *empty = batch * T == 0 || q_heads + k_heads == 0;
  if (*empty) return MUON_OK;
  if ((q_heads && (!a.s[0].x || !a.s[0].out)) || (k_heads && (!a.s[1].x || !a.s[1].out)) ||
      (R && (!a.cosv || !a.sinv))) {
    muon_set_error("%s: null tensor", what);
    return MUON_ERR_ARG;
  }
  a.tokens = batch * T;
  a.T = T;
  a.D = (int)D;
  a.R = (int)R;
  for (int i = 0; i < 2; ++i) {
    a.s[i].heads = (int)(i ? k_heads : q_heads);
    a.s[i].hchunks = (a.s[i].heads + HC - 1) / HC;
    a.units[i] = a.tokens * a.s[i].hchunks;
    if (a.tokens >= (1LL << 31) || a.units[i] >= (1LL << 31)) {  // the kernels count them in 32 bits
      muon_set_error("%s: too many rows (%lld tokens of %d heads)", what, (long long)a.tokens,
                     a.s[i].heads);
      return MUON_ERR_SHAPE;
    }
  }
  return MUON_OK;
}

// Whether rows can be moved in 16-byte pieces: D and R in 16s and every row 16-byte aligned.
bool vectors(const Args& a, int dtype, bool backward) {
  const int64_t es = dtype == MUON_DT_F32 ? 4 : 2;
  if (a.D % 16 || a.R % 16) return false;
  if (a.R && (!aligned16(a.cosv) || !aligned16(a.sinv))) return false;
  for (int i = 0; i < 2; ++i) {
    const Side& s = a.s[i];
    if (!s.heads) continue;
    if (!aligned16(s.x) || !aligned16(s.out) || !aligned16(s.w) || (s.sb | s.st | s.sh) * es % 16) return false;
    if (backward && (!aligned16(s.dy) || (s.gb | s.gt | s.gh) * es % 16)) return false;
  }
  return true;
}

// Lanes per row (vector form) or pairs per lane of a wave (otherwise).
int lanes_for(const Args& a, bool vec) {
  if (vec) return vec_lanes(a.D);
  const int pairs = a.R / 2 + (a.D - a.R + 1) / 2;  // at most D / 2 + 1
  return pairs <= 64 ? 1 : pairs <= 128 ? 2 : pairs <= 256 ? 4 : 9;
}

int run(const Args& a, int dtype, bool backward, bool vec, hipStream_t s) {
  const int lanes = lanes_for(a, vec);
  if (dtype == MUON_DT_F32) return launch_dt<MUON_DT_F32>(a, vec, lanes, backward, s);
  if (dtype == MUON_DT_BF16) return launch_dt<MUON_DT_BF16>(a, vec, lanes, backward, s);
  return launch_dt<MUON_DT_F16>(a, vec, lanes, backward, s);
}

// Workgroups of the backward pass for both sides: at most MAX_BWD_BLOCKS in all (four of 256
// threads per CU), by their units.
void backward_blocks(const int64_t (&units)[2], int groups, int (&blocks)[2]) {
  const double total = (double)units[0] + (double)units[1];
  for (int i = 0; i < 2; ++i) {
    const int64_t need = (units[i] + groups - 1) / groups;
    const int64_t share = std::max<int64_t>(1, (int64_t)(MAX_BWD_BLOCKS * (units[i] / total)));
    blocks[i] = (int)std::min(need, share);
  }
}

}  // namespace

extern "C" {

int muon_qk_norm_rope(const void* q, const void* k, const int64_t* strides, const void* q_weight,
                      const void* k_weight, int w_dtype, const float* cosv, const float* sinv,
                      int64_t table_len, const void* positions, int pos_bits,
                      int64_t pos_batch_stride, void* q_out, void* k_out, int dtype, int64_t batch,
                      int64_t tokens, int64_t q_heads, int64_t k_heads, int64_t dim,
                      int64_t rotary, int interleaved, float eps, void* stream) {
  Args a = {};
  if (!strides) {
    muon_set_error("qk_norm_rope: null strides");
    return MUON_ERR_ARG;
  }
  a.s[0] = {q, q_weight, nullptr, q_out, nullptr, strides[0], strides[1], strides[2], 0, 0, 0, 0, 0};
  a.s[1] = {k, k_weight, nullptr, k_out, nullptr, strides[3], strides[4], strides[5], 0, 0, 0, 0, 0};
  a.cosv = cosv; a.sinv = sinv; a.table_len = table_len;
  a.pos = positions; a.pos64 = pos_bits == 64; a.pos_sb = pos_batch_stride;
  a.inter = interleaved; a.wdt = w_dtype; a.eps = eps;
  bool empty = false;
  const int rc = check("qk_norm_rope", a, dtype, batch, tokens, q_heads, k_heads, dim, rotary, &empty);
  if (rc || empty) return rc;
  const bool vec = vectors(a, dtype, false);
  const int64_t groups = NTHREADS / (vec ? lanes_for(a, true) : 64);
  const int64_t b0 = (a.units[0] + groups - 1) / groups, b1 = (a.units[1] + groups - 1) / groups;
  // a launch holds fewer than 2^32 threads: beyond MAX_FWD_BLOCKS the workgroups walk on
  a.blocks[0] = (int)std::min<int64_t>(b0, MAX_FWD_BLOCKS);
  a.blocks[1] = (int)std::min<int64_t>(b1, MAX_FWD_BLOCKS);
  return run(a, dtype, false, vec, (hipStream_t)stream);
}

int64_t muon_qk_norm_rope_workspace_bytes(int64_t dim) {
  return dim < 1 || dim > MAX_DIM ? -1 : (MAX_BWD_BLOCKS + 2) * dim * 4;
}

int muon_qk_norm_rope_backward(const void* q, const void* k, const void* dq_out,
                               const void* dk_out, const int64_t* strides, const void* q_weight,
                               const void* k_weight, int w_dtype, const float* cosv,
                               const float* sinv, int64_t table_len, const void* positions,
                               int pos_bits, int64_t pos_batch_stride, void* dq, void* dk,
                               void* dq_weight, void* dk_weight, void* ws, int dtype,
                               int64_t batch, int64_t tokens, int64_t q_heads, int64_t k_heads,
                               int64_t dim, int64_t rotary, int interleaved, float eps,
                               void* stream) {
  Args a = {};
  if (!strides) {
    muon_set_error("qk_norm_rope_backward: null strides");
    return MUON_ERR_ARG;
  }
  a.s[0] = {q, q_weight, dq_out, dq, dq_weight, strides[0], strides[1], strides[2],
            strides[6], strides[7], strides[8], 0, 0};
  a.s[1] = {k, k_weight, dk_out, dk, dk_weight, strides[3], strides[4], strides[5],
            strides[9], strides[10], strides[11], 0, 0};
  a.cosv = cosv; a.sinv = sinv; a.table_len = table_len;
  a.pos = positions; a.pos64 = pos_bits == 64; a.pos_sb = pos_batch_stride;
  a.inter = interleaved; a.wdt = w_dtype; a.eps = eps; a.part = (float*)ws;
  bool empty = false;
  const int rc = check("qk_norm_rope_backward", a, dtype, batch, tokens, q_heads, k_heads, dim,
                       rotary, &empty);
  if (rc) return rc;
  const bool dw = dq_weight || dk_weight;
  if ((dq_weight && !q_weight) || (dk_weight && !k_weight) || (dw && !ws) ||
      (!empty && ((q_heads && !dq_out) || (k_heads && !dk_out)))) {
    muon_set_error("qk_norm_rope_backward: null tensor");
    return MUON_ERR_ARG;
  }
  hipStream_t s = (hipStream_t)stream;
  if (empty) a.D = (int)dim;  // no rows: the weights' gradients are sums over nothing
  if (!empty) {
    const bool vec = vectors(a, dtype, true);
    backward_blocks(a.units, NTHREADS / (vec ? lanes_for(a, true) : 64), a.blocks);
    const int rb = run(a, dtype, true, vec, s);
    if (rb) return rb;
  }
  if (!dw) return MUON_OK;
  qk_weight_grad_kernel<<<dim3((a.D + 15) / 16, 2), 1024, 0, s>>>(a);
  MUON_CHECK_LAUNCH("qk_norm_rope_backward weights");
  return MUON_OK;
}

}  // extern "C"
