// Per-head RMS norm of queries and keys and their position rotation in one pass, with the
// backward pass (muon_qk_norm_rope, muon_qk_norm_rope_backward).
//
// One row is one head of one token: x of D values, s = sum x^2, r = 1 / sqrt(s / D + eps),
//   n_i = x_i r w_i,   (y_a, y_b) = (n_a c - n_b s, n_b c + n_a s)   over the R rotated values,
// whose pairs (a, b) are (i, i + R/2), or (2i, 2i + 1) when interleaved; the rest passes.
// Backward, with u the gradient turned back by the same angle (the rotation's transpose):
//   dw_i = sum over rows of u_i x_i r,   dx_i = r u_i w_i - x_i r^3 / D * sum_j u_j w_j x_j.
// r is recomputed from x, which the backward pass reads anyway: nothing is kept between them.
//
// Both passes are bound by memory: they read and write each row once (the angles and weights of a
// token are 4 kB beside 20 kB of bf16 rows). 32768 tokens of 32 + 8 heads of 128 in bf16: forward
// 123 us, 5.4 TB/s, backward with the weights' gradients 197 us, 5.1 TB/s, where a copy of
// 2 GiB moves 5.0. Sums, square roots and rotations are fp32, rounded once at the store.
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
// token's angles and the weights are read once for all of them. Forward / backward of the size
// above with 2, 4 and 8 heads: 134 / 223, 134 / 212 and 137 / 218 us (before the stores below).
constexpr int HC = 4;
constexpr int NTHREADS = 256;
constexpr int MAX_PAIRS = 9;  // SINGLE: up to 2 * 9 * 64 values a row
// Workgroups of the backward pass (each leaves a partial of the weights' gradients): two per CU
// hold as many loads as their registers allow; SINGLE, whose loads are small, takes twice as
// many. 6000 tokens of the size above with 512 and 1024: 39.5 and 41.3 us; 8192 tokens of 162
// values as single values 561 and 334.
constexpr int MAX_BWD_BLOCKS = 1024;
// Outputs of this many bytes (half of the 256 MB last-level cache, which else would lose its inputs to
// lines nobody reads before they are gone) are stored past the caches, if each store instruction
// writes whole pieces of at least 64 bytes. Forward / backward with and without: the size above
// 123 / 198 and 130 / 207 us, 18000 tokens of it 59 / 112 and 76 / 120; heads of 48, whose
// stores make pieces of 48 bytes, 44 / 55 and 26 / 46.
constexpr int64_t NT_FROM = 128 << 20;
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

// How a row's values are shared out over its lanes.
//  WHOLE: two runs of W values (16 bytes) a lane, which hold both partners of each rotated pair, so
//    the rotation needs no exchange between lanes: the runs at W u and R/2 + W u (halves), or
//    2 W u and 2 W u + W (interleaved, and behind R, where nothing turns). D and R in multiples of
//    2 W.
//  RAGGED: the same runs for any other D and R of at least a run a part: a part's last run is moved
//    back to end where the part ends, so that it too is one access; the values it shares with
//    the run before are computed twice, alike, and counted once in sums (the first `skip` of a run
//    are left out).
//  SINGLE: NP pairs of single values a lane, G apart, for what is too small for a run.
// 8192 tokens of 40 heads of 162 values as RAGGED and as SINGLE: forward 44 and 130, backward 92 and
// 334 us.
enum Form { WHOLE, RAGGED, SINGLE };

template <int DT, int G, int NP, Form F, bool NT>
struct Lane {
  static constexpr bool RUNS = F != SINGLE;
  static constexpr int W = DT == MUON_DT_F32 ? 4 : 8;
  static constexpr int N = RUNS ? 2 * W : 2 * NP;
  int lo, hi;              // RUNS: the first elements of the two runs
  int skip_lo, skip_hi;    // RAGGED: values at their start that belong to another lane
  int at[RUNS ? 1 : N];    // SINGLE: the element of each value, -1: none
  int ang[RUNS ? 1 : NP];  // index of a pair's angle, -1: not turned
  bool on;                 // RUNS: this lane has values

  MUON_DEVICE void init(const Args& a, int lane) {
    const int R = a.R, D = a.D, half = R / 2;
    if constexpr (F == WHOLE) {
      on = lane < D / (2 * W);
      const bool turned = lane < R / (2 * W);
      ang[0] = turned ? W * lane : -1;
      lo = turned && !a.inter ? W * lane : 2 * W * lane;
      hi = turned && !a.inter ? half + W * lane : 2 * W * lane + W;
      if (!on) lo = hi = 0;
      skip_lo = skip_hi = 0;
    } else if constexpr (F == RAGGED) {
      const int turning = (half + W - 1) / W;        // lanes of the rotated part
      const int runs = (D - R + W - 1) / W;          // runs behind it, two a lane
      on = lane < turning + (runs + 1) / 2;
      skip_lo = skip_hi = 0;
      if (!on) {
        lo = hi = 0;
        ang[0] = -1;
      } else if (lane < turning) {
        const int first = min(W * lane, half - W);   // first pair
        ang[0] = first;
        lo = a.inter ? 2 * first : first;
        hi = a.inter ? 2 * first + W : first + half;
        const int twice = W * lane - first;          // pairs that the lane before has
        if (a.inter) {
          skip_lo = min(2 * twice, W);
          skip_hi = max(2 * twice - W, 0);
        } else {
          skip_lo = skip_hi = twice;
        }
      } else {
        const int v = 2 * (lane - turning);
        ang[0] = -1;
        lo = min(R + W * v, D - W);
        hi = min(R + W * (v + 1), D - W);
        skip_lo = R + W * v - lo;
        skip_hi = min(R + W * (v + 1) - hi, W);      // W: no second run, all of it another's
      }
    } else {
      on = true;
      const int rest = D - R;
#pragma unroll
      for (int j = 0; j < NP; ++j) {
        const int u = lane + j * G;
        if (u < half) {
          ang[j] = u;
          at[2 * j] = a.inter ? 2 * u : u;
          at[2 * j + 1] = a.inter ? 2 * u + 1 : u + half;
        } else {
          const int v = 2 * (u - half);
          ang[j] = -1;
          at[2 * j] = v < rest ? R + v : -1;
          at[2 * j + 1] = v + 1 < rest ? R + v + 1 : -1;
        }
      }
    }
  }

  MUON_DEVICE int element(int j) const {
    if constexpr (RUNS) return j < W ? lo + j : hi + j - W;
    else return at[j];
  }
  // Whether value j is this lane's to count (where the lane is on).
  MUON_DEVICE bool counts(int j) const {
    if constexpr (F == WHOLE) return true;
    else if constexpr (F == RAGGED) return j < W ? j >= skip_lo : j - W >= skip_hi;
    else return at[j] >= 0;
  }

  template <int T>
  static MUON_DEVICE void load_run(const void* p, int64_t i, float* v) {
    constexpr int M = Vec16<T>::N;
    float h[M];
#pragma unroll
    for (int c = 0; c < W; c += M) {
      if constexpr (W < M) {  // 4 values of two bytes beside runs of fp32
        muon_u4 w = {0, 0, 0, 0};
        __builtin_memcpy(&w, elem_at<T>(p, i), W * 2);
        Vec16<T>::unpack(w, h);
      } else {
        Vec16<T>::unpack(load_u4(elem_at<T>(p, i + c)), h);
      }
#pragma unroll
      for (int e = 0; e < M && e < W; ++e) v[c + e] = h[e];
    }
  }

  MUON_DEVICE void load(const void* p, int64_t base, float (&v)[N]) const {
    if constexpr (RUNS) {
      load_run<DT>(p, base + lo, v);
      load_run<DT>(p, base + hi, v + W);
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j) v[j] = at[j] >= 0 ? Elem<DT>::load(p, base + at[j]) : 0.0f;
    }
  }

  MUON_DEVICE void store(void* p, int64_t base, const float (&v)[N]) const {
    if constexpr (RUNS) {
      if (!on) return;
      float h[W];
#pragma unroll
      for (int e = 0; e < W; ++e) h[e] = v[e];
      put((void*)elem_at<DT>(p, base + lo), Vec16<DT>::pack(h));
#pragma unroll
      for (int e = 0; e < W; ++e) h[e] = v[W + e];
      put((void*)elem_at<DT>(p, base + hi), Vec16<DT>::pack(h));
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (at[j] >= 0) Elem<DT>::store(p, base + at[j], v[j]);
    }
  }
  static MUON_DEVICE void put(void* p, muon_u4 w) {
    if constexpr (NT) store_u4_nt(p, w);
    else store_u4(p, w);
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
    if constexpr (RUNS) {
      load_run<WT>(w, lo, v);
      load_run<WT>(w, hi, v + W);
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
    if constexpr (RUNS) {
      if (a.R && a.table_len) {
        const int i = ang[0] < 0 ? 0 : ang[0];
        load_run<MUON_DT_F32>(a.cosv, row + i, c);
        load_run<MUON_DT_F32>(a.sinv, row + i, s);
      }
#pragma unroll
      for (int e = 0; e < W; ++e) {
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
    if constexpr (RUNS) {
      if (ang[0] < 0) {  // nothing turns here: an infinity stays out of its neighbours
#pragma unroll
        for (int e = 0; e < N; ++e) v[e] *= c[e / 2];
      } else if (a.inter) {
#pragma unroll
        for (int e = 0; e < N / 2; ++e) pair<BACK>(c[e], s[e], v[2 * e], v[2 * e + 1]);
      } else {
#pragma unroll
        for (int e = 0; e < N / 2; ++e) pair<BACK>(c[e], s[e], v[e], v[W + e]);
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

template <int DT, int G, int NP, Form F, bool NT>
__global__ __launch_bounds__(NTHREADS) void qk_forward_kernel(Args a) {
  typedef Lane<DT, G, NP, F, NT> L;
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
#pragma unroll
      for (int e = 0; e < L::N; ++e) q += l.counts(e) ? x[i][e] * x[i][e] : 0.0f;
      const float r = 1.0f / sqrtf(group_sum<G>(l.on ? q : 0.0f) / (float)a.D + a.eps);
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
template <int DT, int G, int NP, Form F, bool NT>
__global__ __launch_bounds__(NTHREADS) void qk_backward_kernel(Args a) {
  typedef Lane<DT, G, NP, F, NT> L;
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
#pragma unroll
      for (int e = 0; e < L::N; ++e) {
        q += l.counts(e) ? x[i][e] * x[i][e] : 0.0f;
        dot += l.counts(e) ? u[i][e] * w[e] * x[i][e] : 0.0f;
      }
      if (!l.on) q = dot = 0.0f;
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
    for (int j = 0; j < L::N; ++j) i = j == v % L::N && own.on && own.counts(j) ? own.element(j) : i;
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

template <int DT, int G, int NP, Form F>
int launch(const Args& a, bool backward, bool nt, hipStream_t s) {
  const int grid = a.blocks[0] + a.blocks[1];
  constexpr bool RUNS = F != SINGLE;  // single values are stored the ordinary way
  if (backward) {
    if (RUNS && nt) qk_backward_kernel<DT, G, NP, F, RUNS><<<grid, NTHREADS, 0, s>>>(a);
    else qk_backward_kernel<DT, G, NP, F, false><<<grid, NTHREADS, 0, s>>>(a);
  } else {
    if (RUNS && nt) qk_forward_kernel<DT, G, NP, F, RUNS><<<grid, NTHREADS, 0, s>>>(a);
    else qk_forward_kernel<DT, G, NP, F, false><<<grid, NTHREADS, 0, s>>>(a);
  }
  MUON_CHECK_LAUNCH("qk_norm_rope");
  return MUON_OK;
}

template <int DT, Form F>
int launch_runs(const Args& a, int lanes, bool backward, bool nt, hipStream_t s) {
  if (lanes <= 4) return launch<DT, 4, 1, F>(a, backward, nt, s);
  if (lanes <= 8) return launch<DT, 8, 1, F>(a, backward, nt, s);
  if (lanes <= 16) return launch<DT, 16, 1, F>(a, backward, nt, s);
  if (lanes <= 32) return launch<DT, 32, 1, F>(a, backward, nt, s);
  if (lanes <= 64) return launch<DT, 64, 1, F>(a, backward, nt, s);
  muon_set_error("qk_norm_rope: %d lanes a row", lanes);  // form_for gives at most 64
  return MUON_ERR_SHAPE;
}

template <int DT>
int launch_dt(const Args& a, Form form, int lanes, bool backward, bool nt, hipStream_t s) {
  if (form == WHOLE) return launch_runs<DT, WHOLE>(a, lanes, backward, nt, s);
  if (form == RAGGED) return launch_runs<DT, RAGGED>(a, lanes, backward, nt, s);
  if (lanes == 1) return launch<DT, 64, 1, SINGLE>(a, backward, false, s);
  return launch<DT, 64, MAX_PAIRS, SINGLE>(a, backward, false, s);
}

bool io_ok(int dt) { return dt == MUON_DT_F32 || dt == MUON_DT_BF16 || dt == MUON_DT_F16; }

constexpr int64_t MAX_DIM = 1024;

// Argument checks shared by both directions. Returns a status; *empty: nothing to do.
int check(const char* what, Args& a, int dtype, int64_t batch, int64_t T, int64_t q_heads,
          int64_t k_heads, int64_t D, int64_t R, int pos_bits, bool* empty) {
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
  if (a.pos && pos_bits != 32 && pos_bits != 64) {
    muon_set_error("%s: positions of %d bits", what, pos_bits);
    return MUON_ERR_ARG;
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

// The form of a row's sharing-out and its lanes (SINGLE: pairs a lane of the wave, 1 or MAX_PAIRS).
// Rows need no alignment: the hardware takes 16 bytes at any element's address.
Form form_for(const Args& a, int dtype, int* lanes) {
  const int W = dtype == MUON_DT_F32 ? 4 : 8;
  const int half = a.R / 2, rest = a.D - a.R;
  Form form = SINGLE;
  if (a.D % (2 * W) == 0 && a.R % (2 * W) == 0) {
    form = WHOLE;
    *lanes = a.D / (2 * W);
  } else if ((a.R == 0 || half >= W) && (rest == 0 || rest >= W)) {
    form = RAGGED;
    *lanes = (half + W - 1) / W + ((rest + W - 1) / W + 1) / 2;
  }
  if (form == SINGLE || *lanes > 64) {
    form = SINGLE;
    *lanes = half + (rest + 1) / 2 <= 64 ? 1 : MAX_PAIRS;
  }
  return form;
}

int group_lanes(Form form, int lanes) {
  int g = form == SINGLE ? 64 : 4;
  while (g < lanes && form != SINGLE) g *= 2;
  return g;
}

bool streams(const Args& a, int dtype) {
  const int64_t es = dtype == MUON_DT_F32 ? 4 : 2;
  // a store instruction writes each half of a row in one piece
  if (a.inter || a.R != a.D || a.R / 2 * es % 16 || a.R / 2 * es < 64) return false;
  return a.tokens * (a.s[0].heads + a.s[1].heads) * a.D * es >= NT_FROM;
}

int run(const Args& a, int dtype, bool backward, Form form, int lanes, hipStream_t s) {
  const bool nt = streams(a, dtype);
  if (dtype == MUON_DT_F32) return launch_dt<MUON_DT_F32>(a, form, lanes, backward, nt, s);
  if (dtype == MUON_DT_BF16) return launch_dt<MUON_DT_BF16>(a, form, lanes, backward, nt, s);
  return launch_dt<MUON_DT_F16>(a, form, lanes, backward, nt, s);
}

// Workgroups of the backward pass for both sides: at most `most` (and one) in all, by their units.
void backward_blocks(const int64_t (&units)[2], int groups, int most, int (&blocks)[2]) {
  const double total = (double)units[0] + (double)units[1];
  for (int i = 0; i < 2; ++i) {
    const int64_t need = (units[i] + groups - 1) / groups;
    const int64_t share = std::max<int64_t>(1, (int64_t)(most * (units[i] / total)));
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
  const int rc = check("qk_norm_rope", a, dtype, batch, tokens, q_heads, k_heads, dim, rotary,
                       pos_bits, &empty);
  if (rc || empty) return rc;
  int lanes = 0;
  const Form form = form_for(a, dtype, &lanes);
  const int64_t groups = NTHREADS / group_lanes(form, lanes);
  const int64_t b0 = (a.units[0] + groups - 1) / groups, b1 = (a.units[1] + groups - 1) / groups;
  // a launch holds fewer than 2^32 threads: beyond MAX_FWD_BLOCKS the workgroups walk on
  a.blocks[0] = (int)std::min<int64_t>(b0, MAX_FWD_BLOCKS);
  a.blocks[1] = (int)std::min<int64_t>(b1, MAX_FWD_BLOCKS);
  return run(a, dtype, false, form, lanes, (hipStream_t)stream);
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
                       rotary, pos_bits, &empty);
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
    int lanes = 0;
    const Form form = form_for(a, dtype, &lanes);
    backward_blocks(a.units, NTHREADS / group_lanes(form, lanes),
                    form == SINGLE ? MAX_BWD_BLOCKS : MAX_BWD_BLOCKS / 2, a.blocks);
    const int rb = run(a, dtype, true, form, lanes, s);
    if (rb) return rb;
  }
  if (!dw) return MUON_OK;
  qk_weight_grad_kernel<<<dim3((a.D + 15) / 16, 2), 1024, 0, s>>>(a);
  MUON_CHECK_LAUNCH("qk_norm_rope_backward weights");
  return MUON_OK;
}

}  // extern "C"
