// The gradient of log probabilities to rows of logits, of logprob.hip (a pass over the logits) and
// rescale.hip (a gradient already made, for another loss gradient). Both include it: with both forms
// of the kernel in one unit the compiler hoists the tests of a row's end out of either, and 8192
// rows of 2000 bf16 values take 17.5 us instead of 14.9.
#pragma once
#include <algorithm>

#include "rowops.h"

namespace {

constexpr double LOG2E_D = 1.4426950408889634074;

// Values [i0, i0 + N) of a row that ends at V; -inf behind it.
template <int DT>
MUON_DEVICE muon_u4 load_tail(const void* x, int64_t at, int64_t i0, int64_t V) {
  constexpr int N = Vec16<DT>::N;
  float v[N];
#pragma unroll
  for (int e = 0; e < N; ++e) v[e] = i0 + e < V ? Elem<DT>::load(x, at + i0 + e) : -INFINITY;
  return Vec16<DT>::pack(v);
}
template <int DT>
MUON_DEVICE void store_tail(void* x, int64_t at, int64_t i0, int64_t V, const float* v) {
#pragma unroll
  for (int e = 0; e < Vec16<DT>::N; ++e)
    if (i0 + e < V) Elem<DT>::store(x, at + i0 + e, v[e]);
}

template <bool STREAM>
MUON_DEVICE void put(void* p, muon_u4 w) {
  if constexpr (STREAM) store_u4_nt(p, w);
  else store_u4(p, w);
}

struct Back {
  const void* x;
  int64_t stride, N, V;
  const int64_t* tokens;
  const float* stats;
  const float* coef;   // per row: the gradient of logp
  const float* scale;  // one value, or null
  float k, tau_inv;
  void* dx;  // contiguous
  int last_first;  // rows from the last to the first
};

// dx of one run of values of a row; tok is the token's place in it, if it is there at all.
template <int DT>
MUON_DEVICE void slopes(const float (&x)[Vec16<DT>::N], float m, float k, float pc, float g,
                        int64_t tok, float (&d)[Vec16<DT>::N]) {
  constexpr int N = Vec16<DT>::N;
#pragma unroll
  for (int e = 0; e < N; ++e) d[e] = -pc * __builtin_amdgcn_exp2f((x[e] - m) * k);
  if ((uint64_t)tok < (uint64_t)N) {  // one run of the row
#pragma unroll
    for (int e = 0; e < N; ++e) d[e] += tok == e ? g : 0.0f;
  }
}

constexpr int BACK_THREADS = 256;
constexpr int BACK_VECS = 4;  // 16-byte pieces per thread

// What a row's gradient takes beside its logits, loaded ahead by the launch that walks over rows.
struct RowBack {
  int64_t tok;
  float up, m, inv;
};
MUON_DEVICE RowBack back_of_row(const Back& a, int64_t y) {
  const int64_t row = a.last_first ? a.N - 1 - y : y;
  return {a.tokens[row], a.coef[row], a.stats[row], a.stats[a.N + row]};
}

// The gradient from the logits again and the kept m and 1 / s. Grid: pieces of a row x rows.
// MADE: dx holds the gradient for a scale of one, and is made again for another scale. (The product
// of what was rounded would be rounded twice.) Rows without a gradient stay zero. A workgroup walks
// over many rows there, and loads the next one's own values while it makes one: 6144 rows of 128000
// bf16 values, a quarter left out, with their loss 980 -> 968 us, 65000 rows of 1000 235 -> 213.
template <int DT, bool STREAM, bool MADE>
__global__ __launch_bounds__(BACK_THREADS) void logp_backward_kernel(Back a) {
  constexpr int N = Vec16<DT>::N;
  const float scale = a.scale ? a.scale[0] : 1.0f;
  RowBack own, next;  // MADE alone
  if constexpr (MADE) {
    if (scale == 1.0f) return;
    next = back_of_row(a, blockIdx.y);
  }
  for (int64_t y = blockIdx.y; y < a.N; y += gridDim.y) {
    const int64_t row = a.last_first ? a.N - 1 - y : y;
    if constexpr (MADE) {
      own = next;
      if (y + gridDim.y < a.N) next = back_of_row(a, y + gridDim.y);
      if (own.tok < 0 || own.up == 0.0f) continue;
    }
    const int64_t tok = MADE ? own.tok : a.tokens[row];
    const float up = tok < 0 ? 0.0f : MADE ? own.up : a.coef[row];
    // no gradient, whatever the scale: one that overflowed makes none of it
    const float g = up == 0.0f ? 0.0f : up * scale * a.tau_inv;
    const int64_t at = row * a.stride, to = row * a.V;
    const int64_t i0 = ((int64_t)blockIdx.x * BACK_VECS * BACK_THREADS + threadIdx.x) * N;
    if (g == 0.0f) {
#pragma unroll
      for (int u = 0; u < BACK_VECS; ++u) {
        const int64_t i = i0 + (int64_t)u * BACK_THREADS * N;
        if (i + N <= a.V) put<STREAM>((void*)elem_at<DT>(a.dx, to + i), muon_u4{0, 0, 0, 0});
        else if (i < a.V) {
          const float z[N] = {};
          store_tail<DT>(a.dx, to, i, a.V, z);
        }
      }
      continue;
    }
    const float m = MADE ? own.m : a.stats[row], pc = g * (MADE ? own.inv : a.stats[a.N + row]);
    muon_u4 w[BACK_VECS];
#pragma unroll
    for (int u = 0; u < BACK_VECS; ++u) {
      const int64_t i = i0 + (int64_t)u * BACK_THREADS * N;
      if (i + N <= a.V) w[u] = load_u4(elem_at<DT>(a.x, at + i));
      else if (i < a.V) w[u] = load_tail<DT>(a.x, at, i, a.V);
    }
#pragma unroll
    for (int u = 0; u < BACK_VECS; ++u) {
      const int64_t i = i0 + (int64_t)u * BACK_THREADS * N;
      if (i >= a.V) break;
      float x[N], d[N];
      Vec16<DT>::unpack(w[u], x);
      slopes<DT>(x, m, a.k, pc, g, tok - i, d);
      if (i + N <= a.V) put<STREAM>((void*)elem_at<DT>(a.dx, to + i), Vec16<DT>::pack(d));
      else store_tail<DT>(a.dx, to, i, a.V, d);
    }
  }
}

bool io_ok(int dt) { return dt == MUON_DT_F32 || dt == MUON_DT_BF16 || dt == MUON_DT_F16; }

int check(const char* what, int dtype, int64_t N, int64_t V, int64_t stride, float tau) {
  if (!io_ok(dtype)) {
    muon_set_error("%s: unsupported dtype %d", what, dtype);
    return MUON_ERR_DTYPE;
  }
  if (N < 0 || N >= (1LL << 31) || V < 1 || V >= (1LL << 31) || stride < 0) {
    muon_set_error("%s: bad extents (rows %lld, vocabulary %lld, row stride %lld)", what,
                   (long long)N, (long long)V, (long long)stride);
    return MUON_ERR_SHAPE;
  }
  // 1 / tau and log2(e) / tau stay in fp32's range
  if (!(tau >= 1e-30f && tau <= 1e30f)) {
    muon_set_error("%s: temperature %g is not within 1e-30 and 1e30", what, (double)tau);
    return MUON_ERR_ARG;
  }
  return MUON_OK;
}

constexpr int64_t MAX_GRID_Y = 65535;
// Gradients of this many bytes are stored past the caches (half of the 256 MB last-level one).
// The gradient of 4096 rows of 128000 bf16 values 406 -> 381 us, of 2047 rows of 50257 73 -> 63.
constexpr int64_t STREAM_FROM = 128 << 20;

// The backward pass follows the forward pass that read the same logits. Where they are more than
// the last-level cache holds, what is left of them there are the last rows, and it begins with
// those: forward and backward of 4096 rows of 128000 bf16 logits 559 -> 547 us, of 4096 x 64000 in
// fp16 288 -> 272; logits that fit go from first to last (2047 rows of 50257: 109 us, the other
// way 111).
constexpr int64_t CACHE_BYTES = 256 << 20;

// Workgroups of MADE, all of which start to look at the scale: with 2048, 4096 and 8192 a scale of
// one costs 4096 rows of 50257 bf16 values 0.8, 1.5 and 3 us, and another one takes 168, 155 and 144.
constexpr int64_t MADE_BLOCKS = 4096;

template <int DT, bool MADE>
void launch_backward(Back a, hipStream_t s) {
  a.last_first = a.N * a.V * (DT == MUON_DT_F32 ? 4 : 2) > CACHE_BYTES;
  const int64_t per = (int64_t)BACK_THREADS * BACK_VECS * Vec16<DT>::N;
  const int64_t pieces = (a.V + per - 1) / per;
  const int64_t most = MADE ? std::max<int64_t>(1, MADE_BLOCKS / pieces) : MAX_GRID_Y;
  const dim3 grid((unsigned)pieces, (unsigned)std::min(a.N, most));
  if (a.N * a.V * (DT == MUON_DT_F32 ? 4 : 2) >= STREAM_FROM)
    logp_backward_kernel<DT, true, MADE><<<grid, BACK_THREADS, 0, s>>>(a);
  else
    logp_backward_kernel<DT, false, MADE><<<grid, BACK_THREADS, 0, s>>>(a);
}

template <bool MADE>
int launch_backward(const char* what, const Back& a, int dtype, hipStream_t s) {
  if (dtype == MUON_DT_F32) launch_backward<MUON_DT_F32, MADE>(a, s);
  else if (dtype == MUON_DT_BF16) launch_backward<MUON_DT_BF16, MADE>(a, s);
  else if constexpr (!MADE) launch_backward<MUON_DT_F16, MADE>(a, s);  // no pass makes one in fp16
  MUON_CHECK_LAUNCH(what);
  return MUON_OK;
}

}  // namespace
