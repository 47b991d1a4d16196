// Tokens to their experts and back (muon_expert_order, muon_dispatch, muon_combine and the latter's
// gradient): the order of the (token, choice) pairs by expert, each token's row at the places of its
// choices, and the sum of the experts' rows with the token's gates.
//
// The order is a stable counting sort of the choices by expert; what names no expert comes last:
//   slot(t, j) = choices of lower experts + earlier choices of the same one       (row of the choice)
//   slot(t, j) = -1 - row for an empty choice, row = kept choices + earlier empty ones.
// So every row of the sorted order belongs to one choice, and who writes all choices has written all
// rows. With s = slot(t, j):
//   dispatch: rows[s] = x[t], 0 for an empty choice      gradient: dx[t] = sum_j drows[s]  (combine, no gates)
//   combine:  y[t] = sum_j g_tj rows[s] over the kept ones
//   gradient: drows[s] = g_tj dy[t], 0 for an empty one;  dg_tj = <dy[t], rows[s]>.
//
// All of it moves bytes. The work is laid out by tokens: a token's row is read once for all its
// choices, and their rows are whole lines wherever they lie. 32768 tokens of 2048 bf16 columns, 8 of 64
// experts, a tenth of the tokens masked: order 5.0 + 9.4 us, dispatch 212 (5.7 TB/s), combine 216 to 250
// (4.4 to 5.1), its gradient 414 (5.2), where a copy of 2 GiB runs at 4.9 TB/s. 16 tokens: 3.4, 4.4 and
// 4.4 us, one launch each and nothing but latency.
#include <algorithm>

#include "rowops.h"

namespace {

constexpr int ORDER_THREADS = 512;
constexpr int ORDER_WAVES = ORDER_THREADS / 64;
constexpr int ORDER_EMAX = 1024;
constexpr int ORDER_BATCH = 8;  // choices of a lane whose loads are under way together
// Choices that one workgroup orders alone, in one launch (2048 of 64 experts 5.7 us, 8192 15; 16384 by
// eight workgroups 9.0).
constexpr int64_t ORDER_ALONE = 4096;
constexpr int64_t ORDER_CHUNK = 2048;
// Every workgroup adds up the counts of all: so many counts at most, of a workgroup a CU at most.
constexpr int64_t ORDER_COUNTS = 65536, ORDER_BLOCKS = 256;

struct OrderArgs {
  const int64_t* experts;
  int64_t n, chunk;  // choices, and those of a workgroup (a multiple of 64 ORDER_WAVES)
  int E, blocks;
  int32_t* slots;
  int32_t* offsets;
  int32_t* counts;  // (blocks, E + 1): choices of each expert, and empty ones, by workgroup
};

// Choice i's expert, E for an empty one, -1 behind the end.
MUON_DEVICE int expert_at(const OrderArgs& a, int64_t i, int64_t end) {
  if (i >= end) return -1;
  const int64_t e = a.experts[i];
  return e >= 0 && e < a.E ? (int)e : a.E;
}

__global__ __launch_bounds__(ORDER_THREADS) void order_count_kernel(OrderArgs a) {
  __shared__ int32_t cnt[ORDER_EMAX + 1];
  const int tid = threadIdx.x;
  for (int c = tid; c <= a.E; c += ORDER_THREADS) cnt[c] = 0;
  __syncthreads();
  const int64_t begin = blockIdx.x * a.chunk, end = std::min(begin + a.chunk, a.n);
  for (int64_t i0 = begin + tid; i0 < end; i0 += ORDER_THREADS * ORDER_BATCH) {
    int e[ORDER_BATCH];
#pragma unroll
    for (int b = 0; b < ORDER_BATCH; ++b) e[b] = expert_at(a, i0 + b * ORDER_THREADS, end);
#pragma unroll
    for (int b = 0; b < ORDER_BATCH; ++b)
      if (e[b] >= 0) atomicAdd(&cnt[e[b]], 1);
  }
  __syncthreads();
  for (int c = tid; c <= a.E; c += ORDER_THREADS)
    a.counts[(int64_t)blockIdx.x * (a.E + 1) + c] = cnt[c];
}

// A workgroup's choices in order: each wave a run of them. First the counts by wave, from which each
// wave's first place for every expert follows; then 64 choices at a time, a lane's place among the
// lanes of its expert from one ballot for each bit of the number.
__global__ __launch_bounds__(ORDER_THREADS) void order_place_kernel(OrderArgs a) {
  extern __shared__ int32_t lds[];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, C = a.E + 1;
  int32_t* cnt = lds;                      // (waves, C)
  int32_t* before = lds + ORDER_WAVES * C;  // (C): choices of the workgroups before this one
  int32_t* total = before + C;              // (C): of all, then the experts' first rows
  __shared__ int32_t wave_sum[ORDER_WAVES];
  for (int c = tid; c < (ORDER_WAVES + 2) * C; c += ORDER_THREADS) lds[c] = 0;
  __syncthreads();
  const int64_t run = a.chunk / ORDER_WAVES;
  const int64_t begin = blockIdx.x * a.chunk + wave * run;
  const int64_t end = std::min(begin + run, a.n);
  for (int64_t i0 = begin + lane; i0 < end; i0 += 64 * ORDER_BATCH) {
    int e[ORDER_BATCH];
#pragma unroll
    for (int b = 0; b < ORDER_BATCH; ++b) e[b] = expert_at(a, i0 + b * 64, end);
#pragma unroll
    for (int b = 0; b < ORDER_BATCH; ++b)
      if (e[b] >= 0) atomicAdd(&cnt[wave * C + e[b]], 1);
  }
  if (a.blocks > 1) {
    const int all = a.blocks * C, mine = blockIdx.x * C;
    for (int i0 = tid; i0 < all; i0 += ORDER_THREADS * ORDER_BATCH) {
      int v[ORDER_BATCH];
#pragma unroll
      for (int b = 0; b < ORDER_BATCH; ++b) v[b] = i0 + b * ORDER_THREADS < all ? a.counts[i0 + b * ORDER_THREADS] : 0;
#pragma unroll
      for (int b = 0; b < ORDER_BATCH; ++b) {
        const int i = i0 + b * ORDER_THREADS;
        if (!v[b]) continue;
        atomicAdd(&total[i % C], v[b]);
        if (i < mine) atomicAdd(&before[i % C], v[b]);
      }
    }
    __syncthreads();
  } else {
    __syncthreads();
    for (int c = tid; c < C; c += ORDER_THREADS) {
      int sum = 0;
#pragma unroll
      for (int w = 0; w < ORDER_WAVES; ++w) sum += cnt[w * C + c];
      total[c] = sum;
    }
    __syncthreads();
  }
  // exclusive sums of the totals: a few experts in a row for each thread
  const int per = (C + ORDER_THREADS - 1) / ORDER_THREADS, c0 = tid * per;
  int sum = 0;
  for (int c = c0; c < std::min(c0 + per, C); ++c) sum += total[c];
  int incl = sum;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int v = __shfl_up(incl, off, 64);
    if (lane >= off) incl += v;
  }
  if (lane == 63) wave_sum[wave] = incl;
  __syncthreads();
  int first = incl - sum;
  for (int w = 0; w < wave; ++w) first += wave_sum[w];
  for (int c = c0; c < std::min(c0 + per, C); ++c) {
    const int t = total[c];
    if (blockIdx.x == 0) a.offsets[c] = first;
    int place = first + before[c];
    for (int w = 0; w < ORDER_WAVES; ++w) {
      const int k = cnt[w * C + c];
      cnt[w * C + c] = place;
      place += k;
    }
    first += t;
  }
  __syncthreads();
  const int bits = 32 - __builtin_clz(a.E | 1);
  const uint64_t below = (1ull << lane) - 1;
  for (int64_t i0 = begin; i0 < end; i0 += 64 * ORDER_BATCH) {
    int es[ORDER_BATCH];
#pragma unroll
    for (int b = 0; b < ORDER_BATCH; ++b) es[b] = expert_at(a, i0 + b * 64 + lane, end);
#pragma unroll
    for (int b = 0; b < ORDER_BATCH; ++b) {
      if (i0 + b * 64 >= end) break;
      const bool in = es[b] >= 0;
      const int e = in ? es[b] : 0;
      uint64_t same = __ballot(in);
      for (int k = 0; k < bits; ++k) {
        const uint64_t ones = __ballot(in && ((e >> k) & 1));
        same &= ((e >> k) & 1) ? ones : ~ones;
      }
      const int rank = __popcll(same & below);
      int place = 0;
      if (in && rank == 0) place = atomicAdd(&cnt[wave * C + e], (int)__popcll(same));
      place = __shfl(place, in ? __builtin_ctzll(same) : lane, 64) + rank;
      if (in) a.slots[i0 + b * 64 + lane] = e < a.E ? place : -1 - place;
    }
  }
}

// ---- rows -----------------------------------------------------------------------------------

constexpr int ROW_THREADS = 256;
// Workgroups of a launch at most (a grid has to stay below 2^32 threads); each walks on by as many.
constexpr int64_t ROW_GRID = 1 << 22;

struct RowArgs {
  const void* in;  // dispatch: a token's rows; combine: the experts' rows
  int64_t in_row;  // their stride in elements
  int64_t T, R;    // tokens; rows of the sorted order
  int k, W;
  int shift;       // log2 of the lanes of a token (one workgroup's threads at most)
  const int32_t* slots;
  const float* gates;  // or null: ones
  void* out;           // contiguous
};

// A lane's 16 bytes of a row. The last lane moves back until its run ends with the row, over columns that
// another one has too, so that no lane's load depends on where the row ends: single values behind a
// condition are waited for before the next row's are asked for (5001 tokens, 6 choices, 1411 fp16
// columns: combine 29.8 us so, its gradient 52.6). Only rows shorter than 16 bytes go by values.
MUON_DEVICE int part_at(int c, int W, int n) { return W < n ? c : std::min(c, W - n); }

// left: columns of the row from this place on, at most 16 bytes of which are meant; the same for all lanes.
template <int DT>
MUON_DEVICE muon_u4 load_part(const void* p, int64_t at, int left) {
  constexpr int N = Vec16<DT>::N;
  if (left >= N) return load_u4(elem_at<DT>(p, at));
  float v[N];
#pragma unroll
  for (int j = 0; j < N; ++j) v[j] = j < left ? Elem<DT>::load(p, at + j) : 0.0f;
  return Vec16<DT>::pack(v);
}
template <int DT>
MUON_DEVICE void store_part(void* p, int64_t at, int left, muon_u4 w) {
  constexpr int N = Vec16<DT>::N;
  if (left >= N) {
    store_u4((void*)elem_at<DT>(p, at), w);
    return;
  }
#pragma unroll
  for (int j = 0; j < N; ++j) {
    if (j >= left) break;
    if constexpr (DT == MUON_DT_F32)
      ((uint32_t*)p)[at + j] = w[j];
    else
      ((uint16_t*)p)[at + j] = (uint16_t)(w[j / 2] >> (16 * (j & 1)));
  }
}

template <int DT>
__global__ __launch_bounds__(ROW_THREADS) void dispatch_kernel(RowArgs a) {
  constexpr int N = Vec16<DT>::N;
  const int lanes = 1 << a.shift, v0 = threadIdx.x & (lanes - 1);
  const int64_t per = ROW_THREADS >> a.shift;
  for (int64_t t = blockIdx.x * per + (threadIdx.x >> a.shift); t < a.T; t += gridDim.x * per) {
    const int32_t* slots = a.slots + t * a.k;
    for (int c0 = v0 * N; c0 < a.W; c0 += lanes * N) {
      const int c = part_at(c0, a.W, N), left = a.W;
      const muon_u4 w = load_part<DT>(a.in, t * a.in_row + c, left);
      for (int j = 0; j < a.k; ++j) {
        const int s = slots[j], row = s < 0 ? ~s : s;
        if (row < a.R) store_part<DT>(a.out, (int64_t)row * a.W + c, left, s < 0 ? muon_u4{0, 0, 0, 0} : w);
      }
    }
  }
}


// BATCH: choices whose rows are in flight together, 8, or fewer where a token has fewer: what is asked
// and masked for the missing ones costs more than the bytes then (32768 tokens of 777 bf16 columns, one
// choice: combine 28 us by eights, 19 by twos; its gradient 52 by eights, 31 by ones).
template <int DT, int BATCH>
__global__ __launch_bounds__(ROW_THREADS) void combine_kernel(RowArgs a) {
  constexpr int N = Vec16<DT>::N;
  const int lanes = 1 << a.shift, v0 = threadIdx.x & (lanes - 1);
  const int64_t per = ROW_THREADS >> a.shift;
  for (int64_t t = blockIdx.x * per + (threadIdx.x >> a.shift); t < a.T; t += gridDim.x * per) {
    for (int c0 = v0 * N; c0 < a.W; c0 += lanes * N) {
      const int c = part_at(c0, a.W, N), left = a.W;
      float sum[N] = {};
      for (int j0 = 0; j0 < a.k; j0 += BATCH) {
        muon_u4 w[BATCH];
        float g[BATCH];
        bool kept[BATCH];
#pragma unroll
        for (int b = 0; b < BATCH; ++b) {
          const int j = j0 + b;
          const int s = j < a.k ? a.slots[t * a.k + j] : -1;
          kept[b] = s >= 0 && s < a.R;
          g[b] = a.gates && j < a.k ? a.gates[t * a.k + j] : 1.0f;
          if (kept[b]) {
            w[b] = load_part<DT>(a.in, (int64_t)s * a.in_row + c, left);
          }
        }
#pragma unroll
        for (int b = 0; b < BATCH; ++b) {
          if (!kept[b]) continue;
          float v[N];
          Vec16<DT>::unpack(w[b], v);
#pragma unroll
          for (int e = 0; e < N; ++e) sum[e] += g[b] * v[e];
        }
      }
      store_part<DT>(a.out, t * a.W + c, left, Vec16<DT>::pack(sum));
    }
  }
}

struct BackArgs {
  const void* dy;
  const void* rows;
  int64_t dy_row, rows_row;
  int64_t T, R;
  int k, W;
  const int32_t* slots;
  const float* gates;
  void* drows;    // contiguous, or null
  float* dgates;  // or null
};

// G lanes a token (a wave at most): the products of a choice's row are summed by each lane over its
// columns, then over the lanes.
template <int DT, int G, int BATCH>
__global__ __launch_bounds__(ROW_THREADS) void combine_backward_kernel(BackArgs a) {
  constexpr int N = Vec16<DT>::N;
  const int v0 = threadIdx.x & (G - 1);
  // whole groups of lanes go on or end
  const int64_t step = gridDim.x * (int64_t)(ROW_THREADS / G);
  for (int64_t t = (int64_t)blockIdx.x * (ROW_THREADS / G) + threadIdx.x / G; t < a.T; t += step) {
    for (int j0 = 0; j0 < a.k; j0 += BATCH) {
      int s[BATCH];
      float g[BATCH], dot[BATCH] = {};
#pragma unroll
      for (int b = 0; b < BATCH; ++b) {
        const int j = j0 + b;
        s[b] = j < a.k ? a.slots[t * a.k + j] : INT32_MAX;  // no row: R is at most that
        g[b] = j < a.k ? a.gates[t * a.k + j] : 0.0f;
      }
      for (int c0 = v0 * N; c0 < a.W; c0 += G * N) {
        const int c = part_at(c0, a.W, N), left = a.W, skip = c0 - c;
        float d[N];
        Vec16<DT>::unpack(load_part<DT>(a.dy, t * a.dy_row + c, left), d);
        if (a.dgates) {
          muon_u4 w[BATCH];
#pragma unroll
          for (int b = 0; b < BATCH; ++b)
            if (s[b] >= 0 && s[b] < a.R) w[b] = load_part<DT>(a.rows, (int64_t)s[b] * a.rows_row + c, left);
#pragma unroll
          for (int b = 0; b < BATCH; ++b) {
            if (!(s[b] >= 0 && s[b] < a.R)) continue;
            float v[N];
            Vec16<DT>::unpack(w[b], v);
#pragma unroll
            for (int e = 0; e < N; ++e) dot[b] += e < skip ? 0.0f : d[e] * v[e];
          }
        }
        if (a.drows) {
#pragma unroll
          for (int b = 0; b < BATCH; ++b) {
            const int row = s[b] < 0 ? ~s[b] : s[b];
            if (row >= a.R) continue;
            float v[N];
#pragma unroll
            for (int e = 0; e < N; ++e) v[e] = s[b] < 0 ? 0.0f : g[b] * d[e];
            store_part<DT>(a.drows, (int64_t)row * a.W + c, left, Vec16<DT>::pack(v));
          }
        }
      }
      if (a.dgates) {
#pragma unroll
        for (int b = 0; b < BATCH; ++b) {
          const float sum = group_sum<G>(dot[b]);
          if (v0 == 0 && j0 + b < a.k) a.dgates[t * a.k + j0 + b] = sum;
        }
      }
    }
  }
}

int lanes_shift(int dtype, int64_t width, int most) {
  const int64_t runs = (width + (dtype == MUON_DT_F32 ? 3 : 7)) / (dtype == MUON_DT_F32 ? 4 : 8);
  int shift = 0;
  while (shift < most && (1ll << shift) < runs) ++shift;
  return shift;
}

int64_t row_grid(int64_t tokens, int shift) {
  const int64_t per = ROW_THREADS >> shift;
  return std::min((tokens + per - 1) / per, ROW_GRID);
}

int64_t order_chunk(int64_t n, int64_t experts) {
  if (n <= ORDER_ALONE) return round_up(std::max<int64_t>(n, 1), ORDER_THREADS);
  const int64_t blocks = std::min(ORDER_COUNTS / (experts + 1), ORDER_BLOCKS);
  return std::max(ORDER_CHUNK, round_up((n + blocks - 1) / blocks, ORDER_THREADS));
}
int64_t order_blocks(int64_t n, int64_t experts) {
  const int64_t chunk = order_chunk(n, experts);
  return std::max<int64_t>(1, (n + chunk - 1) / chunk);
}

bool fine_dtype(int dtype) { return dtype == MUON_DT_F32 || dtype == MUON_DT_BF16 || dtype == MUON_DT_F16; }

// What the row kernels index by 32 bits: slots, columns, and workgroups.
int check_rows(const char* what, int dtype, int64_t tokens, int64_t top, int64_t width) {
  if (!fine_dtype(dtype)) {
    muon_set_error("%s: unsupported dtype %d", what, dtype);
    return MUON_ERR_DTYPE;
  }
  if (tokens < 0 || top < 1 || width < 0 || width > (1 << 30) || top > INT32_MAX ||
      (tokens && top > INT32_MAX / tokens)) {
    muon_set_error("%s: %lld tokens of %lld choices, width %lld: choices have to stay below 2^31 and the "
                   "width up to 2^30", what, (long long)tokens, (long long)top, (long long)width);
    return MUON_ERR_SHAPE;
  }
  return MUON_OK;
}

}  // namespace

#define BY_TYPE(CALL)                                       \
  switch (dtype) {                                          \
    case MUON_DT_F32: { constexpr int DT = MUON_DT_F32; CALL; break; }   \
    case MUON_DT_BF16: { constexpr int DT = MUON_DT_BF16; CALL; break; } \
    default: { constexpr int DT = MUON_DT_F16; CALL; }                   \
  }

extern "C" int64_t muon_expert_order_workspace_bytes(int64_t choices, int64_t experts) {
  if (choices < 0 || choices > INT32_MAX || experts < 1 || experts > ORDER_EMAX) return -1;
  const int64_t blocks = order_blocks(choices, experts);
  return blocks > 1 ? blocks * (experts + 1) * 4 : 0;
}

extern "C" int muon_expert_order(const int64_t* experts, int64_t choices, int64_t nexperts,
                                 int32_t* slots, int32_t* offsets, void* ws, void* stream) {
  if (choices < 0 || choices > INT32_MAX || nexperts < 1 || nexperts > ORDER_EMAX) {
    muon_set_error("muon_expert_order: %lld choices of %lld experts: below 2^31 of at most %d",
                   (long long)choices, (long long)nexperts, ORDER_EMAX);
    return MUON_ERR_SHAPE;
  }
  if (!offsets || (choices && (!experts || !slots)) ||
      (muon_expert_order_workspace_bytes(choices, nexperts) && !ws)) {
    muon_set_error("muon_expert_order: null pointer");
    return MUON_ERR_ARG;
  }
  OrderArgs a{experts, choices, order_chunk(choices, nexperts), (int)nexperts, (int)order_blocks(choices, nexperts),
              slots, offsets, (int32_t*)ws};
  hipStream_t s = (hipStream_t)stream;
  if (a.blocks > 1) {
    order_count_kernel<<<a.blocks, ORDER_THREADS, 0, s>>>(a);
    MUON_CHECK_LAUNCH("muon_expert_order: count");
  }
  const int lds = (ORDER_WAVES + 2) * ((int)nexperts + 1) * 4;
  order_place_kernel<<<a.blocks, ORDER_THREADS, lds, s>>>(a);
  MUON_CHECK_LAUNCH("muon_expert_order: place");
  return MUON_OK;
}

extern "C" int muon_dispatch(const void* x, int dtype, int64_t row_stride, int64_t tokens, int64_t top,
                             int64_t width, const int32_t* slots, void* rows, void* stream) {
  if (int rc = check_rows("muon_dispatch", dtype, tokens, top, width)) return rc;
  if (!tokens || !width) return MUON_OK;
  if (!x || !slots || !rows) {
    muon_set_error("muon_dispatch: null pointer");
    return MUON_ERR_ARG;
  }
  RowArgs a{x, row_stride, tokens, tokens * top, (int)top, (int)width, lanes_shift(dtype, width, 8),
            slots, nullptr, rows};
  const int64_t grid = row_grid(tokens, a.shift);
  BY_TYPE((dispatch_kernel<DT><<<(unsigned)grid, ROW_THREADS, 0, (hipStream_t)stream>>>(a)))
  MUON_CHECK_LAUNCH("muon_dispatch");
  return MUON_OK;
}

extern "C" int muon_combine(const void* rows, int dtype, int64_t row_stride, int64_t tokens, int64_t top,
                            int64_t width, const int32_t* slots, const float* gates, void* y,
                            void* stream) {
  if (int rc = check_rows("muon_combine", dtype, tokens, top, width)) return rc;
  if (!tokens || !width) return MUON_OK;
  if (!rows || !slots || !y) {
    muon_set_error("muon_combine: null pointer");
    return MUON_ERR_ARG;
  }
  RowArgs a{rows, row_stride, tokens, tokens * top, (int)top, (int)width, lanes_shift(dtype, width, 8),
            slots, gates, y};
  const int64_t grid = row_grid(tokens, a.shift);
  if (top <= 2) {
    BY_TYPE((combine_kernel<DT, 2><<<(unsigned)grid, ROW_THREADS, 0, (hipStream_t)stream>>>(a)))
  } else {
    BY_TYPE((combine_kernel<DT, 8><<<(unsigned)grid, ROW_THREADS, 0, (hipStream_t)stream>>>(a)))
  }
  MUON_CHECK_LAUNCH("muon_combine");
  return MUON_OK;
}

extern "C" int muon_combine_backward(const void* dy, int64_t dy_stride, const void* rows,
                                     int64_t row_stride, int dtype, int64_t tokens, int64_t top,
                                     int64_t width, const int32_t* slots, const float* gates,
                                     void* drows, float* dgates, void* stream) {
  if (int rc = check_rows("muon_combine_backward", dtype, tokens, top, width)) return rc;
  if (!tokens || (!drows && !dgates)) return MUON_OK;
  if (!slots || !gates || (width && (!dy || (dgates && !rows)))) {
    muon_set_error("muon_combine_backward: null pointer");
    return MUON_ERR_ARG;
  }
  BackArgs a{dy, rows, dy_stride, row_stride, tokens, tokens * top, (int)top, (int)width,
             slots, gates, drows, dgates};
  const int shift = std::max(3, lanes_shift(dtype, width, 6));
  const int64_t grid = row_grid(tokens, shift);
  hipStream_t s = (hipStream_t)stream;
#define BACK_KERNEL(G, B) BY_TYPE((combine_backward_kernel<DT, G, B><<<(unsigned)grid, ROW_THREADS, 0, s>>>(a)))
#define BACK(G) if (top == 1) { BACK_KERNEL(G, 1) } else { BACK_KERNEL(G, 8) }
  switch (shift) {
    case 3: BACK(8) break;
    case 4: BACK(16) break;
    case 5: BACK(32) break;
    default: BACK(64)
  }
#undef BACK
#undef BACK_KERNEL
  MUON_CHECK_LAUNCH("muon_combine_backward");
  return MUON_OK;
}
