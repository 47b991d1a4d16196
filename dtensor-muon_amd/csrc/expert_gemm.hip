// Products of the experts' matrices with their own rows (muon_expert_linear and its gradients). The
// rows of expert e are offsets[e] .. offsets[e + 1] - 1 of all; weights are (E, out, in):
//   FWD:  y_e  = x_e W_e^T     (rows x out, over in)
//   ROWS: dx_e = dy_e W_e      (rows x in, over out)
//   WGT:  dW_e = dy_e^T x_e    (out x in, over the expert's rows)
// Rows behind the last expert's give zeros, and reach no weight; an expert without rows gets a zero
// gradient.
//
// The offsets stay on the device, so the grid is the most tiles that R rows of E experts can make, and
// each workgroup finds its tile from the offsets; those left over end at once. 16-bit types run on
// MFMA with fp32 accumulators, fp32 on the fp32 MFMA.
//
// 64 experts of 1408 x 2048 in bf16 (an 8192-cubed library product runs at 1431 TFLOP/s, a copy at 4.9 TB/s):
//   262144 rows: FWD 1217 to 1346 us, ROWS 1259 to 1308, WGT 1186 to 1257, 1.12 to 1.27 PFLOP/s; 1408
//     fills 5.5 tiles of 256, so the matrix units do 9% more than that;
//   128 rows: 60 to 63 us, the bytes of the weights that they meet at 6 TB/s (part of them from the
//     last-level cache).
#include <algorithm>
#include <type_traits>

#include "rowops.h"

namespace {

enum { FWD = 0, ROWS = 1, WGT = 2 };

struct GArgs {
  const void* a;  // FWD: rows; ROWS, WGT: dy
  const void* b;  // FWD, ROWS: weights; WGT: rows
  void* c;        // contiguous
  int64_t lda, ldb;  // strides in elements: of the rows of a; of the rows of b
  int64_t sb;        // FWD, ROWS: elements of an expert's weights; WGT: unused
  const int32_t* offsets;
  int64_t R;  // rows in all
  int E, N, K, M;  // FWD: N out, K in; ROWS: N in, K out; WGT: M out, N in
  int tiles_m, tiles_n;  // FWD, ROWS: the most row tiles there can be
  int first;             // number of this launch's first workgroup
};
MUON_DEVICE int workgroup(const GArgs& g) { return g.first + (int)blockIdx.x; }


// The bounds of expert e's rows, whatever the offsets hold: within 0 .. R, the end no less than the
// start; the first expert's start at 0. e == E: the rows behind the last expert's.
MUON_DEVICE void bounds(const GArgs& g, int e, int& start, int& n) {
  const int R = (int)g.R;
  start = e ? std::min(std::max(g.offsets[e], 0), R) : 0;
  n = (e < g.E ? std::min(std::max(g.offsets[e + 1], start), R) : R) - start;
}

// Tiles of BY among n, up to 2^31 - 1 of them.
template <int BY>
MUON_DEVICE int tiles_in(int n) { return (int)(((unsigned)n + (BY - 1)) / BY); }

// Workgroup L's tile of `total`: one contiguous range of tiles for each of the 8 XCDs (consecutive
// workgroups are dealt round robin), so those that share panels share an L2. -1: none is left.
MUON_DEVICE int xcd_range(int L, int total) {
  const int x = L & 7, i = L >> 3, q = total >> 3, r = total & 7;
  return i < q + (x < r) ? x * q + std::min(x, r) + i : -1;
}
// A tile's row and column: GM rows of tiles for each column after the other.
MUON_DEVICE void tile_of(int t, int tiles_m, int tiles_n, int& tm, int& tn) {
  constexpr int GM = 8;
  const int group = t / (GM * tiles_n), first = group * GM, size = std::min(tiles_m - first, GM);
  const int local = t - group * (GM * tiles_n);
  tm = first + local % size;
  tn = local / size;
}

// Workgroup L's row tile of the experts one after another (g.tiles_n tiles of columns each) -> expert,
// first row, rows left of the expert from there, and column tile. Each lane counts the tiles of a few
// experts in a row; a scan over the wave gives their number, over which the workgroups are dealt, and
// the lane that has the tile. False where a workgroup is left over.
template <int BM>
MUON_DEVICE bool find_tile(const GArgs& g, int L, int& e, int& row0, int& left, int& tn) {
  const int lane = threadIdx.x & 63, per = (g.E + 64) / 64;
  const int e0 = lane * per, e1 = std::min(e0 + per, g.E + 1);
  int mine = 0, start, n;
  for (int i = e0; i < e1; ++i) {
    bounds(g, i, start, n);
    mine += tiles_in<BM>(n);
  }
  int incl = mine;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int v = __shfl_up(incl, off, 64);
    if (lane >= off) incl += v;
  }
  const int tiles_m = __shfl(incl, 63, 64);
  int t;
  L = xcd_range(L, tiles_m * g.tiles_n);
  if (L < 0) return false;
  tile_of(L, tiles_m, g.tiles_n, t, tn);
  const uint64_t past = __ballot(incl > t);
  if (!past) return false;  // offsets that do not rise can count beyond 32 bits
  const int src = __builtin_ctzll(past);
  int first = __shfl(incl - mine, src, 64);
  e = std::min(src * per, g.E);
  for (;; ++e) {
    bounds(g, e, start, n);
    const int tiles = tiles_in<BM>(n);
    if (t < first + tiles || e >= g.E) break;
    first += tiles;
  }
  e = __builtin_amdgcn_readfirstlane(e);
  const int skip = (t - first) * BM;
  row0 = __builtin_amdgcn_readfirstlane(start + skip);
  left = __builtin_amdgcn_readfirstlane(n - skip);
  return skip >= 0 && left > 0;
}

template <int DT>
MUON_DEVICE f32x4 mfma16(muon_u4 a, muon_u4 b, f32x4 c) {
  if constexpr (DT == MUON_DT_BF16) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_mfma, a),
                                                   __builtin_bit_cast(bf16x8_mfma, b), c, 0, 0, 0);
  } else {
    typedef __attribute__((ext_vector_type(8))) _Float16 h8;
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
  }
}

typedef __attribute__((ext_vector_type(2))) _Float16 muon_h2x;
// Two values to 16 bits each, to nearest even.
template <int DT>
MUON_DEVICE uint32_t pack2(float x, float y) {
  if constexpr (DT == MUON_DT_BF16)
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(muon_f2x{x, y}, muon_bf2x));
  else
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(muon_f2x{x, y}, muon_h2x));
}

// ---- 16-bit types ---------------------------------------------------------------------------
//
// Panels in LDS, one K-tile of 64 at a time. A panel whose rows run along k (KC) holds its rows of 64 k
// as 8 chunks of 16 bytes, chunk c of row r at place c ^ ((r >> 1) & 7); one whose rows are k (KR) holds
// 64 rows of the tile's width, chunk c of row k at c ^ ((k & 3) << 2) ^ (((k >> 3) & 1) << 1): both spread
// the 16 lanes of a fragment read over all banks. A KC fragment is one 16-byte read; a KR one is two
// transposing reads, each four k of one column for every lane.
constexpr int BK = 64;
typedef __attribute__((ext_vector_type(4))) short i16x4;
typedef __attribute__((address_space(3))) i16x4* lds_i16x4;

MUON_DEVICE int swz_kc(int r) { return (r >> 1) & 7; }
MUON_DEVICE int swz_kr(int k) { return ((k & 3) << 2) ^ (((k >> 3) & 1) << 1); }

// w without its first n values (16 bits each), zeros behind.
MUON_DEVICE muon_u4 drop(muon_u4 w, int n) {
  uint64_t lo = (uint64_t)w[1] << 32 | w[0], hi = (uint64_t)w[3] << 32 | w[2];
  if (n & 4) {
    lo = hi;
    hi = 0;
  }
  const int bits = 16 * (n & 3);
  if (bits) {
    lo = lo >> bits | hi << (64 - bits);
    hi >>= bits;
  }
  if (n >= 8) lo = hi = 0;
  return muon_u4{(uint32_t)lo, (uint32_t)(lo >> 32), (uint32_t)hi, (uint32_t)(hi >> 32)};
}

// One operand's share of a K-tile: PANEL rows (KC) or columns (KR) of the tile, NT threads.
//
// Every chunk is one load, at an address that no condition on a lane changes: single values behind a
// condition are waited for before the next chunk is asked for. Rows of a KC panel behind the last repeat it
// (they are not stored), a run of columns that leaves the matrix moves back to end with it, and what
// it brought too many is dropped on the way to LDS, where a k behind the last becomes zero.
template <int PANEL, bool KR, int NT, bool ALIGNED>
struct Stage {
  static constexpr int CHUNKS = PANEL * BK / 8 / NT;  // 16-byte chunks of a thread
  static constexpr int PER_ROW = KR ? PANEL / 8 : 8;
  static constexpr int ROWS_PASS = NT / PER_ROW;
  muon_u4 w[CHUNKS];

  // base: the panel's first row and column at k = 0; `in`: valid rows (KC) or columns (KR) from
  // there, k left: valid k from k0 on; wide: a row of the matrix has eight values
  MUON_DEVICE void load(const uint16_t* base, int64_t ld, int in, int k0, int kleft, bool wide) {
    const int row = threadIdx.x / PER_ROW, ch = threadIdx.x % PER_ROW * 8;
    const int cols = KR ? in : kleft, last = (KR ? kleft : in) - 1;
#pragma unroll
    for (int q = 0; q < CHUNKS; ++q) {
      const int r = std::min(row + q * ROWS_PASS, last), c = std::min(ch, cols - 8);
      const uint16_t* p = KR ? base + (k0 + r) * ld + c : base + r * ld + k0 + c;
      if (ALIGNED || wide) {
        if constexpr (ALIGNED) w[q] = *(const muon_u4*)p;
        else w[q] = load_u4(p);
      } else {  // fewer than eight columns, all of them in the first chunk
        uint32_t u[4] = {0, 0, 0, 0};
#pragma unroll
        for (int j = 0; j < 7; ++j)
          if (ch == 0 && j < cols) u[j / 2] |= (uint32_t)p[j - c] << (16 * (j & 1));
        w[q] = muon_u4{u[0], u[1], u[2], u[3]};
      }
    }
  }
  MUON_DEVICE void store(uint8_t* lds, int in, int kleft, bool wide) const {
    if (kleft < BK || (KR && in < PANEL)) {
      const int c = threadIdx.x % PER_ROW * 8, cols = KR ? in : kleft;
      const int moved = wide ? c - std::min(c, cols - 8) : 0;
#pragma unroll
      for (int q = 0; q < CHUNKS; ++q) {
        muon_u4 v = w[q];
        if constexpr (!ALIGNED) v = drop(v, moved);
        if (KR ? (int)threadIdx.x / PER_ROW + q * ROWS_PASS >= kleft : ALIGNED && moved) v = muon_u4{0, 0, 0, 0};
        put(lds, q, v);
      }
    } else {
#pragma unroll
      for (int q = 0; q < CHUNKS; ++q) put(lds, q, w[q]);
    }
  }
  static MUON_DEVICE void put(uint8_t* lds, int q, muon_u4 v) {
    const int r = threadIdx.x / PER_ROW + q * ROWS_PASS, c = threadIdx.x % PER_ROW;
    const int at = KR ? r * PANEL * 2 + ((c ^ swz_kr(r)) << 4) : r * BK * 2 + ((c ^ swz_kc(r)) << 4);
    *(muon_u4*)(lds + at) = v;
  }
};

// The same of whole K-tiles, two of which are under way: the pointers move on, and nothing depends on a
// lane, so that loads are waited for by count.
template <int PANEL, bool KR, int NT, bool ALIGNED>
struct Runs {
  typedef Stage<PANEL, KR, NT, ALIGNED> One;
  const uint16_t* p[One::CHUNKS];
  int64_t step;
  int moved;
  muon_u4 w[2][One::CHUNKS];

  MUON_DEVICE void set(const uint16_t* base, int64_t ld, int in) {
    const int row = threadIdx.x / One::PER_ROW, ch = threadIdx.x % One::PER_ROW * 8;
    const int c = KR ? std::min(ch, in - 8) : ch;
#pragma unroll
    for (int q = 0; q < One::CHUNKS; ++q) {
      const int r = row + q * One::ROWS_PASS;
      p[q] = base + (KR ? r : std::min(r, in - 1)) * ld + c;
    }
    step = KR ? BK * ld : BK;
    moved = !ALIGNED && KR && in < PANEL ? ch - c : 0;
  }
  // the K-tile at p, and on to the next one if there is one
  template <int TO>
  MUON_DEVICE void load(bool on) {
#pragma unroll
    for (int q = 0; q < One::CHUNKS; ++q) {
      if constexpr (ALIGNED) w[TO][q] = *(const muon_u4*)p[q];
      else w[TO][q] = load_u4(p[q]);
      p[q] += on ? step : 0;
    }
  }
  template <int FROM>
  MUON_DEVICE void store(uint8_t* lds, bool ragged) {
#pragma unroll
    for (int q = 0; q < One::CHUNKS; ++q) {
      muon_u4 v = w[FROM][q];
      if (!ALIGNED && ragged) v = drop(v, moved);
      One::put(lds, q, v);
    }
  }
};

// 8 consecutive k (ks 32-k substep, lane / 16) of row or column r0 + lane % 16.
template <int PANEL, bool KR>
MUON_DEVICE muon_u4 fragment(uint8_t* lds, int r0, int ks) {
  const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  if constexpr (!KR) {
    const int row = r0 + r;
    return *(const muon_u4*)(lds + row * BK * 2 + (((ks * 4 + g) ^ swz_kc(row)) << 4));
  } else {
    const int c = r0 / 8 + ((r & 3) >> 1), in = (r & 1) * 8;
    const int k = ks * 32 + g * 8 + (r >> 2);
    const uint8_t* lo = lds + k * PANEL * 2 + ((c ^ swz_kr(k)) << 4) + in;
    const uint8_t* hi = lds + (k + 4) * PANEL * 2 + ((c ^ swz_kr(k + 4)) << 4) + in;
    const i16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4)lo);
    const i16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4)hi);
    const uint64_t ua = __builtin_bit_cast(uint64_t, a), ub = __builtin_bit_cast(uint64_t, b);
    return muon_u4{(uint32_t)ua, (uint32_t)(ua >> 32), (uint32_t)ub, (uint32_t)(ub >> 32)};
  }
}

// A BM x BN tile by WM x WN waves: for few tiles and for ragged sizes (262144 rows, 64 experts of 1409 x
// 2041: 2835, 2654 and 2729 us, 530 to 570 TFLOP/s). Four waves a SIMD, two workgroups a CU.
template <int DT, int FORM, int BM, int BN, int WM, int WN, bool ALIGNED>
__global__ __launch_bounds__(64 * WM * WN, 4) void expert_gemm_kernel(GArgs g) {
  constexpr int NT = 64 * WM * WN;
  constexpr int FM = BM / WM / 16, FN = BN / WN / 16;
  constexpr bool KRA = FORM == WGT, KRB = FORM != FWD;
  constexpr int PANEL_A = BM * BK * 2, STAGE = (BM + BN) * BK * 2;
  extern __shared__ __align__(16) uint8_t smem[];

  int e, tm, tn, row0 = 0, left = 0, K, M;
  if constexpr (FORM == WGT) {
    // an expert's tiles, which take as long as its rows, on all XCDs
    const int per = g.tiles_m * g.tiles_n, L = workgroup(g);
    e = L / per;
    tile_of(L - e * per, g.tiles_m, g.tiles_n, tm, tn);
    bounds(g, e, row0, K);
    M = std::min(g.M - tm * BM, BM);
  } else {
    if (!find_tile<BM>(g, workgroup(g), e, row0, left, tn)) return;
    M = std::min(left, BM);
    K = e < g.E ? g.K : 0;
    tm = 0;
  }
  const int N = std::min(g.N - tn * BN, BN);
  const uint16_t* A = (const uint16_t*)g.a + (int64_t)row0 * g.lda + (FORM == WGT ? tm * BM : 0);
  const uint16_t* B = (const uint16_t*)g.b;
  if constexpr (FORM == FWD) B += e * g.sb + (int64_t)tn * BN * g.ldb;
  if constexpr (FORM == ROWS) B += e * g.sb + tn * BN;
  if constexpr (FORM == WGT) B += (int64_t)row0 * g.ldb + tn * BN;

  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int wm = wave % WM, wn = wave / WM;
  f32x4 acc[FM][FN];
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j) acc[i][j] = f32x4{0, 0, 0, 0};

  auto multiply = [&](int kt) {
    uint8_t* st = smem + (kt & 1) * STAGE;
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      muon_u4 fa[FM], fb[FN];
#pragma unroll
      for (int i = 0; i < FM; ++i) fa[i] = fragment<BM, KRA>(st, wm * FM * 16 + i * 16, ks);
#pragma unroll
      for (int j = 0; j < FN; ++j) fb[j] = fragment<BN, KRB>(st + PANEL_A, wn * FN * 16 + j * 16, ks);
#pragma unroll
      for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = mfma16<DT>(fb[j], fa[i], acc[i][j]);
    }
  };
  const int KT = tiles_in<BK>(K);
  const bool wide_a = (KRA ? g.M : g.K) >= 8, wide_b = (KRB ? g.N : g.K) >= 8;
  // Pairs of whole K-tiles; the last loads repeat the last of them, so that as many are under way in every
  // turn. (Few tiles gain: 8 experts of 100 x 4001, 6000 rows 76 -> 50 us, 64 of 1408 x 2048, 1024 rows 98 -> 80.
  // WGT does not, nor do ragged columns, whose runs are shifted in registers that are short then: 262144
  // rows of 64 experts of 1409 x 2041 2729 -> 3172.)
  constexpr bool AHEAD = FORM == FWD || (FORM == ROWS && ALIGNED);
  const int whole = AHEAD && (!KRB || wide_b) ? K / BK / 2 * 2 : 0;
  if (whole) {
    Runs<BM, KRA, NT, ALIGNED> ra;
    Runs<BN, KRB, NT, ALIGNED> rb;
    ra.set(A, g.lda, M);
    rb.set(B, g.ldb, N);
    auto load = [&](auto to, int kt) {
      ra.template load<decltype(to)::value>(kt + 1 < whole);
      rb.template load<decltype(to)::value>(kt + 1 < whole);
    };
    auto store = [&](auto from, int kt) {
      ra.template store<decltype(from)::value>(smem + (kt & 1) * STAGE, KRA && M < BM);
      rb.template store<decltype(from)::value>(smem + (kt & 1) * STAGE + PANEL_A, KRB && N < BN);
    };
    typedef std::integral_constant<int, 0> Zero;
    typedef std::integral_constant<int, 1> One;
    load(Zero{}, 0);
    load(One{}, 1);
    store(Zero{}, 0);
    load(Zero{}, 2);
    __syncthreads();
#pragma unroll 1
    for (int kt = 0; kt < whole; kt += 2) {
      multiply(kt);
      store(One{}, kt + 1);
      load(One{}, kt + 3);
      __syncthreads();
      multiply(kt + 1);
      store(Zero{}, kt + 2);
      load(Zero{}, kt + 4);
      __syncthreads();
    }
  }
  if (whole < KT) {
    Stage<BM, KRA, NT, ALIGNED> sa;
    Stage<BN, KRB, NT, ALIGNED> sb;
    auto load = [&](int kt) {
      sa.load(A, g.lda, M, kt * BK, K - kt * BK, wide_a);
      sb.load(B, g.ldb, N, kt * BK, K - kt * BK, wide_b);
    };
    auto store = [&](int kt) {
      sa.store(smem + (kt & 1) * STAGE, M, K - kt * BK, wide_a);
      sb.store(smem + (kt & 1) * STAGE + PANEL_A, N, K - kt * BK, wide_b);
    };
    load(whole);
    store(whole);
    __syncthreads();
#pragma unroll 1
    for (int kt = whole; kt < KT; ++kt) {
      if (kt + 1 < KT) load(kt + 1);
      multiply(kt);
      if (kt + 1 < KT) store(kt + 1);
      __syncthreads();
    }
  }

  // the b fragment is the first operand: a lane holds four consecutive columns of one row
  const int r = lane & 15, gq = lane >> 4;
  uint16_t* C = (uint16_t*)g.c + (FORM == WGT ? ((int64_t)e * g.M + tm * BM) * g.N : (int64_t)row0 * g.N);
#pragma unroll
  for (int i = 0; i < FM; ++i) {
    const int m = wm * FM * 16 + i * 16 + r;
    if (m >= M) continue;
    uint16_t* out = C + (int64_t)m * g.N + tn * BN;
#pragma unroll
    for (int j = 0; j < FN; ++j) {
      const int n = wn * FN * 16 + j * 16 + gq * 4;
      const uint32_t lo = pack2<DT>(acc[i][j][0], acc[i][j][1]), hi = pack2<DT>(acc[i][j][2], acc[i][j][3]);
      if (ALIGNED ? n < N : n + 4 <= N) {
        if constexpr (ALIGNED) {
          *(uint2*)(out + n) = make_uint2(lo, hi);
        } else {
          const uint2 v = make_uint2(lo, hi);
          __builtin_memcpy(out + n, &v, 8);
        }
      } else if (!ALIGNED) {
        const uint32_t u[2] = {lo, hi};
#pragma unroll
        for (int q = 0; q < 4; ++q)
          if (n + q < N) out[n + q] = (uint16_t)(u[q / 2] >> (16 * (q & 1)));
      }
    }
  }
}

// ---- 16-bit types, whole 16-byte runs: operands straight to LDS --------------------------------
//
// 256 x 256 tile, K-tiles of 64, four waves of 128 x 128 (8 x 8 accumulators of 16 x 16). A K-tile is two
// steps, of the upper and of the lower 64 rows of every wave, over all 64 k. The panels of two K-tiles
// stand in LDS, that of a as two halves of the rows of one step each; they come by loads that write LDS
// themselves. A step multiplies one set of fragments while the next step's are read, so that during K-tile t
//   step 0 reads the lower a of t, and loads the b of t + 2 into the place of t's;
//   step 1 reads the b and the upper a of t + 1, and loads the a of t + 2 into the places of t's:
// each load has two to three steps to arrive, and covers whole lines of 128 bytes along k. (With steps
// of 32 k of all rows, whose loads take half lines of a KC panel, FWD ran at 1141 TFLOP/s where WGT did
// at 1228.)
//
// Nothing is masked beyond what the buffer's size cuts off (what lies behind it arrives as zeros): rows and
// columns of a tile behind its own are others' values or zeros, and are not stored. Along k, a KR panel's
// buffer ends with its last k; of a KC panel the lanes behind the last k point behind the buffer.
constexpr int P_HALF = 128 * BK * 2, P_PANEL = 2 * P_HALF, P_STAGE = 2 * P_PANEL;
constexpr int P_OUT_ROW = 256 + 16, P_OUT = 16 * P_OUT_ROW;  // a wave's rows on their way out
typedef __attribute__((ext_vector_type(4))) unsigned int u32x4;

// One load of 1 KB, 16 bytes a lane in order, to the LDS address m0, which takes a wait state. Scalar
// registers that a vector instruction wrote (a readfirstlane) take five before a load reads them, which
// the compiler does not see here: scalar_wait, or products, stand between.
MUON_DEVICE void dma_1k(u32x4 rs, uint32_t vo, uint32_t so, uint32_t m0) {
  asm volatile("s_mov_b32 m0, %3\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, %2 offen lds"
               ::"v"(vo), "s"(rs), "s"(so), "s"(m0) : "m0");
}

MUON_DEVICE void scalar_wait() {
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("s_nop 7" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}

// One operand of a tile as its loads see it, 8 a K-tile for each wave. SPLIT: the a panel, in halves of
// the first and the second 64 of every 128 rows (KC) or columns (KR).
template <bool KR, bool SPLIT>
struct Source {
  const char* base;  // where the buffer begins: the panel at k = 0, or a later k
  int64_t bytes;     // from there to the end of what may be read
  u32x4 rs;          // the buffer
  uint32_t so;       // the next K-tile's offset in it
  uint32_t step;     // bytes of a row
  uint32_t vo[2];    // this lane's place: of even and odd loads (KR), or of all K-tiles and of the last (KC)

  // rows: from the panel's first row (KC) or k = 0 (KR); columns: k (KC) or from the panel's first (KR)
  MUON_DEVICE void set(const uint16_t* p, int64_t ld, int64_t rows, int columns, int K) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    base = (const char*)p;
    step = (uint32_t)ld * 2;
    bytes = rows && columns ? ((rows - 1) * ld + columns) * 2 : 0;
    buffer();
    if constexpr (KR && SPLIT) {  // four k a load, 16 chunks of each
      const int r = wave * 4 + (lane >> 4), c = (lane & 15) ^ swz_kr(r);
      vo[0] = vo[1] = r * step + (c & 7) * 16 + (c >> 3) * 256;
    } else if constexpr (KR) {  // two k a load, 32 chunks
      const int r = wave * 2 + (lane >> 5), c = (lane & 31) ^ ((r & 3) << 2);
      vo[0] = r * step + c * 16;
      vo[1] = r * step + (c ^ 2) * 16;
    } else {  // eight rows a load, 8 chunks
      const int r = wave * 8 + (lane >> 3), c = (lane & 7) ^ swz_kc(r);
      vo[0] = r * step + c * 16;
      vo[1] = c * 8 < K - std::max(0, (K - 1) / BK) * BK ? vo[0] : 0x80000000u;
    }
  }
  MUON_DEVICE void buffer() {
    const uint64_t a = (uint64_t)base;
    const uint32_t n = bytes <= 0 ? 0u : (uint32_t)std::min<int64_t>(bytes, 0x7fffffff);
    rs = u32x4{(uint32_t)__builtin_amdgcn_readfirstlane((int)a),
               (uint32_t)__builtin_amdgcn_readfirstlane((int)(a >> 32)) & 0xffffu,
               (uint32_t)__builtin_amdgcn_readfirstlane((int)n), 0x00020000u};
    so = 0;
  }
  // Nothing is left: loads write zeros. The compiler moved the bare insertion of the 0 onto one of the ways to
  // here, and left the buffer unwritten on the other, where no tile is left: loads of a garbage buffer. What an
  // asm returns stays in its place.
  MUON_DEVICE void close() {
    rs[2] = 0;
    asm volatile("" : "+s"(rs));
  }
  // To the next K-tile; long before the offset leaves 31 bits the buffer begins anew.
  MUON_DEVICE void advance() {
    so += KR ? BK * step : BK * 2;
    if (KR && so >= (1u << 30)) {
      base += so;
      bytes -= so;
      buffer();
    }
  }
  // load q of 8 of this wave (SPLIT: 4 of either half; `last`: K's last K-tile) to LDS at `to`
  MUON_DEVICE void load(int q, bool last, uint32_t to) const {
    const int h = q >> 2, p = q & 3;
    uint32_t at;
    if constexpr (KR && SPLIT) at = p * 16 * step + h * 128;
    else if constexpr (KR) at = q * 8 * step;
    else if constexpr (SPLIT) at = ((p >> 1) * 128 + h * 64 + (p & 1) * 32) * step;
    else at = q * 32 * step;
    dma_1k(rs, KR ? vo[q & 1] : last ? vo[1] : vo[0], so + at, to + q * 4096);
  }
};

// acc += a b with the accumulator in AGPRs all along: left to the compiler, the 64 of a wave are copied
// between registers in every K-tile.
template <int DT>
MUON_DEVICE void mfma_acc(f32x4& c, muon_u4 a, muon_u4 b) {
  if constexpr (DT == MUON_DT_BF16)
    asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
  else
    asm volatile("v_mfma_f32_16x16x32_f16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
}
// c = 0, by a product of zeros: what other instructions wrote would have to be waited for, and the
// compiler, which does not see that, puts such writes right before the products.
template <int DT>
MUON_DEVICE void mfma_zero(f32x4& c, muon_u4 zero) {
  if constexpr (DT == MUON_DT_BF16)
    asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %1, 0" : "=a"(c) : "v"(zero));
  else
    asm volatile("v_mfma_f32_16x16x32_f16 %0, %1, %1, 0" : "=a"(c) : "v"(zero));
}
// Reads of the accumulators by other instructions wait for the last product, as do vector
// instructions' results that products read.
MUON_DEVICE void mfma_wait() {
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 7" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}

// The tiles of a launch as its workgroups walk them, one workgroup a CU. Neighbouring tiles, whose panels
// are the same, are dealt to one XCD (workgroups go to the 8 round robin), whose L2 they meet in.
// FWD, ROWS: the XCDs have contiguous ranges of equal numbers of tiles, each workgroup every 32nd of them.
// WGT, where a tile lasts as long as its expert has rows: the experts' tiles from the longest on, in
// rounds of 256 that are dealt out in turn from the first workgroup on and from the last one, so that
// what a round gives one more of the next gives it less of.
constexpr int P_GROUPS = 256, P_LANE = P_GROUPS / 8;
struct Tile {
  int e, row0, tm, tn, M, N, K;  // row0: the first of the tile's rows (WGT: of the expert's)
};
template <int FORM>
struct Walk {
  const GArgs& g;
  // in LDS, E + 2 of each: row tiles before each expert (WGT: the experts from the one of most rows on),
  // its first row and its rows
  int *first, *start_of, *rows_of;
  int at, end;  // next tile (WGT: round) of this workgroup, and the last ones' end

  static constexpr int NEXT = FORM == WGT ? 1 : P_LANE;

  MUON_DEVICE Walk(const GArgs& g_, int* lds)
      : g(g_), first(lds), start_of(lds + g_.E + 2), rows_of(lds + 2 * (g_.E + 2)) {
    for (int i = threadIdx.x; i <= g.E; i += 256) {
      int start, n;
      bounds(g, i, start, n);
      start_of[i] = start;
      rows_of[i] = n;
    }
    __syncthreads();
    if constexpr (FORM == WGT) {
      for (int i = threadIdx.x; i < g.E; i += 256) {
        int rank = 0;
        const int mine = rows_of[i];
        for (int k = 0; k < g.E; ++k) rank += rows_of[k] > mine || (rows_of[k] == mine && k < i);
        first[rank] = i;
      }
      __syncthreads();
      at = 0;
      end = (g.E * g.tiles_m * g.tiles_n + P_GROUPS - 1) / P_GROUPS;
    } else {
      const int lane = threadIdx.x & 63, per = (g.E + 64) / 64;
      const int e0 = lane * per, e1 = std::min(e0 + per, g.E + 1);
      int mine = 0;
      for (int i = e0; i < e1; ++i) mine += tiles_in<256>(rows_of[i]);
      int incl = mine;
#pragma unroll
      for (int off = 1; off < 64; off <<= 1) {
        const int v = __shfl_up(incl, off, 64);
        if (lane >= off) incl += v;
      }
      if (threadIdx.x < 64) {
        int sum = incl - mine;
        for (int i = e0; i < e1; ++i) {
          first[i] = sum;
          sum += tiles_in<256>(rows_of[i]);
        }
        if (e1 == g.E + 1 && e0 < e1) first[g.E + 1] = sum;
      }
      __syncthreads();
      const int64_t x = blockIdx.x & 7, all = (int64_t)__builtin_amdgcn_readfirstlane(first[g.E + 1]) * g.tiles_n;
      at = (int)(all * x / 8) + (int)(blockIdx.x >> 3);
      end = (int)(all * (x + 1) / 8);
    }
  }
  // The expert whose row tiles hold number t.
  MUON_DEVICE int expert(int t) const {
    const int lane = threadIdx.x & 63, per = (g.E + 64) / 64;
    const int seg = __popcll(__ballot(lane * per <= g.E && first[std::min(lane * per, g.E)] <= t)) - 1;
    const int i = seg * per + lane;
    const int in = __popcll(__ballot(lane < per && i <= g.E && first[std::min(i, g.E)] <= t));
    return std::max(0, std::min(seg * per + in - 1, g.E));
  }
  MUON_DEVICE bool tile(int t, Tile& o) const {
    if (t >= end) return false;
    if constexpr (FORM == WGT) {
      const int per = g.tiles_m * g.tiles_n;
      // of a round of n tiles, fewer in the last one, an XCD has an eighth
      const int n = std::min(g.E * per - t * P_GROUPS, P_GROUPS), x = blockIdx.x & 7;
      int k = n * x / 8 + (int)(blockIdx.x >> 3);
      if (k >= n * (x + 1) / 8) return false;  // none in the last round
      k = t * P_GROUPS + (t & 1 ? n - 1 - k : k);
      const int rank = k / per;
      o.e = __builtin_amdgcn_readfirstlane(first[rank]);
      tile_of(k - rank * per, g.tiles_m, g.tiles_n, o.tm, o.tn);
      o.row0 = start_of[o.e];
      o.K = rows_of[o.e];
      o.M = std::min(g.M - o.tm * 256, 256);
    } else {
      int row;
      tile_of(t, __builtin_amdgcn_readfirstlane(first[g.E + 1]), g.tiles_n, row, o.tn);
      o.e = expert(row);
      const int skip = (row - first[o.e]) * 256, rows = rows_of[o.e];
      const bool fine = skip >= 0 && skip < rows;  // also where offsets that fall count beyond 32 bits
      o.row0 = start_of[o.e] + (fine ? skip : 0);
      o.M = fine ? std::min(rows - skip, 256) : 0;
      o.K = fine && o.e < g.E ? g.K : 0;
      o.tm = 0;
    }
    o.N = std::min(g.N - o.tn * 256, 256);
#define UNIFORM(X) o.X = __builtin_amdgcn_readfirstlane(o.X)
    UNIFORM(e); UNIFORM(row0); UNIFORM(tm); UNIFORM(tn); UNIFORM(M); UNIFORM(N); UNIFORM(K);
#undef UNIFORM
    return true;
  }
};

// K-tiles go by twos, since two sets of b fragments take turns; one at least, of nothing, so that every
// tile is written.
MUON_DEVICE int k_pairs(int K) { return std::max(1, tiles_in<2 * BK>(K)); }

template <int DT, int FORM>
__global__ __launch_bounds__(256, 1) void expert_gemm_pipe_kernel(GArgs g) {
  constexpr int BM = 256, BN = 256;
  constexpr bool KRA = FORM == WGT, KRB = FORM != FWD;
  extern __shared__ __align__(16) uint8_t smem[];
  Walk<FORM> walk(g, (int*)(smem + 2 * P_STAGE + 4 * P_OUT));
  Tile t;
  if (!walk.tile(walk.at, t)) return;

  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int wm = wave & 1, wn = wave >> 1;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)smem + wave * 1024;

  // What the loads are at: a tile's sources, and its next K-tile. They run two K-tiles ahead of the
  // products, across tiles.
  Source<KRA, true> a;
  Source<KRB, false> b;
  int next = walk.at, kt_next = 0, kt_last = 0, kt_all = 0;
  auto open = [&](const Tile& o) {
    const uint16_t *A = (const uint16_t*)g.a, *B = (const uint16_t*)g.b;
    if constexpr (FORM == WGT) {
      a.set(A + (int64_t)o.row0 * g.lda + o.tm * BM, g.lda, o.K, g.M - o.tm * BM, o.K);
      b.set(B + (int64_t)o.row0 * g.ldb + o.tn * BN, g.ldb, o.K, g.N - o.tn * BN, o.K);
    } else {
      a.set(A + (int64_t)o.row0 * g.lda, g.lda, o.K ? g.R - o.row0 : 0, g.K, o.K);
      if constexpr (FORM == FWD)
        b.set(B + o.e * g.sb + (int64_t)o.tn * BN * g.ldb, g.ldb,
              o.K ? (int64_t)(g.E - o.e) * g.N - o.tn * BN : 0, g.K, o.K);
      else
        b.set(B + o.e * g.sb + o.tn * BN, g.ldb, o.K, g.N - o.tn * BN, o.K);
    }
    kt_next = 0;
    kt_last = tiles_in<BK>(o.K) - 1;
    kt_all = 2 * k_pairs(o.K);
  };
  // to the next K-tile, of the next tile where this one has no more
  auto advance = [&] {
    a.advance();
    b.advance();
    if (++kt_next <= kt_last) return;
    if (kt_next >= kt_all) {
      next += walk.NEXT;
      Tile o;
      if (walk.tile(next, o)) {
        open(o);
        return;
      }
    }
    a.close();  // the second of a pair that has one, or no more tiles
    b.close();
  };
  auto load_a = [&](int q, int st) { a.load(q, kt_next == kt_last, lds0 + st * P_STAGE); };
  auto load_b = [&](int q, int st) { b.load(q, kt_next == kt_last, lds0 + st * P_STAGE + P_PANEL); };
  f32x4 acc[8][8];
  muon_u4 fa[2][8], fb[2][16];  // [k half * 4 + i], [k half * 8 + j], of two steps and of two K-tiles
  auto read_a = [&](int half, int st, int n) {
    fa[half][n] = fragment<KRA ? 128 : 256, KRA>(smem + st * P_STAGE + half * P_HALF, wm * 64 + (n & 3) * 16, n >> 2);
  };
  auto read_b = [&](int to, int st, int n) {
    fb[to][n] = fragment<BN, KRB>(smem + st * P_STAGE + P_PANEL, wn * 128 + (n & 7) * 16, n >> 3);
  };
  // Step `half` of the K-tile in place st (`set`, the b fragments): 64 products, and between them the reads
  // of the next step's fragments and the loads. A wave issues in order, and each product leaves
  // three slots before the next can start: what stands together between two products holds the
  // second one up.
  int stores = 0;  // a bit for each step whose end does not wait for a finished tile's stores
  auto step = [&](auto half_c, auto set_c) {
    constexpr int half = decltype(half_c)::value, set = decltype(set_c)::value;
#pragma unroll
    for (int n = 0; n < 64; ++n) {
      const int ks = n >> 5, i = (n >> 3) & 3, j = n & 7;
      mfma_acc<DT>(acc[half * 4 + i][j], fb[set][ks * 8 + j], fa[half][ks * 4 + i]);
      if (half == 0 && n % 4 == 1 && n < 32) {
        __builtin_amdgcn_sched_barrier(0);
        read_a(1, set, n / 4);
      }
      if (half == 1 && n % 2 == 1 && n < 48) {
        __builtin_amdgcn_sched_barrier(0);
        if (n < 32) read_b(set ^ 1, set ^ 1, n / 2);
        else read_a(0, set ^ 1, n / 2 - 16);
      }
      if (n % 8 == 6) {
        if (half == 0) load_b(n / 8, set);
        else load_a(n / 8, set);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    // What the next step reads has arrived: at the end of step 0 the b and upper a of the next K-tile, at
    // that of step 1 its lower a. Newer than those are 4 + 8 or 8 + 8 loads, and, right after a tile, its 32 stores.
    if constexpr (half == 0)
      asm volatile("s_waitcnt vmcnt(44) lgkmcnt(0)\n\ts_cmp_lg_u32 %0, 0\n\ts_cbranch_scc1 .Lstores%=\n\t"
                   "s_waitcnt vmcnt(12)\n.Lstores%=:\n\ts_barrier" ::"s"(stores) : "scc", "memory");
    else
      asm volatile("s_waitcnt vmcnt(48) lgkmcnt(0)\n\ts_cmp_lg_u32 %0, 0\n\ts_cbranch_scc1 .Lstores%=\n\t"
                   "s_waitcnt vmcnt(16)\n.Lstores%=:\n\ts_barrier" ::"s"(stores) : "scc", "memory");
    stores >>= 1;
    __builtin_amdgcn_sched_barrier(0);
  };
  typedef std::integral_constant<int, 0> Zero;
  typedef std::integral_constant<int, 1> One;
  open(t);
#pragma unroll
  for (int st = 0; st < 2; ++st) {
    scalar_wait();
#pragma unroll
    for (int q = 0; q < 8; ++q) load_b(q, st);
#pragma unroll
    for (int q = 0; q < 8; ++q) load_a(q, st);
    advance();
  }
  asm volatile("s_waitcnt vmcnt(16)\n\ts_barrier" ::: "memory");
#pragma unroll
  for (int n = 0; n < 16; ++n) read_b(0, 0, n);
#pragma unroll
  for (int n = 0; n < 8; ++n) read_a(0, 0, n);
  // every wave has these fragments before their place is loaded anew
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");

  for (int at = walk.at;;) {
    const int pairs = k_pairs(t.K);
    const muon_u4 zero = {0, 0, 0, 0};
    mfma_wait();
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) mfma_zero<DT>(acc[i][j], zero);
#pragma clang loop unroll(disable)
    for (int p = 0; p < pairs; ++p) {
      step(Zero{}, Zero{});
      step(One{}, Zero{});
      advance();
      step(Zero{}, One{});
      step(One{}, One{});
      advance();
    }
    mfma_wait();

    // 16 rows of the wave's 128 columns at a time through its own LDS: a lane has four consecutive columns
    // of one row, and stores 16 bytes of a line; what is none of the tile's points behind the buffer,
    // so that every wave has 32 stores
    int r = lane & 15, l = lane >> 4;
    asm volatile("" : "+v"(r), "+v"(l));  // or their products are made before the loop, and spilled
    uint8_t* mine = smem + 2 * P_STAGE + wave * P_OUT;
    const int c = wn * 128 + r * 8, m = t.M - wm * 128 - l;
    const uint64_t out = (uint64_t)((uint16_t*)g.c + (FORM == WGT ? (int64_t)t.e * g.M + t.tm * BM : (int64_t)t.row0) * g.N +
                                    (int64_t)(wm * 128) * g.N + t.tn * BN);
    const __amdgpu_buffer_rsrc_t rc = __builtin_amdgcn_make_buffer_rsrc((void*)out, 0, 0x7fffffff, 0x00020000);
    const uint32_t vo = c < t.N ? (uint32_t)l * g.N * 2 + c * 2 : 0x80000000u;
    const uint32_t four = (uint32_t)g.N * 8;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t w[2] = {pack2<DT>(acc[i][j][0], acc[i][j][1]), pack2<DT>(acc[i][j][2], acc[i][j][3])};
        __builtin_memcpy(__builtin_assume_aligned(mine + r * P_OUT_ROW + j * 32 + l * 8, 8), w, 8);
      }
#pragma unroll
      for (int p = 0; p < 4; ++p) {
        muon_u4 w;
        __builtin_memcpy(&w, __builtin_assume_aligned(mine + (p * 4 + l) * P_OUT_ROW + r * 16, 16), 16);
        __builtin_amdgcn_raw_buffer_store_b128(w, rc, i * 16 + p * 4 < m ? vo : 0x80000000u, (i * 4 + p) * four, 0);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    stores = 3;
    at += walk.NEXT;
    if (!walk.tile(at, t)) break;
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the last loads, of nothing, into this LDS
}

// ---- 16-bit types, few rows an expert ---------------------------------------------------------
//
// y = x W_e^T where every expert has a few rows (single tokens): the weights are read once and nothing
// else counts. A workgroup has 16 rows of an expert and 32 columns of its output, its four waves a quarter
// of k each. Fragments come from memory as the products take them, 16 weight rows by 64 bytes a load,
// several of them under way in every wave; the four sums are joined through LDS in fixed order.
constexpr int R_N = 32, R_DEEP = 4;  // columns of a workgroup; k fragments under way

// 8 values of a row from k on, 0 behind K.
template <bool ALIGNED>
MUON_DEVICE muon_u4 row_fragment(const uint16_t* row, int k, int K) {
  if (k + 8 <= K) {
    if constexpr (ALIGNED) return *(const muon_u4*)(row + k);
    else return load_u4(row + k);
  }
  uint32_t u[4] = {0, 0, 0, 0};
  if constexpr (!ALIGNED) {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (k + j < K) u[j / 2] |= (uint32_t)row[k + j] << (16 * (j & 1));
  }
  return muon_u4{u[0], u[1], u[2], u[3]};
}

template <int DT, bool ALIGNED>
__global__ __launch_bounds__(256) void expert_rows_kernel(GArgs g) {
  __shared__ f32x4 part[4][2][64];
  int e, row0, left, tn;
  if (!find_tile<16>(g, workgroup(g), e, row0, left, tn)) return;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, r = lane & 15, gq = lane >> 4;
  const int K = e < g.E ? g.K : 0, n0 = tn * R_N;
  // rows and columns behind the last ones repeat them, and are not stored
  const uint16_t* w[2];
#pragma unroll
  for (int j = 0; j < 2; ++j)
    w[j] = (const uint16_t*)g.b + (e < g.E ? e : 0) * g.sb + (int64_t)std::min(n0 + j * 16 + r, g.N - 1) * g.ldb;
  const uint16_t* x = (const uint16_t*)g.a + (int64_t)(row0 + std::min(r, left - 1)) * g.lda;
  f32x4 acc[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
  const int quarter = (K + 127) / 128 * 32;
  const int end = std::min((wave + 1) * quarter, K);
  for (int k0 = wave * quarter; k0 < end; k0 += 32 * R_DEEP) {
    muon_u4 fw[R_DEEP][2], fx[R_DEEP];
#pragma unroll
    for (int d = 0; d < R_DEEP; ++d) {
      const int k = k0 + d * 32 + gq * 8;
#pragma unroll
      for (int j = 0; j < 2; ++j) fw[d][j] = row_fragment<ALIGNED>(w[j], k, end);
      fx[d] = row_fragment<ALIGNED>(x, k, end);
    }
#pragma unroll
    for (int d = 0; d < R_DEEP; ++d)
#pragma unroll
      for (int j = 0; j < 2; ++j) acc[j] = mfma16<DT>(fw[d][j], fx[d], acc[j]);
  }
#pragma unroll
  for (int j = 0; j < 2; ++j) part[wave][j][lane] = acc[j];
  __syncthreads();
  if (wave >= 2 || r >= left) return;
  f32x4 v = part[0][wave][lane];
#pragma unroll
  for (int q = 1; q < 4; ++q) v += part[q][wave][lane];
  const int n = n0 + wave * 16 + gq * 4;
  uint16_t* out = (uint16_t*)g.c + (int64_t)(row0 + r) * g.N + n;
  const uint32_t u[2] = {pack2<DT>(v[0], v[1]), pack2<DT>(v[2], v[3])};
  if (n + 4 <= g.N) {
    __builtin_memcpy(out, u, 8);
  } else {
#pragma unroll
    for (int q = 0; q < 4; ++q)
      if (n + q < g.N) out[q] = (uint16_t)(u[q / 2] >> (16 * (q & 1)));
  }
}

// ---- fp32 -----------------------------------------------------------------------------------
//
// 128 x 128 or 64 x 64 tile (S blocks of 32 a wave and side, 2 or 1), K-tiles of 16, four waves on
// v_mfma_f32_32x32x2_f32. Panels stand in LDS as they do in memory, rows 4 values apart from whole ones. A
// lane holds four k in a row for four products, the other half of the wave the next four: in that order a KC
// fragment of all four is one read. The sums of 256 k are added up apart from the products' own: a
// sum that runs over all of k takes a rounding of its whole size at each. 4094 rows of 8 experts of
// 1001 x 769: 72 to 76 us each among many passes, 83 to 87 TFLOP/s of 154 (8192 cubed): about 1090 tiles of
// 64, so that some CUs have five of them and others four, whose edges hold a tenth of nothing. Two K-tiles
// are under way, in counted loads (with one, behind conditions, all three took 255 us for 220 to 227). More
// of these workgroups on a CU help, wider tiles and K-tiles do not.
constexpr int F_K = 16, F_SUM = 256 / F_K;

// A thread's V = 4 S values: KR: of row k; KC: of row r, V k in a row.
template <bool KR, int V>
MUON_DEVICE void f32_load(float (&w)[V], const float* base, int64_t ld, int in, int k0, int kleft) {
  const int tid = threadIdx.x;
  constexpr int EACH = F_K / V;  // threads of a KC row
  const int row = KR ? tid / 16 : tid / EACH, ch = KR ? tid % 16 * V : tid % EACH * V;
  const bool ok = KR ? row < kleft : row < in;
  const int have = ok ? (KR ? in : kleft) - ch : 0;
  const float* p = KR ? base + (k0 + row) * ld + ch : base + row * ld + k0 + ch;
  if (have >= V) {
    __builtin_memcpy(w, p, 4 * V);
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) w[j] = j < have ? p[j] : 0.0f;
  }
}
template <bool KR, int V>
MUON_DEVICE void f32_store(float* lds, const float (&w)[V]) {
  constexpr int EACH = KR ? 16 : F_K / V, P = KR ? 16 * V + 4 : F_K + 4;
  float* p = lds + (int)threadIdx.x / EACH * P + threadIdx.x % EACH * V;
#pragma unroll
  for (int j = 0; j < V; j += 4) *(float4*)(p + j) = make_float4(w[j], w[j + 1], w[j + 2], w[j + 3]);
}
// A thread's values of whole K-tiles, whose loads no condition delays: rows behind the last repeat it, and a
// run of columns that would leave the matrix moves back to end with it (`moved` values) and drops them on
// the way to LDS.
template <bool KR, int V>
struct F32Source {
  const float* p;
  int64_t step;
  int moved;
  float w[2][V];  // K-tiles under way

  MUON_DEVICE void set(const float* base, int64_t ld, int in) {
    constexpr int EACH = KR ? 16 : F_K / V;
    const int row = threadIdx.x / EACH, ch = threadIdx.x % EACH * V, c = KR ? std::min(ch, in - V) : ch;
    p = base + (KR ? row : std::min(row, in - 1)) * ld + c;
    step = KR ? F_K * ld : F_K;
    moved = KR && in < 16 * V ? ch - c : 0;
  }
  // the K-tile at p, and on to the next one if there is one
  template <int TO>
  MUON_DEVICE void load(bool on) {
    __builtin_memcpy(w[TO], p, 4 * V);
    p += on ? step : 0;
  }
  template <int FROM>
  MUON_DEVICE void store(float* lds, bool ragged) {
    if (ragged) {
#pragma unroll
      for (int bit = 1; bit < V; bit *= 2)
#pragma unroll
        for (int j = 0; j < V; ++j)
          if (moved & bit) w[FROM][j] = j + bit < V ? w[FROM][j + bit] : 0.0f;
    }
    f32_store<KR, V>(lds, w[FROM]);
  }
};
// Values k .. k + 3 of row or column r of a panel.
template <bool KR, int V>
MUON_DEVICE f32x4 f32_fragment(const float* lds, int r, int k) {
  constexpr int P = KR ? 16 * V + 4 : F_K + 4;
  if constexpr (!KR) return *(const f32x4*)(lds + r * P + k);
  f32x4 v;
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] = lds[(k + j) * P + r];
  return v;
}

template <int FORM, int S>
__global__ __launch_bounds__(256, 2) void expert_gemm_f32_kernel(GArgs g) {
  constexpr int F_B = 64 * S, V = 4 * S;
  constexpr bool KRA = FORM == WGT, KRB = FORM != FWD;
  __shared__ __align__(16) float lds[2][2][F_B * (F_K + 4)];
  int e, tm, tn, row0 = 0, left = 0, K, M;
  if constexpr (FORM == WGT) {
    const int per = g.tiles_m * g.tiles_n, L = workgroup(g);
    e = L / per;
    tile_of(L - e * per, g.tiles_m, g.tiles_n, tm, tn);
    bounds(g, e, row0, K);
    M = std::min(g.M - tm * F_B, F_B);
  } else {
    if (!find_tile<F_B>(g, workgroup(g), e, row0, left, tn)) return;
    M = std::min(left, F_B);
    K = e < g.E ? g.K : 0;
    tm = 0;
  }
  const int N = std::min(g.N - tn * F_B, F_B);
  const float* A = (const float*)g.a + (int64_t)row0 * g.lda + (FORM == WGT ? tm * F_B : 0);
  const float* B = (const float*)g.b;
  if constexpr (FORM == FWD) B += e * g.sb + (int64_t)tn * F_B * g.ldb;
  if constexpr (FORM == ROWS) B += e * g.sb + tn * F_B;
  if constexpr (FORM == WGT) B += (int64_t)row0 * g.ldb + tn * F_B;

  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, wm = wave & 1, wn = wave >> 1;
  const int fr = lane & 31, fk = lane >> 5;
  f32x16 acc[S][S], sum[S][S];
#pragma unroll
  for (int i = 0; i < S; ++i)
#pragma unroll
    for (int j = 0; j < S; ++j)
#pragma unroll
      for (int q = 0; q < 16; ++q) acc[i][j][q] = sum[i][j][q] = 0.0f;
  auto multiply = [&](int kt) {
    const float* la = lds[kt & 1][0];
    const float* lb = lds[kt & 1][1];
#pragma unroll
    for (int k = 0; k < F_K; k += 8) {
      f32x4 fa[S], fb[S];
#pragma unroll
      for (int i = 0; i < S; ++i) {
        fa[i] = f32_fragment<KRA, V>(la, wm * 32 * S + i * 32 + fr, k + fk * 4);
        fb[i] = f32_fragment<KRB, V>(lb, wn * 32 * S + i * 32 + fr, k + fk * 4);
      }
#pragma unroll
      for (int q = 0; q < 4; ++q)
#pragma unroll
        for (int i = 0; i < S; ++i)
#pragma unroll
          for (int j = 0; j < S; ++j)
            acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x2f32(fb[j][q], fa[i][q], acc[i][j], 0, 0, 0);
    }
    if (kt % F_SUM == F_SUM - 1) {
#pragma unroll
      for (int i = 0; i < S; ++i)
#pragma unroll
        for (int j = 0; j < S; ++j)
#pragma unroll
          for (int q = 0; q < 16; ++q) {
            sum[i][j][q] += acc[i][j][q];
            acc[i][j][q] = 0.0f;
          }
    }
  };
  // Whole K-tiles: while one is multiplied the next two are under way. The last loads repeat the last K-tile, so
  // that as many are under way in every turn.
  const int KT = tiles_in<F_K>(K);
  const int whole = (KRA ? g.M >= V : true) && (KRB ? g.N >= V : true) ? K / F_K / 2 * 2 : 0;
  if (whole) {
    F32Source<KRA, V> sa;
    F32Source<KRB, V> sb;
    sa.set(A, g.lda, M);
    sb.set(B, g.ldb, N);
    const bool ra = KRA && M < F_B, rb = KRB && N < F_B;
    auto load = [&](auto to, int kt) {
      sa.template load<decltype(to)::value>(kt + 1 < whole);
      sb.template load<decltype(to)::value>(kt + 1 < whole);
    };
    auto store = [&](auto from, int kt) {
      sa.template store<decltype(from)::value>(lds[kt & 1][0], ra);
      sb.template store<decltype(from)::value>(lds[kt & 1][1], rb);
    };
    typedef std::integral_constant<int, 0> Zero;
    typedef std::integral_constant<int, 1> One;
    load(Zero{}, 0);
    load(One{}, 1);
    store(Zero{}, 0);
    load(Zero{}, 2);
    __syncthreads();
#pragma unroll 1
    for (int kt = 0; kt < whole; kt += 2) {
      multiply(kt);
      store(One{}, kt + 1);
      load(One{}, kt + 3);
      __syncthreads();
      multiply(kt + 1);
      store(Zero{}, kt + 2);
      load(Zero{}, kt + 4);
      __syncthreads();
    }
  }
  for (int kt = whole; kt < KT; ++kt) {
    float wa[V], wb[V];
    f32_load<KRA, V>(wa, A, g.lda, M, kt * F_K, K - kt * F_K);
    f32_load<KRB, V>(wb, B, g.ldb, N, kt * F_K, K - kt * F_K);
    f32_store<KRA, V>(lds[kt & 1][0], wa);
    f32_store<KRB, V>(lds[kt & 1][1], wb);
    __syncthreads();
    multiply(kt);
  }
#pragma unroll
  for (int i = 0; i < S; ++i)
#pragma unroll
    for (int j = 0; j < S; ++j)
#pragma unroll
      for (int q = 0; q < 16; ++q) sum[i][j][q] += acc[i][j][q];
  // a lane holds row fr, columns 8 (q / 4) + 4 fk + q % 4 of each 32 x 32 block
  float* C = (float*)g.c + (FORM == WGT ? ((int64_t)e * g.M + tm * F_B) * g.N : (int64_t)row0 * g.N);
#pragma unroll
  for (int i = 0; i < S; ++i) {
    const int m = wm * 32 * S + i * 32 + fr;
    if (m >= M) continue;
    float* out = C + (int64_t)m * g.N + tn * F_B;
#pragma unroll
    for (int j = 0; j < S; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int n = wn * 32 * S + j * 32 + q * 8 + fk * 4;
        if (n + 4 <= N) {
          const float v[4] = {sum[i][j][4 * q], sum[i][j][4 * q + 1], sum[i][j][4 * q + 2], sum[i][j][4 * q + 3]};
          __builtin_memcpy(out + n, v, 16);
        } else {
#pragma unroll
          for (int p = 0; p < 4; ++p)
            if (n + p < N) out[n + p] = sum[i][j][4 * q + p];
        }
      }
  }
}

// ---- launch ---------------------------------------------------------------------------------

// The most tiles of bm rows that R rows of E experts, and what lies behind them, can make.
int64_t most_tiles(int64_t R, int64_t E, int bm) { return R / bm + std::min(R, E + 1); }

// So many workgroups, launch(g, n) of n of them at a time: an extent of a grid has to stay below 2^32 threads.
template <typename Launch>
int launch_all(GArgs g, int64_t workgroups, Launch launch) {
  if (workgroups > INT32_MAX) {  // of no tensors that fit the card
    muon_set_error("muon_expert_linear: too many tiles");
    return MUON_ERR_SHAPE;
  }
  constexpr int64_t MOST = 1 << 22;
  for (int64_t at = 0; at < workgroups; at += MOST) {
    g.first = (int)at;
    launch(g, (unsigned)std::min(workgroups - at, MOST));
    MUON_CHECK_LAUNCH("muon_expert_linear");
  }
  return MUON_OK;
}

template <int DT, int FORM, int BM, int BN, int WM, int WN>
int launch16(GArgs g, bool aligned, hipStream_t s) {
  g.tiles_m = (int)(FORM == WGT ? (g.M + BM - 1) / BM : most_tiles(g.R, g.E, BM));
  g.tiles_n = (g.N + BN - 1) / BN;
  const int64_t grid = (int64_t)g.tiles_m * g.tiles_n * (FORM == WGT ? g.E : 1);
  constexpr int LDS = 2 * (BM + BN) * BK * 2;
  auto run = [&](auto* kernel) {
    if (hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, LDS) != hipSuccess) {
      muon_set_error("muon_expert_linear: %d bytes of LDS refused", LDS);
      return MUON_ERR_LAUNCH;
    }
    return launch_all(g, grid, [&](const GArgs& a, unsigned n) { kernel<<<n, 64 * WM * WN, LDS, s>>>(a); });
  };
  return aligned ? run(expert_gemm_kernel<DT, FORM, BM, BN, WM, WN, true>)
                 : run(expert_gemm_kernel<DT, FORM, BM, BN, WM, WN, false>);
}

template <int DT>
int launch_rows(GArgs g, bool aligned, hipStream_t s) {
  g.tiles_n = (g.N + R_N - 1) / R_N;
  const int64_t grid = most_tiles(g.R, g.E, 16) * g.tiles_n;
  return launch_all(g, grid, [&](const GArgs& a, unsigned n) {
    if (aligned) expert_rows_kernel<DT, true><<<n, 256, 0, s>>>(a);
    else expert_rows_kernel<DT, false><<<n, 256, 0, s>>>(a);
  });
}

// What the direct loads and stores index by 32 bits: 256 rows of a panel, 64 of one along k, 128 of a result.
constexpr int64_t P_MOST = 1 << 20;

template <int DT, int FORM>
int launch_pipe(GArgs g, hipStream_t s) {
  g.tiles_m = (int)(FORM == WGT ? (g.M + 255) / 256 : 0);  // of rows: counted on the device
  g.tiles_n = (g.N + 255) / 256;
  const int64_t most = (FORM == WGT ? (int64_t)g.tiles_m * g.E : most_tiles(g.R, g.E, 256)) * g.tiles_n;
  if (most > INT32_MAX) {
    muon_set_error("muon_expert_linear: too many tiles");
    return MUON_ERR_SHAPE;
  }
  const int lds = 2 * P_STAGE + 4 * P_OUT + 3 * (g.E + 2) * 4;
  if (hipFuncSetAttribute((const void*)expert_gemm_pipe_kernel<DT, FORM>,
                          hipFuncAttributeMaxDynamicSharedMemorySize, lds) != hipSuccess) {
    muon_set_error("muon_expert_linear: %d bytes of LDS refused", lds);
    return MUON_ERR_LAUNCH;
  }
  expert_gemm_pipe_kernel<DT, FORM><<<P_GROUPS, 256, lds, s>>>(g);
  MUON_CHECK_LAUNCH("muon_expert_linear");
  return MUON_OK;
}

template <int FORM, int S>
int launch32(GArgs g, hipStream_t s) {
  g.tiles_m = (int)(FORM == WGT ? (g.M + 64 * S - 1) / (64 * S) : most_tiles(g.R, g.E, 64 * S));
  g.tiles_n = (g.N + 64 * S - 1) / (64 * S);
  const int64_t grid = (int64_t)g.tiles_m * g.tiles_n * (FORM == WGT ? g.E : 1);
  return launch_all(g, grid, [&](const GArgs& a, unsigned n) { expert_gemm_f32_kernel<FORM, S><<<n, 256, 0, s>>>(a); });
}

// Which kernel, all sides measured on 8 to 128 experts of 1024 x 1024 to 4096 x 4096 (us):
// * FWD of at most 4 rows an expert on the average: the kernel of few rows (64 experts of 1408 x 2048, 128 and
//   256 rows: 60 and 67, 72 and 73 in tiles of 128; 512 rows 85 and 78). Short rows of many experts
//   are an exception (128 of 2048 x 768, 512 rows: 90 and 73), few tiles another, up to 16 rows (8 of
//   1024 x 1024, 128 rows: 9 and 11; ragged ones, 8 of 1001 x 769, 64 rows: 17 and 15).
// * FWD and ROWS in tiles of 256 from 112 of them on (8 experts of 1024 x 1024, 8000 rows: 27 and 27, in
//   tiles of 128 33 and 35; 6000 rows: 27 and 26, 23 and 25), if there are 192 rows an expert: with fewer the weights'
//   bytes count, which more workgroups fetch faster (64 of 1408 x 2048, 8192 rows: 123 and 117, 114 and
//   114; 16384 rows: 160 and 151, 176 and 182).
// * WGT where there is one for every CU (4 experts of 2048 x 2048, 4000 rows 73 and 91), or where fewer
//   of them are very long (2 of 2048 x 2048, 8000 rows: 122 and 98, 32000 rows: 279 and 349) and there are
//   more tiles of 128 than CUs: one tile a CU is multiplied faster the smaller it is (2 of 64 x 64, 65536 rows: 540
//   and 382; 1 of 512 x 512, 8192: 141 and 96; 8 of 512 x 512, 131072: 276 and 215; 1 of 2048 x 2048, 65536:
//   1086 and 960; with 352 of them 2 of 1408 x 2048, 65536: 555 and 636).
// * Else, and where rows are no whole 16-byte runs, tiles of 128.
template <int DT, int FORM>
int launch_typed(const GArgs& g, hipStream_t s) {
  const bool aligned = ((uintptr_t)g.a | (uintptr_t)g.b | (uintptr_t)g.c) % 16 == 0 &&
                       (g.lda | g.ldb | g.sb | g.N | g.K | g.M) % 8 == 0;
  const int64_t columns = (int64_t)g.E * g.N, few = aligned && columns <= 16384 ? 16 : g.K >= 1024 || columns <= 65536 ? 4 : 0;
  if (FORM == FWD && g.R <= few * g.E) return launch_rows<DT>(g, aligned, s);
  const int64_t wa = FORM == WGT ? g.M : g.K, wb = FORM == FWD ? g.K : g.N;
  const bool direct = aligned && g.lda >= wa && g.ldb >= wb && std::max({g.lda, g.ldb, (int64_t)g.N}) <= P_MOST;
  const int64_t area = FORM == WGT ? (int64_t)g.M * g.N * g.E : g.R * g.N, tile = 256 * 256;
  const int64_t small = (int64_t)((g.M + 127) / 128) * ((g.N + 127) / 128) * g.E;
  const bool large = FORM == WGT ? area >= P_GROUPS * tile || (small > P_GROUPS && g.R >= 8192 * (int64_t)g.E)
                                 : area >= 112 * tile && g.R >= 192 * (int64_t)g.E;
  return direct && large ? launch_pipe<DT, FORM>(g, s) : launch16<DT, FORM, 128, 128, 4, 2>(g, aligned, s);
}

template <int FORM>
int launch(const GArgs& g, int dtype, hipStream_t s) {
  switch (dtype) {
    case MUON_DT_F32: {
      // Tiles of 128 where there are ten for every CU (16 experts of 1024 x 1024: 64000 rows 1121 us, in
      // tiles of 64 1142, their gradient 1026 and 1111; 16000 rows 346 and 312); for WGT, whose experts are
      // tiled alone, by the weights (8 of 2048 x 2048, 4000 rows: 270 and 306; 8 of 1001 x 769, 32000 rows: 641 and 517).
      const int64_t tiles = (FORM == WGT ? (int64_t)g.M * g.N * g.E : g.R * g.N) / (128 * 128);
      return tiles >= (FORM == WGT ? 2048 : 2560) ? launch32<FORM, 2>(g, s) : launch32<FORM, 1>(g, s);
    }
    case MUON_DT_BF16: return launch_typed<MUON_DT_BF16, FORM>(g, s);
    default: return launch_typed<MUON_DT_F16, FORM>(g, s);
  }
}

int check_shapes(const char* what, int dtype, int64_t rows, int64_t experts, int64_t out, int64_t in) {
  if (dtype != MUON_DT_F32 && dtype != MUON_DT_BF16 && dtype != MUON_DT_F16) {
    muon_set_error("%s: unsupported dtype %d", what, dtype);
    return MUON_ERR_DTYPE;
  }
  if (rows < 0 || rows > INT32_MAX || experts < 1 || experts > 1024 || out < 0 || in < 0 ||
      out > (1 << 24) || in > (1 << 24)) {
    muon_set_error("%s: %lld rows of %lld experts, %lld x %lld: below 2^31 rows, 1 to 1024 experts and "
                   "extents to 2^24", what, (long long)rows, (long long)experts, (long long)out, (long long)in);
    return MUON_ERR_SHAPE;
  }
  return MUON_OK;
}

}  // namespace

extern "C" int muon_expert_linear(const void* rows, int dtype, int64_t row_stride, int64_t nrows,
                                  int64_t experts, int64_t out, int64_t in, const void* weight,
                                  const int32_t* offsets, void* y, void* stream) {
  if (int rc = check_shapes("muon_expert_linear", dtype, nrows, experts, out, in)) return rc;
  if (!nrows || !out) return MUON_OK;
  if (!offsets || !y || (in && (!rows || !weight))) {
    muon_set_error("muon_expert_linear: null pointer");
    return MUON_ERR_ARG;
  }
  GArgs g{rows, weight, y, row_stride, in, out * in, offsets, nrows, (int)experts, (int)out, (int)in, 0, 0, 0, 0};
  return launch<FWD>(g, dtype, (hipStream_t)stream);
}

extern "C" int muon_expert_linear_backward_rows(const void* dy, int dtype, int64_t dy_stride,
                                                int64_t nrows, int64_t experts, int64_t out, int64_t in,
                                                const void* weight, const int32_t* offsets,
                                                void* drows, void* stream) {
  if (int rc = check_shapes("muon_expert_linear_backward_rows", dtype, nrows, experts, out, in)) return rc;
  if (!nrows || !in) return MUON_OK;
  if (!offsets || !drows || (out && (!dy || !weight))) {
    muon_set_error("muon_expert_linear_backward_rows: null pointer");
    return MUON_ERR_ARG;
  }
  GArgs g{dy, weight, drows, dy_stride, in, out * in, offsets, nrows, (int)experts, (int)in, (int)out, 0, 0, 0, 0};
  return launch<ROWS>(g, dtype, (hipStream_t)stream);
}

extern "C" int muon_expert_linear_backward_weight(const void* dy, int dtype, int64_t dy_stride,
                                                  const void* rows, int64_t row_stride, int64_t nrows,
                                                  int64_t experts, int64_t out, int64_t in,
                                                  const int32_t* offsets, void* dweight, void* stream) {
  if (int rc = check_shapes("muon_expert_linear_backward_weight", dtype, nrows, experts, out, in)) return rc;
  if (!out || !in) return MUON_OK;
  if (!offsets || !dweight || (nrows && (!dy || !rows))) {
    muon_set_error("muon_expert_linear_backward_weight: null pointer");
    return MUON_ERR_ARG;
  }
  GArgs g{dy, rows, dweight, dy_stride, row_stride, 0, offsets, nrows, (int)experts, (int)in, 0, (int)out, 0, 0, 0};
  return launch<WGT>(g, dtype, (hipStream_t)stream);
}
