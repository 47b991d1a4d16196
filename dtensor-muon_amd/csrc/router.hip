// Expert routing: the top-k choice of a token's experts with their gates, the tokens each expert
// gets, the balance loss and the z loss, with the gradient to the logits (muon_route,
// muon_route_backward).
//
// For a token's logits z over E experts: p = softmax(z), lse = log sum exp z; the k largest are
// chosen (ties: the lowest index; a NaN counts as the largest; an expert at -inf is never chosen,
// and a slot that finds none holds -1 and gate 0). Gates are p, or p over the chosen ones' sum.
// Over the N tokens that count (not masked, and not all -inf), with c_e tokens at expert e:
//   balance = E sum_e (c_e / (k N)) (1 / N) sum_t p_te,   z = (1 / N) sum_t lse_t^2.
// Backward, with a_e = db E c_e / (k N^2), G the gates' gradient:
//   dz_e = p_e (a_e - sum p a) + 2 lse dzl / N p_e + [e chosen] g_e (G_e - sum g G)  (normalized)
//   or, with the gates as they are, the last term p_e ([e chosen] G_e - sum over chosen p G).
//
// The counts of all tokens stand between the two passes, so both read the logits and make p.
// The forward pass is bound by vector instructions: a wave's four tokens of 256 bf16 experts with 8
// choices take about 570, and the vector units issue for 93% of the time that its CUs are busy. 131071
// such tokens: 41 us and 6.5 for the totals, where the bytes take 16. The backward pass (37 us, bytes
// 29) has them busy for 61%. 32768 tokens of 64 experts in fp32: 9.7, 6.6 and 8.8 us. (Launches in a
// trace; in passes that follow each other both directions take 43 and 34 us, 14 and 7.)
#include <algorithm>
#include <type_traits>

#include "rowops.h"

namespace {

constexpr int KMAX = 64;
constexpr int EMAX = 1024;
constexpr int FWD_THREADS = 512;
constexpr int BWD_THREADS = 256;
constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;

struct Args {
  const void* z;
  int64_t row;  // stride of a token's logits in elements
  int64_t T;
  int E, k, normalize;
  const uint8_t* mask;  // or null: every token counts
  float* gates;
  int64_t* experts;
  int64_t* counts;
  float* balance;  // one value each: the losses, and the number of tokens that count
  float* zloss;
  float* kept;
  // one partial a workgroup, of E or of one value; of the finishing workgroups (part_b, ticket)
  double* part_b;
  int* ticket;
  float* part_p;
  int* part_c;
  float* part_z;
  int* part_n;
};

struct BackArgs {
  const void* z;
  int64_t row, T;
  int E, k, normalize;
  const uint8_t* mask;
  const int64_t* experts;
  const int64_t* counts;
  const float* kept;
  const float* dgates;    // or null
  const float* dbalance;  // one value each, or null
  const float* dzloss;
  void* dz;  // contiguous
};

// The logits of one token that a lane owns: VPT experts in a row; -inf behind the last one.
template <int DT, int VPT>
MUON_DEVICE void load_logits(const void* z, int64_t at, int e0, int E,
                             muon_u4 (&w)[VPT / Vec16<DT>::N]) {
  constexpr int N = Vec16<DT>::N;
#pragma unroll
  for (int c = 0; c < VPT / N; ++c) {
    const int e = e0 + c * N;
    if (e + N <= E) {
      w[c] = load_u4(elem_at<DT>(z, at + e));
    } else {
      float x[N];
#pragma unroll
      for (int j = 0; j < N; ++j) x[j] = e + j < E ? Elem<DT>::load(z, at + e + j) : -INFINITY;
      w[c] = Vec16<DT>::pack(x);
    }
  }
}
template <int DT, int VPT>
MUON_DEVICE void unpack_logits(const muon_u4 (&w)[VPT / Vec16<DT>::N], float (&v)[VPT]) {
  constexpr int N = Vec16<DT>::N;
#pragma unroll
  for (int c = 0; c < VPT / N; ++c) {
    float x[N];
    Vec16<DT>::unpack(w[c], x);
#pragma unroll
    for (int j = 0; j < N; ++j) v[c * N + j] = x[j];
  }
}

// An order-preserving integer of a value that is no NaN, -0 as 0; +inf gives 0xff800000, the
// lowest finite value 0x00800000, -inf less. The NaN 0x7fc00000 comes above them all.
MUON_DEVICE uint32_t ordered(float v) {
  const uint32_t u = __float_as_uint(v + 0.0f);
  return u ^ ((uint32_t)((int)u >> 31) | 0x80000000u);
}
MUON_DEVICE float unordered(uint32_t o) {
  return __uint_as_float(o ^ ((o >> 31) ? 0x80000000u : 0xffffffffu));
}
constexpr uint32_t ORDERED_LOWEST = 0x00800000u;

// A value and its index as one number, larger for a larger value and, among equal ones, for a
// lower index; -inf, also behind the last expert, gives a number below all that can be chosen.
// All keys of a token are distinct, so the next choice is the largest key below the last one:
// nothing has to be taken out of the registers.
// Values of two bytes have at most 19 significant bits in fp32: 32 bits hold both. fp32 takes
// 63 bits, compared as a positive double (no key reaches the exponent of infinities, since the
// largest ordered value, the NaN's, is 0xffc00000).
template <int DT>
struct Key {
  typedef uint32_t T;
  static MUON_DEVICE T make(float v, int e) {
    return (ordered(v) & 0xffffe000u) | (uint32_t)(0x1fff - e);
  }
  static MUON_DEVICE bool none(T k) { return k < ORDERED_LOWEST; }
  static MUON_DEVICE int index(T k) { return 0x1fff - (int)(k & 0x1fffu); }
  static MUON_DEVICE float value(T k) {
    // a negative value's ordered form has ones in the masked bits
    const uint32_t o = k & 0xffffe000u;
    return unordered((o >> 31) ? o : o | 0x1fffu);
  }
  static MUON_DEVICE T larger(T a, T b) { return max(a, b); }
  template <int G>
  static MUON_DEVICE T largest(T v) {
    return group_reduce<G>(v, [](T a, T b) { return max(a, b); });
  }
  // The largest key below `last`: key - last wraps to the top of the range exactly for the keys
  // below it, in their order, so one subtraction and one maximum serve a key. Past the last key
  // the result is 0.
  template <int VPT, int G>
  static MUON_DEVICE T next(const T (&key)[VPT], T last) {
    T best = 0;
#pragma unroll
    for (int j = 0; j < VPT; ++j) best = max(best, key[j] - last);
    best = largest<G>(best);
    const T found = best + last;
    return found < last ? found : 0;
  }
};
template <>
struct Key<MUON_DT_F32> {
  typedef double T;
  static MUON_DEVICE T make(float v, int e) {
    const uint32_t o = ordered(v);
    return __hiloint2double((int)(o >> 1), (int)((o << 31) | (uint32_t)(0x7fffffff - e)));
  }
  static MUON_DEVICE bool none(T k) { return (uint32_t)__double2hiint(k) < ORDERED_LOWEST >> 1; }
  static MUON_DEVICE int index(T k) { return 0x7fffffff - (__double2loint(k) & 0x7fffffff); }
  static MUON_DEVICE float value(T k) {
    return unordered(((uint32_t)__double2hiint(k) << 1) | ((uint32_t)__double2loint(k) >> 31));
  }
  // No operand is a NaN: fmax's extra step that quiets them is left out. The compiler sees no
  // vector instruction in it and so no need for the wait states before a DPP read of the result:
  // largest() passes it through an instruction of the compiler's own first.
  static MUON_DEVICE T larger(T a, T b) {
    T r;
    asm("v_max_f64 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
    return r;
  }
  template <int G>
  static MUON_DEVICE T largest(T v) {
    return group_reduce<G>(__builtin_fmax(v, 0.0), [](T a, T b) { return __builtin_fmax(a, b); });
  }
  // A key at or above `last` loses its upper half, which leaves it below every key that counts.
  template <int VPT, int G>
  static MUON_DEVICE T next(const T (&key)[VPT], T last) {
    T best = 0.0;
#pragma unroll
    for (int j = 0; j < VPT; ++j)
      best = larger(best, __hiloint2double(key[j] < last ? __double2hiint(key[j]) : 0,
                                           __double2loint(key[j])));
    return largest<G>(best);
  }
};

// What one wave writes to LDS and reads back itself needs no barrier of the workgroup: LDS
// operations of a wave are done in order, and this keeps the compiler from reordering them.
MUON_DEVICE void wave_lds_fence() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// The losses from sum_e c_e sum_t p_te, sum lse^2 and the number of tokens that count.
MUON_DEVICE void write_losses(const Args& a, double balance, double z, int64_t n) {
  const double d = (double)n;
  a.balance[0] = n ? (float)(balance * (double)a.E / ((double)a.k * d * d)) : 0.0f;
  a.zloss[0] = n ? (float)(z / d) : 0.0f;
  a.kept[0] = (float)n;
}

// Groups of G lanes take a token each, VPT experts a lane, and walk over the tokens; each lane
// sums its experts' p in registers over all its tokens, the chosen ones are counted in LDS
// (integers: any order gives the same), and the workgroup writes one partial of E sums and
// counts. A single workgroup writes the results itself.
template <int DT, int G, int VPT>
__global__ __launch_bounds__(FWD_THREADS) void route_kernel(Args a) {
  constexpr int GROUPS = FWD_THREADS / G;
  constexpr int ECAP = G * VPT;
  constexpr int KCAP = ECAP < KMAX ? ECAP : KMAX;
  typedef Key<DT> K;
  constexpr int RAW = VPT / Vec16<DT>::N;
  __shared__ typename K::T picks[GROUPS][KCAP];
  __shared__ float cols[GROUPS][ECAP + 1];
  __shared__ int cnt[ECAP];
  __shared__ float zs[GROUPS];
  __shared__ int ns[GROUPS];
  const int lane = threadIdx.x % G, group = threadIdx.x / G;
  const int e0 = lane * VPT;
  for (int e = threadIdx.x; e < ECAP; e += FWD_THREADS) cnt[e] = 0;
  __syncthreads();
  float acc[VPT];
#pragma unroll
  for (int j = 0; j < VPT; ++j) acc[j] = 0.0f;
  float zsum = 0.0f;
  int n = 0;
  const int64_t step = (int64_t)gridDim.x * GROUPS;
  int64_t t = (int64_t)blockIdx.x * GROUPS + group;
  muon_u4 raw[RAW];
  if (t < a.T) load_logits<DT, VPT>(a.z, t * a.row, e0, a.E, raw);
  for (; t < a.T; t += step) {
    float v[VPT], p[VPT];
    unpack_logits<DT, VPT>(raw, v);
    if (t + step < a.T) load_logits<DT, VPT>(a.z, (t + step) * a.row, e0, a.E, raw);
    float m = v[0];
#pragma unroll
    for (int j = 1; j < VPT; ++j) m = fmaxf(m, v[j]);
    m = group_max<G>(m);
    bool on = !a.mask || a.mask[t];
    if (m == -INFINITY) {  // all -inf counts nowhere (a NaN, which fmaxf passes over, makes no such row)
      float bad = 0.0f;
#pragma unroll
      for (int j = 0; j < VPT; ++j) bad = v[j] != v[j] ? 1.0f : bad;
      on = on && group_max<G>(bad) != 0.0f;
    }
    float total = 0.0f;
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      p[j] = __builtin_amdgcn_exp2f((v[j] - m) * LOG2E);  // 0 behind the last expert
      total += p[j];
    }
    total = group_sum<G>(total);
    const float inv = __builtin_amdgcn_rcpf(total);
    float held = 0.0f;
    if (on) {
#pragma unroll
      for (int j = 0; j < VPT; ++j) acc[j] += p[j] * inv;
      const float lse = m + __builtin_amdgcn_logf(total) * LN2;
      zsum += lse * lse;
      n += 1;
      if (total != total) {  // a NaN somewhere, of whatever sign and payload: as one
#pragma unroll
        for (int j = 0; j < VPT; ++j) v[j] = v[j] != v[j] ? __uint_as_float(0x7fc00000u) : v[j];
      }
      typename K::T key[VPT], best = 0;
#pragma unroll
      for (int j = 0; j < VPT; ++j) {
        key[j] = K::make(v[j], e0 + j);
        best = K::larger(best, key[j]);
      }
      best = K::template largest<G>(best);
      for (int i = 0;;) {
        if (lane == 0) picks[group][i] = best;
        if (++i == a.k) break;
        best = K::template next<VPT, G>(key, best);
      }
      wave_lds_fence();
      for (int i = lane; i < a.k; i += G) {
        const typename K::T q = picks[group][i];
        held += K::none(q) ? 0.0f : __builtin_amdgcn_exp2f((K::value(q) - m) * LOG2E);
      }
      held = group_sum<G>(held);
    }
    const float share = a.normalize ? __builtin_amdgcn_rcpf(held) : inv;
    for (int i = lane; i < a.k; i += G) {
      int64_t e = -1;
      float gate = 0.0f;
      if (on) {
        const typename K::T q = picks[group][i];
        if (!K::none(q)) {
          e = K::index(q);
          gate = __builtin_amdgcn_exp2f((K::value(q) - m) * LOG2E) * share;
          atomicAdd(&cnt[e], 1);
        }
      }
      a.experts[t * a.k + i] = e;
      a.gates[t * a.k + i] = gate;
    }
    wave_lds_fence();
  }
#pragma unroll
  for (int j = 0; j < VPT; ++j) cols[group][e0 + j] = acc[j];
  if (lane == 0) {
    zs[group] = zsum;
    ns[group] = n;
  }
  __syncthreads();
  for (int e = threadIdx.x; e < a.E; e += FWD_THREADS) {
    float sum = 0.0f;
    for (int g = 0; g < GROUPS; ++g) sum += cols[g][e];
    if (gridDim.x == 1) {
      a.counts[e] = cnt[e];
      cols[0][e] = sum;
    } else {
      a.part_p[(int64_t)blockIdx.x * a.E + e] = sum;
      a.part_c[(int64_t)blockIdx.x * a.E + e] = cnt[e];
    }
  }
  __syncthreads();
  if (threadIdx.x >= 64) return;
  double z = 0.0, b = 0.0;
  int c = 0;
  for (int g = threadIdx.x; g < GROUPS; g += 64) {
    z += zs[g];
    c += ns[g];
  }
  if (gridDim.x == 1)
    for (int e = threadIdx.x; e < a.E; e += 64) b += (double)cnt[e] * (double)cols[0][e];
  for (int off = 32; off; off >>= 1) {
    z += __shfl_xor(z, off, 64);
    b += __shfl_xor(b, off, 64);
    c += __shfl_xor(c, off, 64);
  }
  if (threadIdx.x) return;
  if (gridDim.x == 1) {
    write_losses(a, b, z, c);
  } else {
    if (blockIdx.x == 0) *a.ticket = 0;  // for the launch after this one
    a.part_z[blockIdx.x] = (float)z;
    a.part_n[blockIdx.x] = c;
  }
}

// The workgroups' partials summed in a fixed order: 16 experts a workgroup, 64 rows of threads over
// the partials, joined through LDS. The workgroup that ends last (a ticket counts them, zeroed by
// route_kernel) adds their shares of the balance loss, again in order.
__global__ __launch_bounds__(1024) void route_finish_kernel(Args a, int blocks) {
  __shared__ float ps[64][17];
  __shared__ int cs[64][17];
  __shared__ double red[2][16];
  const int col = threadIdx.x % 16, row = threadIdx.x / 16;
  const int e = blockIdx.x * 16 + col;
  float p = 0.0f;
  int c = 0;
  if (e < a.E) {
#pragma unroll 8
    for (int b = row; b < blocks; b += 64) {
      p += a.part_p[(int64_t)b * a.E + e];
      c += a.part_c[(int64_t)b * a.E + e];
    }
  }
  ps[row][col] = p;
  cs[row][col] = c;
  double z = 0.0, n = 0.0;  // token counts below 2^53 are exact
  for (int b = threadIdx.x; b < blocks; b += 1024) {
    z += a.part_z[b];
    n += a.part_n[b];
  }
  for (int off = 32; off; off >>= 1) {
    z += __shfl_xor(z, off, 64);
    n += __shfl_xor(n, off, 64);
  }
  if (threadIdx.x % 64 == 0) {
    red[0][threadIdx.x / 64] = z;
    red[1][threadIdx.x / 64] = n;
  }
  __syncthreads();
  if (threadIdx.x >= 64) return;
  {  // a wave: 4 threads a column
    double sum = 0.0;
    int64_t count = 0;
    for (int r = row; r < 64; r += 4) {
      sum += ps[r][col];
      count += cs[r][col];
    }
    for (int off = 16; off < 64; off *= 2) {
      sum += __shfl_xor(sum, off, 64);
      count += __shfl_xor((long long)count, off, 64);
    }
    if (row == 0 && e < a.E) a.counts[e] = count;
    double bal = e < a.E ? sum * (double)count : 0.0;
    for (int off = 1; off < 16; off *= 2) bal += __shfl_xor(bal, off, 64);
    int ticket = 0;
    if (threadIdx.x == 0) {
      __hip_atomic_store(&a.part_b[blockIdx.x], bal, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      ticket = __hip_atomic_fetch_add(a.ticket, 1, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT);
    }
    if (__shfl(ticket, 0, 64) != (int)gridDim.x - 1) return;
  }
  // the wave of the last workgroup: at most 64 shares of the balance loss, 16 of the others
  static_assert(EMAX / 16 <= 64, "a lane a workgroup");
  const int lane = threadIdx.x;
  double bal = 0.0;
  if (lane < (int)gridDim.x)
    bal = __hip_atomic_load(&a.part_b[lane], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  z = lane < 16 ? red[0][lane] : 0.0;
  n = lane < 16 ? red[1][lane] : 0.0;
  for (int off = 32; off; off >>= 1) {
    bal += __shfl_xor(bal, off, 64);
    z += __shfl_xor(z, off, 64);
    n += __shfl_xor(n, off, 64);
  }
  if (lane == 0) write_losses(a, bal, z, (int64_t)n);
}

// One group a token again: p from the logits, the dense part of the gradient in registers, and
// the chosen experts' part through the group's row in LDS (where it is added at their indices).
// A row holds a lane's VPT values as 16-byte pieces G lanes apart: neighbouring lanes' pieces
// are neighbours, and no two lanes of an access meet in a bank (value after value, 16 of them a
// lane, four lanes met in each: 47 us instead of 41 on 131071 tokens of 256 experts).
template <int G, int VPT>
MUON_DEVICE int row_at(int e) {
  return (((e % VPT) / 4) * G + e / VPT) * 4 + e % 4;
}
template <int G, int VPT>
MUON_DEVICE void put_row(float* row, int lane, const float (&v)[VPT]) {
#pragma unroll
  for (int c = 0; c < VPT / 4; ++c)
    *(f32x4*)(row + (c * G + lane) * 4) = f32x4{v[4 * c], v[4 * c + 1], v[4 * c + 2], v[4 * c + 3]};
}
template <int G, int VPT>
MUON_DEVICE void get_row(const float* row, int lane, float (&v)[VPT]) {
#pragma unroll
  for (int c = 0; c < VPT / 4; ++c) {
    const f32x4 w = *(const f32x4*)(row + (c * G + lane) * 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[4 * c + i] = w[i];
  }
}

// Slot lane + q G of a token is this lane's: the chosen expert and its gate's gradient. An empty slot's
// gate is the constant 0: what comes back for it, infinities too, is none of the token's.
template <int G, int SLOTS>
MUON_DEVICE void load_slots(const BackArgs& a, int64_t t, int lane, int (&at)[SLOTS], float (&up)[SLOTS]) {
#pragma unroll
  for (int q = 0; q < SLOTS; ++q) {
    at[q] = -1;
    up[q] = 0.0f;
    if (q * G >= a.k) continue;  // the same for all
    const int i = lane + q * G;
    if (!a.dgates || i >= a.k) continue;
    const int64_t e = a.experts[t * a.k + i];
    const float g = a.dgates[t * a.k + i];
    const bool held = e >= 0 && e < a.E;
    up[q] = held ? g : 0.0f;
    at[q] = held ? (int)e : -1;
  }
}

template <int DT, int G, int VPT>
__global__ __launch_bounds__(BWD_THREADS) void route_backward_kernel(BackArgs a) {
  constexpr int GROUPS = BWD_THREADS / G;
  constexpr int ECAP = G * VPT;
  constexpr int SLOTS = (ECAP < KMAX ? ECAP : KMAX) / G;
  __shared__ __attribute__((aligned(16))) float rows[GROUPS][ECAP];
  const int lane = threadIdx.x % G, group = threadIdx.x / G;
  const int e0 = lane * VPT;
  const float n = a.kept[0];
  const float db = a.dbalance && n > 0.0f ? a.dbalance[0] : 0.0f;
  const float zc = a.dzloss && n > 0.0f ? 2.0f * a.dzloss[0] / n : 0.0f;
  // a count is at most the tokens, which fit 31 bits; 1 / n twice, since n^2 may leave the range
  const float inv_n = n > 0.0f ? 1.0f / n : 0.0f;
  const float bc = db * (float)a.E / (float)a.k * inv_n;
  float coef[VPT];
#pragma unroll
  for (int j = 0; j < VPT; ++j)
    coef[j] = e0 + j < a.E ? bc * ((float)((const uint32_t*)a.counts)[2 * (e0 + j)] * inv_n) : 0.0f;
  float* mine = rows[group];
  const int64_t step = (int64_t)gridDim.x * GROUPS;
  int64_t t = (int64_t)blockIdx.x * GROUPS + group;
  muon_u4 raw[VPT / Vec16<DT>::N];
  int next_at[SLOTS];
  float next_up[SLOTS];
  if (t < a.T) {
    load_logits<DT, VPT>(a.z, t * a.row, e0, a.E, raw);
    load_slots<G, SLOTS>(a, t, lane, next_at, next_up);
  }
  for (; t < a.T; t += step) {
    float v[VPT], part[SLOTS], up[SLOTS];
    int at[SLOTS];
    unpack_logits<DT, VPT>(raw, v);
#pragma unroll
    for (int q = 0; q < SLOTS; ++q) {
      at[q] = next_at[q];
      up[q] = next_up[q];
    }
    if (t + step < a.T) {  // the next token's loads are in flight meanwhile
      load_logits<DT, VPT>(a.z, (t + step) * a.row, e0, a.E, raw);
      load_slots<G, SLOTS>(a, t + step, lane, next_at, next_up);
    }
    float m = v[0];
#pragma unroll
    for (int j = 1; j < VPT; ++j) m = fmaxf(m, v[j]);
    m = group_max<G>(m);
    bool on = !(a.mask && !a.mask[t]);
    if (m == -INFINITY) {
      float bad = 0.0f;
#pragma unroll
      for (int j = 0; j < VPT; ++j) bad = v[j] != v[j] ? 1.0f : bad;
      on = on && group_max<G>(bad) != 0.0f;
    }
    float total = 0.0f, dot = 0.0f;
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      v[j] = __builtin_amdgcn_exp2f((v[j] - m) * LOG2E);  // 0 behind the last expert
      total += v[j];
    }
    total = group_sum<G>(total);
    const float inv = __builtin_amdgcn_rcpf(total);
    const float lse = m + __builtin_amdgcn_logf(total) * LN2;
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      v[j] *= inv;
      dot += v[j] * coef[j];
    }
    dot = group_sum<G>(dot);
    put_row<G, VPT>(mine, lane, v);
    wave_lds_fence();
    float held = 0.0f, inner = 0.0f;  // sums of p and of p G over the chosen
#pragma unroll
    for (int q = 0; q < SLOTS; ++q) {
      part[q] = 0.0f;
      if (q * G >= a.k) continue;
      part[q] = on && at[q] >= 0 ? mine[row_at<G, VPT>(at[q])] : 0.0f;
      held += part[q];
      inner += part[q] * up[q];
    }
    held = group_sum<G>(held);
    inner = group_sum<G>(inner);
    wave_lds_fence();
    const float shift = zc * lse - dot - (a.normalize ? 0.0f : inner);
#pragma unroll
    for (int j = 0; j < VPT; ++j) v[j] *= coef[j] + shift;
    put_row<G, VPT>(mine, lane, v);
    wave_lds_fence();
    const float scale = a.normalize ? __builtin_amdgcn_rcpf(held) : 1.0f;
    const float mean = a.normalize ? inner * scale : 0.0f;
#pragma unroll
    for (int q = 0; q < SLOTS; ++q)  // a token's experts are distinct: no two lanes meet
      if (q * G < a.k && on && at[q] >= 0) mine[row_at<G, VPT>(at[q])] += part[q] * scale * (up[q] - mean);
    wave_lds_fence();
    get_row<G, VPT>(mine, lane, v);
    wave_lds_fence();
    constexpr int N = Vec16<DT>::N;
#pragma unroll
    for (int c = 0; c < VPT; c += N) {
      float x[N];
#pragma unroll
      for (int j = 0; j < N; ++j) x[j] = on ? v[c + j] : 0.0f;
      const int e = e0 + c;
      if (e + N <= a.E) {
        store_u4((void*)elem_at<DT>(a.dz, t * a.E + e), Vec16<DT>::pack(x));
      } else {
#pragma unroll
        for (int j = 0; j < N; ++j)
          if (e + j < a.E) Elem<DT>::store(a.dz, t * a.E + e + j, x[j]);
      }
    }
  }
}

// Lanes and experts per lane for E experts: 8 experts a lane up to 16 lanes, then 16. More
// lanes cost more exchange steps per choice, more experts a lane more registers. 65536 tokens of 256
// fp32 experts on 16 lanes of 16 and 8 lanes of 32: forward 47 and 43, backward 36 and 57 us;
// 131072 tokens of 64 on 8 lanes of 8 and 4 of 16: 27 and 27, 18 and 54 us.
template <typename F>
int by_experts(int64_t E, F f) {
  if (E <= 8) return f(std::integral_constant<int, 1>(), std::integral_constant<int, 8>());
  if (E <= 16) return f(std::integral_constant<int, 2>(), std::integral_constant<int, 8>());
  if (E <= 32) return f(std::integral_constant<int, 4>(), std::integral_constant<int, 8>());
  if (E <= 64) return f(std::integral_constant<int, 8>(), std::integral_constant<int, 8>());
  if (E <= 128) return f(std::integral_constant<int, 16>(), std::integral_constant<int, 8>());
  if (E <= 256) return f(std::integral_constant<int, 16>(), std::integral_constant<int, 16>());
  if (E <= 512) return f(std::integral_constant<int, 32>(), std::integral_constant<int, 16>());
  return f(std::integral_constant<int, 64>(), std::integral_constant<int, 16>());
}

int lanes_of(int64_t E) {
  return by_experts(E, [](auto G, auto) { return (int)decltype(G)::value; });
}

// Forward workgroups: two of 512 threads per CU (of fp32 logits of more than 128 experts, whose 153 to 157
// registers leave room for one, half of them wait: 131072 tokens of 256 take 71 us, in bf16 41); their
// partials (E sums and counts each) are what
// the finishing workgroups read. 131071 tokens of 256 bf16 experts with 256, 512 and 1024 of
// them: 52, 45 and 48 us.
constexpr int MAX_BLOCKS = 512;
// Backward workgroups: four of 256 threads per CU. With 512, 1024 and 2048 of them the backward pass of
// 131071 x 256 bf16 took 39, 34 and 41 us, of 65536 x 256 fp32 33, 36 and 45 (each has the experts'
// coefficients to make first).
constexpr int MAX_BWD_BLOCKS = 1024;
constexpr int64_t WS_HEAD = (EMAX / 16) * 8 + 8;  // part_b, ticket
int forward_blocks(int64_t T, int64_t E) {
  const int64_t groups = FWD_THREADS / lanes_of(E);
  return (int)std::max<int64_t>(1, std::min<int64_t>((T + groups - 1) / groups, MAX_BLOCKS));
}

bool io_ok(int dt) { return dt == MUON_DT_F32 || dt == MUON_DT_BF16 || dt == MUON_DT_F16; }

int check(const char* what, int dtype, int64_t T, int64_t E, int64_t k, int64_t row) {
  if (!io_ok(dtype)) {
    muon_set_error("%s: unsupported dtype %d", what, dtype);
    return MUON_ERR_DTYPE;
  }
  if (T < 0 || T >= (1LL << 31) || E < 1 || E > EMAX || k < 1 || k > E || k > KMAX || (T > 1 && row < 0)) {
    muon_set_error("%s: bad extents (tokens %lld, experts %lld in 1..%d, top %lld in 1..%d and at "
                   "most the experts)", what, (long long)T, (long long)E, EMAX, (long long)k, KMAX);
    return MUON_ERR_SHAPE;
  }
  return MUON_OK;
}

}  // namespace

extern "C" {

int64_t muon_route_workspace_bytes(int64_t tokens, int64_t experts) {
  if (tokens < 0 || experts < 1 || experts > EMAX) return -1;
  return WS_HEAD + (int64_t)forward_blocks(tokens, experts) * (experts * 8 + 8);
}

int muon_route(const void* logits, int dtype, int64_t row_stride, int64_t tokens, int64_t experts,
               int64_t top, int normalize, const void* token_mask, float* gates,
               int64_t* chosen, int64_t* counts, float* balance, float* zloss, float* kept, void* ws,
               void* stream) {
  const int rc = check("route", dtype, tokens, experts, top, row_stride);
  if (rc) return rc;
  if (!counts || !balance || !zloss || !kept || !ws || (tokens && (!logits || !gates || !chosen))) {
    muon_set_error("route: null tensor");
    return MUON_ERR_ARG;
  }
  const int blocks = forward_blocks(tokens, experts);
  Args a = {logits, row_stride, tokens, (int)experts, (int)top, normalize,
            (const uint8_t*)token_mask, gates, chosen, counts, balance,
            zloss, kept, (double*)ws, nullptr, nullptr, nullptr, nullptr, nullptr};
  a.ticket = (int*)(a.part_b + EMAX / 16);
  a.part_p = (float*)((char*)ws + WS_HEAD);
  a.part_c = (int*)(a.part_p + (int64_t)blocks * experts);
  a.part_z = (float*)(a.part_c + (int64_t)blocks * experts);
  a.part_n = (int*)(a.part_z + blocks);
  hipStream_t s = (hipStream_t)stream;
  const int r = by_experts(experts, [&](auto G, auto V) {
    constexpr int g = decltype(G)::value, v = decltype(V)::value;
    if (dtype == MUON_DT_F32) route_kernel<MUON_DT_F32, g, v><<<blocks, FWD_THREADS, 0, s>>>(a);
    else if (dtype == MUON_DT_BF16) route_kernel<MUON_DT_BF16, g, v><<<blocks, FWD_THREADS, 0, s>>>(a);
    else route_kernel<MUON_DT_F16, g, v><<<blocks, FWD_THREADS, 0, s>>>(a);
    MUON_CHECK_LAUNCH("route");
    return MUON_OK;
  });
  if (r || blocks == 1) return r;
  route_finish_kernel<<<(unsigned)((experts + 15) / 16), 1024, 0, s>>>(a, blocks);
  MUON_CHECK_LAUNCH("route totals");
  return MUON_OK;
}

int muon_route_backward(const void* logits, int dtype, int64_t row_stride, int64_t tokens,
                        int64_t experts, int64_t top, int normalize, const void* token_mask,
                        const int64_t* chosen, const int64_t* counts, const float* kept,
                        const float* dgates, const float* dbalance, const float* dzloss,
                        void* dlogits, void* stream) {
  const int rc = check("route_backward", dtype, tokens, experts, top, row_stride);
  if (rc || tokens == 0) return rc;
  if (!logits || !chosen || !counts || !kept || !dlogits) {
    muon_set_error("route_backward: null tensor");
    return MUON_ERR_ARG;
  }
  const BackArgs a = {logits, row_stride, tokens, (int)experts, (int)top, normalize,
                      (const uint8_t*)token_mask, chosen, counts, kept, dgates, dbalance, dzloss,
                      dlogits};
  hipStream_t s = (hipStream_t)stream;
  return by_experts(experts, [&](auto G, auto V) {
    constexpr int g = decltype(G)::value, v = decltype(V)::value;
    const int64_t groups = BWD_THREADS / g;
    const int grid = (int)std::min<int64_t>((tokens + groups - 1) / groups, MAX_BWD_BLOCKS);
    if (dtype == MUON_DT_F32) route_backward_kernel<MUON_DT_F32, g, v><<<grid, BWD_THREADS, 0, s>>>(a);
    else if (dtype == MUON_DT_BF16) route_backward_kernel<MUON_DT_BF16, g, v><<<grid, BWD_THREADS, 0, s>>>(a);
    else route_backward_kernel<MUON_DT_F16, g, v><<<grid, BWD_THREADS, 0, s>>>(a);
    MUON_CHECK_LAUNCH("route_backward");
    return MUON_OK;
  });
}

}  // extern "C"
