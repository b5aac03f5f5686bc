// The MoE router on the device: the choice of topk experts per token with its gradient, and the balance
// loss with the experts' counts and its gradient.  C-ABI: flygemm_moe_topk, flygemm_moe_topk_grad,
// flygemm_moe_balance, flygemm_moe_balance_grad (include/flygemm.h has the formulas).
//
// A wave holds whole rows of logits (one to four of them): lane l the V consecutive experts from l * V (V = 1, 2,
// 4, 8 for up to 512 experts).  Sums and maxima over a row go through DPP (row shifts, then row broadcasts), in a fixed
// order, so every result is the same from run to run.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "../../include/flygemm.h"
#include "abi_error.h"

using namespace flygemm;

namespace {

constexpr int kMaxExperts = FLYGEMM_MOE_SORT_MAX_EXPERTS;
constexpr int kMaxTokens = FLYGEMM_MOE_ROUTER_MAX_TOKENS;
constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr float kInf = __builtin_inff();

// HIP launches fewer than 2^32 threads in a dimension: grids go on in y behind kGridX workgroups (of at most 1024
// threads), and those past the last row or sequence return.
constexpr int kGridX = 1 << 20;
dim3 grid_of(int64_t groups) {
  return groups <= kGridX ? dim3((unsigned)groups) : dim3(kGridX, (unsigned)((groups + kGridX - 1) / kGridX));
}
__device__ __forceinline__ long workgroup() { return (long)blockIdx.y * kGridX + blockIdx.x; }

// ---- reductions over a wave ------------------------------------------------------------
// one DPP step: lanes without a source keep `old`
template <int CTRL, int ROWS>
__device__ __forceinline__ float dpp(float old, float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(__builtin_bit_cast(int, old), __builtin_bit_cast(int, v),
                                                               CTRL, ROWS, 0xf, false));
}
template <int CTRL, int ROWS>
__device__ __forceinline__ double dpp(double old, double v) {
  const uint64_t o = __builtin_bit_cast(uint64_t, old), x = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp((int)(uint32_t)o, (int)(uint32_t)x, CTRL, ROWS, 0xf, false);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp((int)(o >> 32), (int)(x >> 32), CTRL, ROWS, 0xf, false);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ float at_lane(float v, int lane) {
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane));
}
__device__ __forceinline__ double at_lane(double v, int lane) {
  const uint64_t x = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)x, lane);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(x >> 32), lane);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
template <typename T>
__device__ __forceinline__ T larger(T a, T b) { return a < b ? b : a; }
__device__ __forceinline__ float larger(float a, float b) { return __builtin_fmaxf(a, b); }

// row_shr 1, 2, 4, 8 gather each row of 16 lanes in its last lane, row_bcast 15 and 31 join the rows: the
// result is in lane 63 and comes back to all lanes as a scalar
template <typename T>
__device__ __forceinline__ T wave_max(T v) {
  v = larger(v, dpp<0x111, 0xf>(v, v));
  v = larger(v, dpp<0x112, 0xf>(v, v));
  v = larger(v, dpp<0x114, 0xf>(v, v));
  v = larger(v, dpp<0x118, 0xf>(v, v));
  v = larger(v, dpp<0x142, 0xa>(v, v));
  v = larger(v, dpp<0x143, 0xc>(v, v));
  return at_lane(v, 63);
}
template <typename T>
__device__ __forceinline__ T wave_sum(T v) {
  const T z = T(0);
  v += dpp<0x111, 0xf>(z, v);
  v += dpp<0x112, 0xf>(z, v);
  v += dpp<0x114, 0xf>(z, v);
  v += dpp<0x118, 0xf>(z, v);
  v += dpp<0x142, 0xa>(z, v);
  v += dpp<0x143, 0xc>(z, v);
  return at_lane(v, 63);
}

// Floats as integers of the same order (-0 as 0, which it equals): integer minima and maxima take a DPP
// operand in the same instruction, where fmaxf needs a move and a canonicalization in front of it.
constexpr int kNone = -2147483647 - 1;   // below every number
__device__ __forceinline__ int order_int(float v) {
  const int i = __builtin_bit_cast(int, v + 0.f);
  return i ^ ((i >> 31) & 0x7fffffff);
}
__device__ __forceinline__ float order_float(int i) { return __builtin_bit_cast(float, i ^ ((i >> 31) & 0x7fffffff)); }
template <int CTRL, int ROWS = 0xf>
__device__ __forceinline__ int dpp_max(int v) {   // lanes without a source: v
  return max(v, __builtin_amdgcn_update_dpp(kNone, v, CTRL, ROWS, 0xf, false));
}
template <int CTRL>
__device__ __forceinline__ int dpp_all(int v) {   // patterns in which every lane has a source
  return __builtin_amdgcn_update_dpp(0, v, CTRL, 0xf, 0xf, true);
}
__device__ __forceinline__ int wave_max(int v) {
  v = dpp_max<0x111>(v);
  v = dpp_max<0x112>(v);
  v = dpp_max<0x114>(v);
  v = dpp_max<0x118>(v);
  v = dpp_max<0x142, 0xa>(v);
  v = dpp_max<0x143, 0xc>(v);
  return __builtin_amdgcn_readlane(v, 63);
}
__device__ __forceinline__ uint64_t lanes_below(int lane) { return (1ull << lane) - 1; }

// ---- rows ------------------------------------------------------------------------------
template <typename T, int N>
struct alignas(sizeof(T) * N) Pack {
  T v[N];
};

// this lane's V logits of a row (kInf's negative past the last expert); VEC: E % V == 0 and every row
// starts at a multiple of the pack
template <typename T, int V>
__device__ __forceinline__ void load_row(const T* row, int E, int lane, bool vec, float (&x)[V]) {
  const int e0 = lane * V;
#pragma unroll
  for (int j = 0; j < V; ++j) x[j] = -kInf;
  if (vec) {
    if (e0 < E) {
      const Pack<T, V> p = *(const Pack<T, V>*)(row + e0);
#pragma unroll
      for (int j = 0; j < V; ++j) x[j] = (float)p.v[j];
    }
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (e0 + j < E) x[j] = (float)row[e0 + j];
  }
}

template <typename T, int V>
__device__ __forceinline__ void store_row(T* row, int E, int lane, bool vec, const float (&x)[V]) {
  const int e0 = lane * V;
  if (vec) {
    if (e0 < E) {
      Pack<T, V> p;
#pragma unroll
      for (int j = 0; j < V; ++j) p.v[j] = (T)x[j];
      *(Pack<T, V>*)(row + e0) = p;
    }
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (e0 + j < E) row[e0 + j] = (T)x[j];
  }
}

// exp of a difference to a row's maximum: the hardware's exp2 (1 ulp), whose argument is rounded by 2^-24 of itself.  For
// sums of a row and terms next to them, where that is R 2^-24 of the value, R the row's range (expf keeps its argument
// exact, for several instructions more); weights that are returned take expf.
__device__ __forceinline__ float exp_fast(float x) { return __builtin_amdgcn_exp2f(x * 1.4426950408889634f); }
// expf rather than exp_fast: for x far below 0 the relative error of the result is that of exp(-x).  The hardware's
// reciprocal is within 1 ulp; a division, within half of one, takes several instructions more.
__device__ __forceinline__ float sigmoid(float x) { return __builtin_amdgcn_rcpf(1.f + expf(-x)); }
__device__ __forceinline__ double sigmoid(double x) { return 1.0 / (1.0 + exp(-x)); }

// ---- the choice ------------------------------------------------------------------------
struct TopkArgs {
  int32_t* ids;         // [T][k]
  float* weights;       // [T][k]
  const void* x;        // logits, rows `stride` elements apart
  const float* bias;    // [E] or null
  const uint8_t* mask;  // [T] or null
  int64_t stride;
  int T, E, k, G, gsel;
  int sigmoid, renorm, vec;
  float scale;
};

// Rows that a wave takes: four (two of 8 logits a lane, for the registers), or one.  Row r leaves its ids in
// lanes 16 r to 16 r + 15, so that the weights of all are computed at once; above 16 ids a wave takes one row.
constexpr int choice_rows(int V) { return V == 8 ? 2 : 4; }
// Where a wave takes them: from 8192 tokens, below which one row to a wave has the shorter way (graph-timed on
// MI355X, top-8 sigmoid, one row / several: 2048 x 256 4.2 us / 5.9, 4096 x 256 5.4 / 6.1, 8192 x 256 7.6 / 6.9, 16384 x 256
// 12.4 / 9.0, 8192 x 128 5.7 / 5.8, 16384 x 64 7.5 / 6.8); with more than 256 experts always, whose lists of eight choose_row sorts
// in every lane (2048 x 512 8.8 / 5.7, 16384 x 512 45.3 / 12.6).  The gradients differ by less (16384 x 256 6.9 / 6.1).
// Above 16 ids there is one row to a wave, and its time grows with k (softmax without a bias, k = 16 / 17 / 32 / 64:
// 32768 x 256 22.5 / 36 / 57 / 102, 16384 x 512 18 / 67 / 104 / 182).
constexpr int kManyTokens = 8192;
bool several_rows(int tokens, int experts, int topk) {
  return topk <= 16 && (experts > 256 || tokens >= kManyTokens);
}

// Reductions over the ids of one row: 16 lanes (a DPP row, rotated by 8, 4, 2, 1), or the wave
template <bool MAX>
__device__ __forceinline__ float row16(float v) {
  float o = dpp<0x128, 0xf>(v, v);
  v = MAX ? larger(v, o) : v + o;
  o = dpp<0x124, 0xf>(v, v);
  v = MAX ? larger(v, o) : v + o;
  o = dpp<0x122, 0xf>(v, v);
  v = MAX ? larger(v, o) : v + o;
  o = dpp<0x121, 0xf>(v, v);
  return MAX ? larger(v, o) : v + o;
}
__device__ __forceinline__ float ids_max(bool one, float v) { return one ? wave_max(v) : row16<true>(v); }
__device__ __forceinline__ float ids_sum(bool one, float v) { return one ? wave_sum(v) : row16<false>(v); }

// Weights of the chosen experts, a lane holding expert id (or -1) and its logit xi; `one`: one row in the
// wave, else one in every 16 lanes.
//   renorm   s_i / sum of the chosen s.  Softmax: the softmax of the chosen logits, whatever the others are.
//            Sigmoid: where every chosen logit is below -60, sigmoid(x) is exp(x) to 1e-26 and the quotient
//            again a softmax, which does not underflow.
//   else     s_i itself; m and sum are the row's maximum and sum of exp(x - m) (softmax only).
__device__ __forceinline__ float chosen_score(bool one, bool sig, bool renorm, bool have, float xi, float m, float sum) {
  if (renorm) {
    const float top = ids_max(one, have ? xi : -kInf);
    const float s = !have ? 0.f : (sig && top > -60.f) ? sigmoid(xi) : expf(xi - top);
    const float total = ids_sum(one, s);
    return have ? s / total : 0.f;
  }
  return !have ? 0.f : sig ? sigmoid(xi) : expf(xi - m) / sum;
}

// Two fp32 keys closer than this may be in the other order in 64 bits: twice a key's error.  u = 2^-24:
//   sigmoid  exp2 2 u and its argument 1.22 |x| u, both of e = exp(-x), count s (1 - s) <= 0.25 and s (1 - s) |x| <= 0.23
//            times; 1 + e and the reciprocal u each (s < 1): 2.8 u in all
//   softmax  of p: the same two errors of its own exp2 and the difference's u |x - m| (p |x - m| <= 0.37), and the sum's:
//            the terms' differences and arguments 2.22 ln 512 u on average, 14 additions, exp2, reciprocal and product:
//            33 u p + 0.9 u in all
// and the sum with the bias u |key|.  Taken are 4 u, 40 u pmax + 2 u, and 2 u |key|.
__device__ __forceinline__ float near(float key, bool sig, float pmax) {
  return sig ? 0x1p-21f + 0x1p-22f * __builtin_fabsf(key)
             : 0x1.4p-18f * pmax + 0x1p-22f * (1.f + __builtin_fabsf(key));
}

// The k experts with the largest keys in 64 bits, in order: expert i's id in lane `first` + i (the other lanes keep
// id).  Lane l holds the keys of experts l * V + j, -inf where an expert cannot be chosen.  The plain form:
// groups through LDS, then k times the largest head of the lanes' sorted lists.
template <int V>
__device__ __forceinline__ void choose64(const TopkArgs& p, int lane, int first, double (&key)[V], double* group_keys, int& id) {
  const double low = -(double)kInf;
  const int e0 = lane * V;
  if (p.G > 1) {
    const int per = p.E / p.G;
#pragma unroll
    for (int j = 0; j < V; ++j) group_keys[e0 + j] = key[j];
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    double a = low, b = low;
    if (lane < p.G)
      for (int i = 0; i < per; ++i) {
        const double v = group_keys[lane * per + i];
        b = v > a ? a : larger(b, v);
        a = larger(a, v);
      }
    const double score = b > low ? a + b : a;
    int rank = 0;
    for (int g = 0; g < p.G; ++g) {
      const double other = at_lane(score, g);
      rank += g < lane ? other >= score : other > score;
    }
    const uint64_t kept = __ballot(lane < p.G && rank < p.gsel);
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (!((kept >> ((unsigned)(e0 + j) / (unsigned)per & 63)) & 1)) key[j] = low;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
  int idx[V];
#pragma unroll
  for (int j = 0; j < V; ++j) idx[j] = e0 + j;
#pragma unroll
  for (int r = 0; r < V; ++r)
#pragma unroll
    for (int j = r & 1; j + 1 < V; j += 2) {
      const bool swap = key[j] < key[j + 1];
      const double ka = swap ? key[j + 1] : key[j], kb = swap ? key[j] : key[j + 1];
      const int ia = swap ? idx[j + 1] : idx[j], ib = swap ? idx[j] : idx[j + 1];
      key[j] = ka, key[j + 1] = kb, idx[j] = ia, idx[j + 1] = ib;
    }
  for (int i = 0; i < p.k; ++i) {
    const double best = wave_max(key[0]);
    if (!(best > low)) break;
    const int src = __builtin_ctzll(__ballot(key[0] == best));
    const int e = __builtin_amdgcn_readlane(idx[0], src);
    if (lane == first + i) id = e;
    if (lane == src) {
#pragma unroll
      for (int j = 0; j + 1 < V; ++j) key[j] = key[j + 1], idx[j] = idx[j + 1];
      key[V - 1] = low;
    }
  }
}

// Drops the experts of the groups that are not among the best, for R rows at once (keys in order_int's form,
// kNone: none).  Bit r of the result: fp32 keys may have chosen other groups of row r than exact ones
// (`approx`: they carry errors).
template <int V, int R>
__device__ __forceinline__ uint32_t keep_groups(const TopkArgs& p, int lane, int (&key)[R][V], bool approx,
                                                const float (&pmax)[R], int* lds) {
  const int e0 = lane * V, per = p.E / p.G, lanes = per / V;
  const bool aligned = lanes * V == per && (lanes & (lanes - 1)) == 0;
  int a[R], b[R];   // the two largest keys of this lane's group
  int group = lane;
#pragma unroll
  for (int r = 0; r < R; ++r) a[r] = b[r] = kNone;
  if (aligned) {
    // whole lanes, a power of two of them: in registers
    group = lane / lanes;
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        b[r] = max(b[r], min(a[r], key[r][j]));
        a[r] = max(a[r], key[r][j]);
      }
    auto join = [&](auto other) {
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const int oa = other(a[r]), ob = other(b[r]);
        b[r] = max(max(b[r], ob), min(a[r], oa));
        a[r] = max(a[r], oa);
      }
    };
    if (lanes >= 2) join([](int v) { return dpp_all<0xb1>(v); });     // quad_perm: neighbours
    if (lanes >= 4) join([](int v) { return dpp_all<0x4e>(v); });     // pairs of a quad
    if (lanes >= 8) join([](int v) { return dpp_all<0x141>(v); });    // row_half_mirror: the quads of eight lanes
    if (lanes >= 16) join([](int v) { return dpp_all<0x140>(v); });   // row_mirror: the halves of a row
    if (lanes >= 32) join([](int v) { return __shfl_xor(v, 16, 64); });
  } else {
    // through LDS: lane g scans group g
#pragma unroll
    for (int r = 0; r < R; ++r) {
#pragma unroll
      for (int j = 0; j < V; ++j) lds[e0 + j] = key[r][j];
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
      if (lane < p.G)
        for (int i = 0; i < per; ++i) {
          const int v = lds[lane * per + i];
          b[r] = max(b[r], min(a[r], v));
          a[r] = max(a[r], v);
        }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
    }
  }
  // a group's score: its largest key, or with a bias the sum of its two largest (of one where it has one);
  // its rank: the groups that score more, and the lower ones that score the same
  const int width = aligned ? lanes : 1;   // lanes that hold one group's score
  int score[R], rank[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    score[r] = p.bias && b[r] > kNone ? order_int(order_float(a[r]) + order_float(b[r])) : a[r];
    rank[r] = 0;
  }
  for (int g = 0; g < p.G; ++g) {
    const int tie = g < group ? 1 : 0;
#pragma unroll
    for (int r = 0; r < R; ++r)   // no score is kNone + 1, so that the difference does not wrap where it counts
      rank[r] += __builtin_amdgcn_readlane(score[r], g * width) > max(score[r], kNone + 1) - tie ? 1 : 0;
  }
  const bool real = group < p.G;
  uint32_t unsure = 0;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const bool in = real && rank[r] < p.gsel;
    if (approx) {
      // the errors of the two keys (by their sizes, which their sum may not show) and of the sum.  They differ from group
      // to group, so a rejected group's most is held against the least of all kept ones, not of the last alone; scores
      // that are infinite in fp32 may differ in 64 bits.
      const float fs = order_float(score[r]);
      const float close = 0.5f * (near(order_float(a[r]), p.sigmoid, pmax[r]) +
                                  (b[r] > kNone ? near(order_float(b[r]), p.sigmoid, pmax[r]) : 0.f)) +
                          0x1p-24f * __builtin_fabsf(fs);
      const bool scored = real && a[r] > kNone;
      const float edge = order_float(~wave_max(in && scored ? ~order_int(fs - close) : kNone));   // ~ turns the order round
      if (__ballot(scored && (!(__builtin_fabsf(fs) + close < kInf) || (!in && fs + close > edge)))) unsure |= 1u << r;
    }
    if (aligned) {
#pragma unroll
      for (int j = 0; j < V; ++j) key[r][j] = in ? key[r][j] : kNone;
    } else {
      const uint64_t kept = __ballot(in);
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (!((kept >> ((unsigned)(e0 + j) / (unsigned)per & 63)) & 1)) key[r][j] = kNone;
    }
  }
  return unsure;
}

// The k experts with the largest keys of one row: expert i in lane first + i of id, its key in kv (the other
// lanes keep theirs).  Returns the largest key that is left.
template <int V>
__device__ __forceinline__ int choose_row(int k, int lane, int first, const int (&keys)[V], int& id, int& kv) {
  // each lane's experts in order of their keys (equal keys keep their order), their indexes as nibbles
  int key[V];
  uint32_t j4[V], order = 0;
#pragma unroll
  for (int j = 0; j < V; ++j) key[j] = keys[j], j4[j] = j;
#pragma unroll
  for (int q = 0; q < V; ++q)
#pragma unroll
    for (int j = q & 1; j + 1 < V; j += 2) {
      const bool swap = key[j] < key[j + 1];
      const int ka = max(key[j], key[j + 1]), kb = min(key[j], key[j + 1]);
      const uint32_t ja = swap ? j4[j + 1] : j4[j], jb = swap ? j4[j] : j4[j + 1];
      key[j] = ka, key[j + 1] = kb, j4[j] = ja, j4[j + 1] = jb;
    }
#pragma unroll
  for (int j = V - 1; j >= 0; --j) order = order << 4 | j4[j];
  // the largest head of all lanes, the lowest lane's on equality (lanes hold consecutive experts): its
  // lane hands out that expert and moves to its next
  for (int i = 0; i < k; ++i) {
    const int best = wave_max(key[0]);
    const int src = __builtin_ctzll(__ballot(key[0] == best));
    const int e = src * V + (__builtin_amdgcn_readlane(order, src) & 15);
    const bool out = lane == first + i;
    id = out ? (best > kNone ? e : -1) : id;
    kv = out ? best : kv;
    const bool pop = lane == src;
#pragma unroll
    for (int j = 0; j + 1 < V; ++j) key[j] = pop ? key[j + 1] : key[j];
    key[V - 1] = pop ? kNone : key[V - 1];
    order >>= pop ? 4 : 0;
  }
  return wave_max(key[0]);
}

// The same of R rows and k up to 16, row r's in lanes 16 r to 16 r + 15.  Per row, a threshold that k to 16 keys reach
// is found by counting (downwards from the largest key in growing steps, then by halves); the keys that
// reach it go to the row's 16 lanes in order of their experts, through LDS, and there every lane counts the
// larger ones, which is its place.  Against taking the largest k times (choose_row, whose lists are popped in every
// lane for each), the whole kernel took 289 vector instructions a row of 256 experts with groups and a bias in place of
// 471; what settles doubts in 64 bits has made them 327.  A row with more than 16 keys
// that tie at its threshold takes choose_row.  The lanes behind the k-th hold the next candidates; their number is
// returned (of the lane's row), and rest is at least the largest key that is no candidate.
template <int V, int R>
__device__ __forceinline__ int choose_rows(int k, int lane, const int (&key)[R][V], int2 (*cand)[16], int& id, int& kv,
                                           int (&rest)[R]) {
  constexpr int kLeast = kNone + 1;
  uint32_t tied = 0;
  int count[R], limit[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    auto reach = [&](int t) {
      int n = 0;
#pragma unroll
      for (int j = 0; j < V; ++j) n += __builtin_popcountll(__ballot(key[r][j] >= t));
      return n;
    };
    int top = key[r][0];
#pragma unroll
    for (int j = 1; j < V; ++j) top = max(top, key[r][j]);
    top = wave_max(top);
    // hi: the largest key, or a threshold that fewer than k reach.  The steps end at kLeast: no key is above +inf's,
    // so after 2^20 + ... + 2^30 less than 2^31 is left, which the next step covers before it could wrap.
    int hi = top, t, n;
    uint32_t step = 1u << 20;
    for (;;) {
      const uint32_t room = (uint32_t)hi - (uint32_t)kLeast;
      t = top == kNone || step >= room ? kLeast : (int)((uint32_t)hi - step);
      n = reach(t);
      if (n >= k || t == kLeast) break;
      hi = t;
      step <<= 1;
    }
    if (n > 16) {
      int lo = t;   // n(lo) > 16, and n(hi) < k or hi is the largest key
      hi = hi == top ? top + 1 : hi;
      while (n > 16 || n < k) {
        t = (int)((uint32_t)lo + ((uint32_t)hi - (uint32_t)lo) / 2);
        if (t == lo) break;
        n = reach(t);
        if (n >= k) lo = t;
        else hi = t;
      }
      if (n > 16 || n < k) tied |= 1u << r;
    }
    count[r] = n, limit[r] = t;
    if (tied >> r & 1) {
      count[r] = 0;
      continue;
    }
    int pos = 0;   // candidates in lower lanes
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const uint64_t m = __ballot(key[r][j] >= t);
      pos = __builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, pos));
    }
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (key[r][j] >= t) cand[r][pos++] = int2{key[r][j], lane * V + j};
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
  const int at = lane & 15, row = lane >> 4;
  int mine = 0;
#pragma unroll
  for (int r = 0; r < R; ++r) mine = row == r ? count[r] : mine;
  int2 c = int2{kLeast, -1};   // below every number's key
  if (at < mine) c = cand[row][at];
  // larger keys, and equal ones of lower experts: the lane that row_ror:n reads from is n lower, or wraps
  int rank = 0;
#define LARGER(N) rank += dpp_all<0x120 + N>(c.x) > c.x - (at >= N ? 1 : 0) ? 1 : 0;
  LARGER(1) LARGER(2) LARGER(3) LARGER(4) LARGER(5) LARGER(6) LARGER(7) LARGER(8)
  LARGER(9) LARGER(10) LARGER(11) LARGER(12) LARGER(13) LARGER(14) LARGER(15)
#undef LARGER
  const int to = ((lane & 48) + rank) * 4;
  const int sid = __builtin_amdgcn_ds_permute(to, c.y), skey = __builtin_amdgcn_ds_permute(to, c.x);
  const bool out = at < mine;
  id = out ? sid : -1;
  kv = out ? skey : kNone;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    rest[r] = limit[r] > kLeast ? limit[r] - 1 : kNone;
    if (tied >> r & 1) {
      rest[r] = choose_row<V>(k, lane, 16 * r, key[r], id, kv);
      mine = row == r ? k : mine;
    }
  }
  return mine;
}

// Puts every row's candidates in the order of their 64-bit keys, the lower expert first where they are equal (lanes
// without one: id -1, key -inf).
__device__ __forceinline__ void order64(int lane, double key, int& id) {
  const int own = id < 0 ? 1 << 16 | lane : id;
  int rank = 0;
  auto beat = [&](double k, int i) { rank += k > key || (k == key && i < own) ? 1 : 0; };
#define BEAT(N) beat(dpp<0x120 + N, 0xf>(key, key), dpp_all<0x120 + N>(own));
  BEAT(1) BEAT(2) BEAT(3) BEAT(4) BEAT(5) BEAT(6) BEAT(7) BEAT(8) BEAT(9) BEAT(10) BEAT(11) BEAT(12) BEAT(13) BEAT(14) BEAT(15)
#undef BEAT
  id = __builtin_amdgcn_ds_permute(((lane & 48) + rank) * 4, id);
}

// R rows to a wave: choice_rows, or one.  BIAS: the choice compares scores plus a correction bias.  Rounded to
// fp32, such sums tie or swap for logits that differ, so where fp32 keys come closer than their errors, keys in 64
// bits decide: among a row's candidates, or, where the candidates or the groups are in doubt, the row again.  Without a bias the keys are
// the logits, and exact.
// Bound by issue: 32768 x 256 rows with groups and a bias 25 us (0.4 of it the bounds of every kept group; 2 more with
// every row in doubt chosen again, of which ten made the whole launch wait), all of it in 64 bits one row at a time 68;
// 13.5 without a bias.
template <typename T, int V, bool BIAS, int R>
__global__ void __launch_bounds__(kThreads) moe_topk_kernel(TopkArgs p) {
  __shared__ double lds[kWaves][64 * V];
  __shared__ int2 cand[kWaves][R][16];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const long row0 = (workgroup() * kWaves + wave) * R;
  if (row0 >= p.T) return;
  constexpr bool one = R == 1;
  const int E = p.E, e0 = lane * V;
  const bool sig = p.sigmoid;

  float x[R][V], bias[V];
  bool on[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    on[r] = row0 + r < p.T && !(p.mask && !p.mask[row0 + r]);
#pragma unroll
    for (int j = 0; j < V; ++j) x[r][j] = -kInf;
    if (on[r]) load_row<T, V>((const T*)p.x + (row0 + r) * p.stride, E, lane, p.vec, x[r]);
  }
  if constexpr (BIAS) {
#pragma unroll
    for (int j = 0; j < V; ++j) bias[j] = e0 + j < E ? p.bias[e0 + j] : 0.f;
  }

  int key[R][V];
  float m[R], sum[R], pmax[R];
  uint32_t bad = 0;
  [[maybe_unused]] uint32_t unsure = 0;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    m[r] = -kInf, sum[r] = 1.f, pmax[r] = 0.f;
    bool nan = false;
#pragma unroll
    for (int j = 0; j < V; ++j) nan |= x[r][j] != x[r][j];
    float ex[V];
    if (!sig) {
      int top = kNone;
#pragma unroll
      for (int j = 0; j < V; ++j) top = x[r][j] > -kInf ? max(top, order_int(x[r][j])) : top;
      top = wave_max(top);
      m[r] = top > kNone ? order_float(top) : -kInf;
      nan |= m[r] == kInf;   // inf - inf in the softmax
      if (m[r] > -kInf && (BIAS || !p.renorm)) {
        sum[r] = 0.f;
#pragma unroll
        for (int j = 0; j < V; ++j) {
          ex[j] = exp_fast(x[r][j] - m[r]);
          sum[r] += x[r][j] > -kInf ? ex[j] : 0.f;
        }
        sum[r] = wave_sum(sum[r]);
        pmax[r] = 1.f / sum[r];
      }
    }
    bad |= (__ballot(nan) != 0 ? 1u : 0u) << r;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      float v = x[r][j];
      if constexpr (BIAS) {
        const float s = sig ? __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(v * -1.4426950408889634f)) : ex[j] * pmax[r];
        v = v > -kInf ? s + bias[j] : -kInf;
      }
      key[r][j] = v > -kInf ? order_int(v) : kNone;
    }
  }
  if (p.G > 1) unsure = keep_groups<V, R>(p, lane, key, BIAS, pmax, (int*)lds[wave]);
  int id = -1, kv = kNone, rest[R], count = p.k;
  if constexpr (one) rest[0] = choose_row<V>(p.k, lane, 0, key[0], id, kv);
  else count = choose_rows<V, R>(p.k, lane, key, cand[wave], id, kv, rest);

  const int at = one ? lane : lane & 15;
  float m_ids = m[0], sum_ids = sum[0];   // of the row whose ids this lane holds
#pragma unroll
  for (int r = 1; r < R; ++r)
    if (lane >> 4 == r) m_ids = m[r], sum_ids = sum[r];
  if constexpr (BIAS) {
    // Gaps that fp32 cannot vouch for: behind a chosen key to the next candidate, which 64-bit keys of the
    // candidates settle; from the last chosen one to the keys that are no candidates, or between groups: the whole row
    float tail = pmax[0];
    int left = rest[0];
#pragma unroll
    for (int r = 1; r < R; ++r)
      if (lane >> 4 == r) tail = pmax[r], left = rest[r];
    const int next = __shfl_down(kv, 1, 64);
    const float mine = order_float(kv), floor = mine - near(mine, sig, tail);
    const bool chosen = at < p.k && id >= 0;
    uint64_t tight = __ballot(chosen && at + 1 < count && next > kNone && order_float(next) > floor);
    const uint64_t open = __ballot(chosen && at == p.k - 1 && left > kNone && order_float(left) > floor);
    if constexpr (one) {
      if (tight | open) unsure = 1;
    } else {
#pragma unroll
      for (int r = 0; r < R; ++r)
        if (open >> (16 * r) & 0xffff) unsure |= 1u << r;
      if (tight) {
        const long own = row0 + (lane >> 4);
        const bool have = id >= 0;
        const double xd = have ? (double)(float)((const T*)p.x + own * p.stride)[id] : 0.0;
        double sd;
        if (sig) {
          sd = sigmoid(xd);
        } else {
          double total = 1.0;
#pragma unroll 1
          for (int r = 0; r < R; ++r) {
            if (!(tight >> (16 * r) & 0xffff)) continue;
            float xr[V];
            load_row<T, V>((const T*)p.x + (row0 + r) * p.stride, E, lane, p.vec, xr);
            const double top = (double)at_lane(m_ids, 16 * r);
            double part = 0.0;
#pragma unroll
            for (int j = 0; j < V; ++j) part += xr[j] > -kInf ? exp((double)xr[j] - top) : 0.0;
            part = wave_sum(part);
            total = lane >> 4 == r ? part : total;
          }
          sd = exp(xd - (double)m_ids) / total;
        }
        int sorted = id;
        order64(lane, have ? sd + (double)p.bias[id] : -(double)kInf, sorted);
        id = tight >> (lane & 48) & 0xffff ? sorted : id;
      }
    }
#pragma unroll 1
    for (int r = 0; r < R; ++r) {
      if (!(unsure >> r & 1) || row0 + r >= p.T || (p.mask && !p.mask[row0 + r])) continue;
      // logits and biases read again: held for this, they cost the other rows registers
      float xr[V];
      load_row<T, V>((const T*)p.x + (row0 + r) * p.stride, E, lane, p.vec, xr);
      const double top = (double)at_lane(m_ids, 16 * r);
      double dkey[V], dsum = 0.0;
      if (!sig) {
#pragma unroll
        for (int j = 0; j < V; ++j) dsum += xr[j] > -kInf ? exp((double)xr[j] - top) : 0.0;
        dsum = wave_sum(dsum);
      }
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const double s = sig ? sigmoid((double)xr[j]) : exp((double)xr[j] - top) / dsum;
        const double v = s + (double)(e0 + j < E ? p.bias[e0 + j] : 0.f);
        dkey[j] = xr[j] > -kInf && v == v ? v : -(double)kInf;
      }
      const int first = 16 * r;
      if (one || lane >> 4 == r) id = -1;
      choose64<V>(p, lane, first, dkey, lds[wave], id);
    }
  }

  const long row = one ? row0 : row0 + (lane >> 4);
  const bool live = at < p.k && row < p.T && (one || lane < 16 * R);   // two rows leave half the lanes without one
  const bool have = live && id >= 0;
  const float xi = have ? (float)((const T*)p.x + row * p.stride)[id] : 0.f;
  const float w = chosen_score(one, sig, p.renorm, have, xi, m_ids, sum_ids);
  if (live) {
    p.ids[row * p.k + at] = id;
    p.weights[row * p.k + at] = bad >> (one ? 0 : lane >> 4) & 1 ? __builtin_nanf("") : w * p.scale;
  }
}

struct TopkGradArgs {
  void* dx;             // [T][E]
  const float* dw;      // [T][k]
  const int32_t* ids;   // [T][k]
  const void* x;
  int64_t stride;
  int T, E, k;
  int sigmoid, renorm, vec, vec_out;
  float scale;
};

// With t_i = q_i (dw_i - sum q dw) scale (renorm, q the weights before the scale) or s_i dw_i scale:
// dx_i = t_i (softmax) or t_i sigmoid(-x_i) for the chosen, and without renorm the softmax's
// -p_e sum t for every expert.  R rows to a wave as in the choice, row r's ids in lanes 16 r to 16 r + 15; their
// values go to the rows' experts through LDS.  Bound by writing [T][E]: 32768 x 256 fp32 9.0 us, one row to a wave and its
// ids handed round one by one 18.6.  A dense gradient (softmax without renorm) takes exp_fast for p, as the row's sum.
template <typename T, int V, int R>
__global__ void __launch_bounds__(kThreads) moe_topk_grad_kernel(TopkGradArgs p) {
  __shared__ __attribute__((aligned(32))) float lds[kWaves][R][64 * V];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const long row0 = (workgroup() * kWaves + wave) * R;
  if (row0 >= p.T) return;
  constexpr bool one = R == 1;
  const int E = p.E, e0 = lane * V, at = one ? lane : lane & 15, mine = one ? 0 : lane >> 4;
  const long row = row0 + mine;
  int id = -1;
  float dw = 0.f;
  if (at < p.k && row < p.T && (one || lane < 16 * R)) {   // two rows leave half the lanes without one
    id = p.ids[row * p.k + at];
    dw = p.dw[row * p.k + at];
  }
  const bool have = id >= 0 && id < E;
  const float xi = have ? (float)((const T*)p.x + row * p.stride)[id] : 0.f;
  const bool dense = !p.sigmoid && !p.renorm;
  float x[R][V], m_ids = 0.f, sum_ids = 1.f;
  if (dense) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (row0 + r >= p.T) break;
      load_row<T, V>((const T*)p.x + (row0 + r) * p.stride, E, lane, p.vec, x[r]);
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (row0 + r >= p.T) break;
      float m = -kInf, sum = 0.f;
#pragma unroll
      for (int j = 0; j < V; ++j) m = __builtin_fmaxf(m, x[r][j]);
      m = wave_max(m);
#pragma unroll
      for (int j = 0; j < V; ++j) sum += x[r][j] = exp_fast(x[r][j] - m);
      sum = wave_sum(sum);
#pragma unroll
      for (int j = 0; j < V; ++j) x[r][j] /= sum;
      if (mine == r) m_ids = m, sum_ids = sum;
    }
  }
  const float q = chosen_score(one, p.sigmoid, p.renorm, have, xi, m_ids, sum_ids);
  float t = have ? q * dw : 0.f;
  const float all = ids_sum(one, t);
  if (p.renorm) t -= q * all;
  t *= p.scale;
  if (p.sigmoid) t *= sigmoid(-xi);
  Pack<float, V> zero;
#pragma unroll
  for (int j = 0; j < V; ++j) zero.v[j] = 0.f;
#pragma unroll
  for (int r = 0; r < R; ++r) *(Pack<float, V>*)&lds[wave][r][e0] = zero;
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
  if (have) atomicAdd(&lds[wave][mine][id], t);   // one id, one expert: nothing to order
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
#pragma unroll
  for (int r = 0; r < R; ++r) {
    if (row0 + r >= p.T) break;
    float out[V];
    const Pack<float, V> v = *(const Pack<float, V>*)&lds[wave][r][e0];
    const bool any = (__ballot(have) >> (one ? 0 : 16 * r) & (one ? ~0ull : 0xffffull)) != 0;
    const float f = at_lane(all, 16 * r) * p.scale;
#pragma unroll
    for (int j = 0; j < V; ++j) out[j] = dense && any ? v.v[j] - x[r][j] * f : v.v[j];
    store_row<T, V>((T*)p.dx + (row0 + r) * E, E, lane, p.vec_out, out);
  }
}

// ---- the balance loss ------------------------------------------------------------------
// Tokens are cut into chunks of `chunk` rows, one workgroup each, and a chunk at the sequences' borders.
// The part of sequence b in chunk c goes to slot c + b of the scratch: parts in order of rows step in c or
// b, so no two share a slot, and there are at most chunks + sequences of them.
struct BalArgs {
  float* loss;          // [1]
  int32_t* counts;      // [E]
  float* aux;           // [B][E] f / n, then [1] 1 / (sequences with tokens)
  float* psum;          // [slots][64 V]
  int32_t* pcnt;        // [slots][64 V]
  int32_t* pn;          // [slots]
  double* seq_loss;     // [B]
  int32_t* seq_cnt;     // [B][E]
  int32_t* seq_n;       // [B]
  const void* x;
  const void* ids;
  const uint8_t* mask;
  const int32_t* cu;    // [B + 1] or null
  int64_t stride;
  int T, E, k, B, chunk, ids64;
  int sigmoid, vec;
};

__device__ __forceinline__ int seq_begin(const int32_t* cu, int b, int T) { return min(max(cu[b], 0), T); }

// first b in [0, B) whose end lies behind row r (B: none)
__device__ __forceinline__ int seq_of(const int32_t* cu, int B, int r) {
  int lo = 0, hi = B;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (cu[mid + 1] > r) hi = mid;
    else lo = mid + 1;
  }
  return lo;
}

// p of U rows: softmax, or sigmoid over its sum; straight-line code, so that the rows' reductions fill each
// other's waits.  Bit u of the result is clear for a row without a logit above -inf (a NaN counts as one), whose p is 0.
template <int V, int U>
__device__ __forceinline__ uint32_t row_probs(const float (&x)[U][V], bool sig, float (&pr)[U][V]) {
  float m[U];
  uint32_t any = 0;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    float top = x[u][0];
#pragma unroll
    for (int j = 1; j < V; ++j) top = __builtin_fmaxf(top, x[u][j]);   // of the numbers
    m[u] = order_float(wave_max(top == top ? order_int(top) : order_int(-kInf)));
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    bool have = m[u] > -kInf;
    if (!have) {
      bool nan = false;
#pragma unroll
      for (int j = 0; j < V; ++j) nan |= x[u][j] != x[u][j];
      have = __ballot(nan) != 0;
      m[u] = 0.f;
    }
    any |= (have ? 1u : 0u) << u;
  }
  float r[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    // sigmoids where the largest logit is not too low for them (see chosen_score)
    if (sig && m[u] > -60.f) {
#pragma unroll
      for (int j = 0; j < V; ++j) pr[u][j] = sigmoid(x[u][j]);
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) pr[u][j] = exp_fast(x[u][j] - m[u]);
    }
    float s = pr[u][0];
#pragma unroll
    for (int j = 1; j < V; ++j) s += pr[u][j];
    r[u] = s;
  }
#pragma unroll
  for (int u = 0; u < U; ++u) r[u] = wave_sum(r[u]);
#pragma unroll
  for (int u = 0; u < U; ++u) {
    r[u] = any >> u & 1 ? 1.f / r[u] : 0.f;
#pragma unroll
    for (int j = 0; j < V; ++j) pr[u][j] *= r[u];
  }
  return any;
}

// Rows of a wave in flight.  The gradient: 2, so that a wave's loads run under another's arithmetic (32768 x 256
// 16.8 us, 4 rows 17.4; 8192 x 128 bf16 6.2 / 7.5).
constexpr int part_rows(int V) { return V == 8 ? 4 : 8; }
constexpr int kGradRows = 2;
constexpr int kMaxChunk = 4096;   // kMaxTokens leaves room for a chunk behind the last token, so row numbers are ints

// A lane adds its experts' probabilities over the rows of its wave in fp32, the waves' sums in fp32 too: at most 4096 / 16
// additions of terms that are all positive, 2^-16 of the sum at worst and 6e-8 of the loss as measured, for half the registers of 64 bits;
// the chunks' sums are added in 64 bits (moe_balance_sum_kernel).
// One read of the logits; 32768 x 256 fp32 11.5-12 us with 16 waves to a workgroup and 8 rows of each in flight; 14.6 with
// 4 rows one after the other, 37 with 4 waves: one wave per SIMD waits for memory.
constexpr int kPartThreads = 1024, kPartWaves = kPartThreads / 64;
template <typename T, int V>
__global__ void __launch_bounds__(kPartThreads) moe_balance_part_kernel(BalArgs p) {
  __shared__ __attribute__((aligned(32))) float lsum[kPartWaves][64 * V];
  __shared__ int lcnt[64 * V];
  __shared__ uint8_t lvalid[kMaxChunk];
  __shared__ int ln;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int E = p.E;
  const int r0 = (int)blockIdx.x * p.chunk, r1 = (int)min((long)r0 + p.chunk, (long)p.T);
  int b = p.cu ? seq_of(p.cu, p.B, r0) : 0;
  for (; b < p.B; ++b) {
    const int lo = p.cu ? max(seq_begin(p.cu, b, p.T), r0) : r0, hi = p.cu ? min(seq_begin(p.cu, b + 1, p.T), r1) : r1;
    if (lo >= r1) break;
    if (lo >= hi) continue;
    for (int e = tid; e < 64 * V; e += kPartThreads) lcnt[e] = 0;
    if (tid == 0) ln = 0;
    float acc[V];
#pragma unroll
    for (int j = 0; j < V; ++j) acc[j] = 0.f;
    auto take = [&](auto rows, int r) {
      constexpr int U = decltype(rows)::value;
      float x[U][V], pr[U][V];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int row = r + u * kPartWaves;
#pragma unroll
        for (int j = 0; j < V; ++j) x[u][j] = -kInf;
        if (row < hi && !(p.mask && !p.mask[row])) load_row<T, V>((const T*)p.x + row * p.stride, E, lane, p.vec, x[u]);
      }
      const uint32_t any = row_probs<V, U>(x, p.sigmoid, pr);
#pragma unroll
      for (int u = 0; u < U; ++u) {
#pragma unroll
        for (int j = 0; j < V; ++j) acc[j] += pr[u][j];
      }
      const int mine = r + lane * kPartWaves;
      if (lane < U && mine < hi) lvalid[mine - r0] = any >> lane & 1;
    };
    // rows past the end cost as much as others: two at a time where few are left
    for (int r = lo + wave; r < hi;) {
      if (hi - r > 2 * kPartWaves) {
        take(std::integral_constant<int, part_rows(V)>{}, r);
        r += part_rows(V) * kPartWaves;
      } else {
        take(std::integral_constant<int, 2>{}, r);
        r += 2 * kPartWaves;
      }
    }
    Pack<float, V> pack;
#pragma unroll
    for (int j = 0; j < V; ++j) pack.v[j] = acc[j];
    *(Pack<float, V>*)&lsum[wave][lane * V] = pack;
    __syncthreads();
    const int n_ids = (hi - lo) * p.k;
    int n = 0;
    for (int i = tid; i < n_ids; i += kPartThreads) {
      const int rr = lo + i / p.k;
      if (!lvalid[rr - r0]) continue;
      n += i % p.k == 0;
      const int64_t at = (int64_t)lo * p.k + i;
      const int64_t e = p.ids64 ? ((const int64_t*)p.ids)[at] : (int64_t)((const int32_t*)p.ids)[at];
      if (e >= 0 && e < E) atomicAdd(&lcnt[e], 1);
    }
    if (n) atomicAdd(&ln, n);
    __syncthreads();
    const int64_t slot = (int64_t)blockIdx.x + b;
    for (int e = tid; e < 64 * V; e += kPartThreads) {
      float s = 0.f;
#pragma unroll
      for (int w = 0; w < kPartWaves; ++w) s += lsum[w][e];
      p.psum[slot * (64 * V) + e] = s;
      p.pcnt[slot * (64 * V) + e] = lcnt[e];
    }
    if (tid == 0) p.pn[slot] = ln;
    __syncthreads();
  }
}

// One workgroup per sequence: its parts' sums (in 64 bits), f, P and loss; with one sequence the whole
// result.  A wave takes every 16th part, a lane the V experts that it has in the other kernels, so that a
// wave's loads of several parts are in flight together.
constexpr int kSumThreads = 1024, kSumWaves = kSumThreads / 64;
template <int V>
__global__ void __launch_bounds__(kSumThreads) moe_balance_sum_kernel(BalArgs p) {
  __shared__ __attribute__((aligned(32))) double lp[kSumWaves / 2][64 * V];
  __shared__ __attribute__((aligned(32))) int lc[kSumWaves / 2][64 * V];
  __shared__ int ln;
  if (workgroup() >= p.B) return;
  const int tid = threadIdx.x, lane = tid & 63, b = (int)workgroup(), E = p.E, e0 = lane * V;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lo = p.cu ? seq_begin(p.cu, b, p.T) : 0, hi = p.cu ? seq_begin(p.cu, b + 1, p.T) : p.T;
  const int c0 = lo / p.chunk, c1 = lo < hi ? (hi - 1) / p.chunk + 1 : c0;
  if (tid == 0) ln = 0;
  double s[V];
  int c[V], n = 0;
#pragma unroll
  for (int j = 0; j < V; ++j) s[j] = 0.0, c[j] = 0;
  constexpr int U = V == 8 ? 4 : 8;   // parts in flight
  for (int i = c0 + wave; i < c1; i += kSumWaves * U) {
    Pack<float, V> ps[U];
    Pack<int, V> pc[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t slot = (int64_t)min(i + u * kSumWaves, c1 - 1) + b;
      ps[u] = *(const Pack<float, V>*)(p.psum + slot * (64 * V) + e0);
      pc[u] = *(const Pack<int, V>*)(p.pcnt + slot * (64 * V) + e0);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (i + u * kSumWaves >= c1) break;
#pragma unroll
      for (int j = 0; j < V; ++j) s[j] += (double)ps[u].v[j], c[j] += pc[u].v[j];
    }
  }
  for (int i = c0 + tid; i < c1; i += kSumThreads) n += p.pn[(int64_t)i + b];
  __syncthreads();
  if (n) atomicAdd(&ln, n);
#pragma unroll
  for (int half = kSumWaves / 2; half >= 1; half /= 2) {
    if (wave >= half && wave < 2 * half) {
#pragma unroll
      for (int j = 0; j < V; ++j) lp[wave - half][e0 + j] = s[j], lc[wave - half][e0 + j] = c[j];
    }
    __syncthreads();
    if (wave < half) {
#pragma unroll
      for (int j = 0; j < V; ++j) s[j] += lp[wave][e0 + j], c[j] += lc[wave][e0 + j];
    }
    __syncthreads();
  }
  if (wave) return;
  n = ln;
  double t = 0.0;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    if (e0 + j >= E) break;
    const double f = n ? (double)c[j] * E / ((double)p.k * n) : 0.0;
    if (n) t += f * s[j] / n;
    p.aux[(int64_t)b * E + e0 + j] = n ? (float)(f / n) : 0.f;
    if (p.B == 1) p.counts[e0 + j] = c[j];
    else p.seq_cnt[(int64_t)b * E + e0 + j] = c[j];
  }
  t = wave_sum(t);
  if (lane == 0) {
    if (p.B == 1) {
      *p.loss = (float)t;
      p.aux[E] = 1.f;
    } else {
      p.seq_loss[b] = t;
      p.seq_n[b] = n;
    }
  }
}

__global__ void __launch_bounds__(kThreads) moe_balance_finish_kernel(BalArgs p) {
  const int tid = threadIdx.x;
  for (int e = tid; e < p.E; e += kThreads) {
    int c = 0;
#pragma unroll 8
    for (int b = 0; b < p.B; ++b) c += p.seq_cnt[(int64_t)b * p.E + e];
    p.counts[e] = c;
  }
  if (tid < 64) {
    double t = 0.0, g = 0.0;
    for (int b = tid; b < p.B; b += 64)
      if (p.seq_n[b]) t += p.seq_loss[b], g += 1.0;
    t = wave_sum(t);
    g = wave_sum(g);
    if (tid == 0) {
      *p.loss = g > 0.0 ? (float)(t / g) : 0.f;
      p.aux[(int64_t)p.B * p.E] = g > 0.0 ? (float)(1.0 / g) : 0.f;
    }
  }
}

struct BalGradArgs {
  void* dx;             // [T][E]
  const float* dloss;   // [1]
  const float* aux;
  const void* x;
  const uint8_t* mask;
  const int32_t* cu;
  int64_t stride;
  int T, E, B;
  int sigmoid, vec, vec_out;
};

// dx = p (h - sum p h) [sigmoid: times sigmoid(-x)], h = dloss f / (n G); 0 in rows that count for no
// sequence.  Bound by reading and writing [T][E].
template <typename T, int V>
__global__ void __launch_bounds__(kThreads) moe_balance_grad_kernel(BalGradArgs p) {
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int E = p.E, e0 = lane * V;
  const long first = (workgroup() * kWaves + wave) * kGradRows;
  if (first >= p.T) return;
  const float scale = *p.dloss * p.aux[(int64_t)p.B * E];
  int b = p.cu ? seq_of(p.cu, p.B, (int)first) : 0;
  float x[kGradRows][V], pr[kGradRows][V], h[kGradRows][V], dot[kGradRows];
  uint32_t in = 0;
#pragma unroll
  for (int u = 0; u < kGradRows; ++u) {
    const long row = first + u;
#pragma unroll
    for (int j = 0; j < V; ++j) x[u][j] = -kInf, h[u][j] = 0.f;
    bool on = row < p.T && !(p.mask && !p.mask[row]);
    if (p.cu && on) {
      while (b < p.B && p.cu[b + 1] <= row) ++b;
      on = b < p.B && p.cu[b] <= row;
    }
    if (on) {
      in |= 1u << u;
      load_row<T, V>((const T*)p.x + row * p.stride, E, lane, p.vec, x[u]);
#pragma unroll
      for (int j = 0; j < V; ++j) h[u][j] = e0 + j < E ? p.aux[(int64_t)b * E + e0 + j] : 0.f;
    }
  }
  in &= row_probs<V, kGradRows>(x, p.sigmoid, pr);
#pragma unroll
  for (int u = 0; u < kGradRows; ++u) {
    dot[u] = pr[u][0] * h[u][0];
#pragma unroll
    for (int j = 1; j < V; ++j) dot[u] += pr[u][j] * h[u][j];
  }
#pragma unroll
  for (int u = 0; u < kGradRows; ++u) dot[u] = wave_sum(dot[u]);
#pragma unroll
  for (int u = 0; u < kGradRows; ++u) {
    if (first + u >= p.T) break;
    float out[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
      out[j] = pr[u][j] * (h[u][j] - dot[u]) * scale;
      if (p.sigmoid) out[j] *= sigmoid(-x[u][j]);
      if (!(in >> u & 1)) out[j] = 0.f;
    }
    store_row<T, V>((T*)p.dx + (first + u) * E, E, lane, p.vec_out, out);
  }
}

// ---- host ------------------------------------------------------------------------------
int elem_bytes(int dtype) { return dtype == FLYGEMM_QIN_F32 ? 4 : 2; }
int row_pack(int E) { return E <= 64 ? 1 : E <= 128 ? 2 : E <= 256 ? 4 : 8; }
bool packs_fit(const void* base, int64_t stride, int E, int dtype) {
  const int v = row_pack(E), b = v * elem_bytes(dtype);
  return E % v == 0 && stride % v == 0 && (uintptr_t)base % (b > 16 ? 16 : b) == 0 && (uintptr_t)base % b == 0;
}

// calls f with a value of the logits' type and the experts per lane
template <typename F>
void by_row(int dtype, int E, F f) {
  auto with_type = [&](auto t) {
    typedef decltype(t) T;
    if (E <= 64) f(T{}, std::integral_constant<int, 1>{});
    else if (E <= 128) f(T{}, std::integral_constant<int, 2>{});
    else if (E <= 256) f(T{}, std::integral_constant<int, 4>{});
    else f(T{}, std::integral_constant<int, 8>{});
  };
  if (dtype == FLYGEMM_QIN_F32) with_type(float{});
  else if (dtype == FLYGEMM_QIN_BF16) with_type((__bf16)0.f);
  else with_type((_Float16)0.f);
}

int check_router(const char* what, int64_t stride, int T, int E, int dtype, int scoring) {
  if (T < 0 || E < 1) return fail(hipErrorInvalidValue, "%s: invalid sizes tokens=%d experts=%d", what, T, E);
  if (E > kMaxExperts) return fail(hipErrorInvalidValue, "%s: experts=%d must be at most %d", what, E, kMaxExperts);
  if (T > kMaxTokens) return fail(hipErrorInvalidValue, "%s: tokens=%d must be at most %d", what, T, kMaxTokens);
  if (stride < 0) return fail(hipErrorInvalidValue, "%s: negative row stride", what);
  if (dtype < FLYGEMM_QIN_F16 || dtype > FLYGEMM_QIN_F32)
    return fail(hipErrorInvalidValue, "%s: dtype %d not supported", what, dtype);
  if (scoring != FLYGEMM_SCORE_SOFTMAX && scoring != FLYGEMM_SCORE_SIGMOID)
    return fail(hipErrorInvalidValue, "%s: scoring %d not supported", what, scoring);
  return 0;
}

int launched(const char* what) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? 0 : fail(e, "launch of %s failed: %s", what, hipGetErrorString(e));
}

// Rows per chunk of the balance loss: one workgroup per CU where there are rows enough for its 16 rows in
// flight, and at most kMaxChunk.
int balance_chunk(int T) {
  const int c = (T + 255) / 256;
  return c < 16 ? 16 : c > kMaxChunk ? kMaxChunk : c;
}
int64_t round16(int64_t n) { return (n + 15) / 16 * 16; }

}  // namespace

extern "C" {

int flygemm_moe_topk(int32_t* topk_ids, float* topk_weights, const void* logits, int64_t row_stride, const float* bias,
                     const uint8_t* token_mask, int32_t tokens, int32_t experts, int32_t topk, int32_t groups,
                     int32_t topk_groups, int32_t dtype, int32_t scoring, int32_t renormalize, float scale,
                     void* stream) {
  const char* what = "moe_topk";
  const int rc = check_router(what, row_stride, tokens, experts, dtype, scoring);
  if (rc) return rc;
  if (topk < 1 || topk > experts || topk > 64)
    return fail(hipErrorInvalidValue, "%s: topk=%d must be in 1 .. min(experts, 64)", what, topk);
  if (groups < 1 || groups > 64 || experts % groups || topk_groups < 1 || topk_groups > groups)
    return fail(hipErrorInvalidValue, "%s: groups=%d (at most 64, a divisor of the experts), topk_groups=%d", what, groups,
                topk_groups);
  if (topk > experts / groups * topk_groups)
    return fail(hipErrorInvalidValue, "%s: topk=%d above the experts of %d groups", what, topk, topk_groups);
  if (tokens == 0) return 0;
  if (!topk_ids || !topk_weights || !logits) return fail(hipErrorInvalidValue, "%s: null tensor pointer", what);
  TopkArgs a{topk_ids, topk_weights, logits, bias, token_mask, row_stride, tokens, experts, topk,
             topk_groups == groups ? 1 : groups, topk_groups, scoring == FLYGEMM_SCORE_SIGMOID, renormalize != 0,
             packs_fit(logits, row_stride, experts, dtype), scale};
  const bool many = several_rows(tokens, experts, topk);
  const long per_wg = (long)kWaves * (many ? choice_rows(row_pack(experts)) : 1);
  const dim3 grid = grid_of((tokens + per_wg - 1) / per_wg);
  by_row(dtype, experts, [&](auto t, auto v) {
    typedef decltype(t) T;
    constexpr int V = decltype(v)::value;
    auto go = [&](auto fn) { hipLaunchKernelGGL(fn, grid, dim3(kThreads), 0, (hipStream_t)stream, a); };
    if (bias && many) go(moe_topk_kernel<T, V, true, choice_rows(V)>);
    else if (bias) go(moe_topk_kernel<T, V, true, 1>);
    else if (many) go(moe_topk_kernel<T, V, false, choice_rows(V)>);
    else go(moe_topk_kernel<T, V, false, 1>);
  });
  return launched(what);
}

int flygemm_moe_topk_grad(void* dlogits, const float* dweights, const int32_t* topk_ids, const void* logits,
                          int64_t row_stride, int32_t tokens, int32_t experts, int32_t topk, int32_t dtype,
                          int32_t scoring, int32_t renormalize, float scale, void* stream) {
  const char* what = "moe_topk_grad";
  const int rc = check_router(what, row_stride, tokens, experts, dtype, scoring);
  if (rc) return rc;
  if (topk < 1 || topk > experts || topk > 64)
    return fail(hipErrorInvalidValue, "%s: topk=%d must be in 1 .. min(experts, 64)", what, topk);
  if (tokens == 0) return 0;
  if (!dlogits || !dweights || !topk_ids || !logits) return fail(hipErrorInvalidValue, "%s: null tensor pointer", what);
  TopkGradArgs a{dlogits, dweights, topk_ids, logits, row_stride, tokens, experts, topk, scoring == FLYGEMM_SCORE_SIGMOID,
                 renormalize != 0, packs_fit(logits, row_stride, experts, dtype), packs_fit(dlogits, experts, experts, dtype),
                 scale};
  const bool many = several_rows(tokens, experts, topk);
  const long per_wg = (long)kWaves * (many ? choice_rows(row_pack(experts)) : 1);
  const dim3 grid = grid_of((tokens + per_wg - 1) / per_wg);
  by_row(dtype, experts, [&](auto t, auto v) {
    typedef decltype(t) T;
    constexpr int V = decltype(v)::value;
    auto go = [&](auto fn) { hipLaunchKernelGGL(fn, grid, dim3(kThreads), 0, (hipStream_t)stream, a); };
    if (many) go(moe_topk_grad_kernel<T, V, choice_rows(V)>);
    else go(moe_topk_grad_kernel<T, V, 1>);
  });
  return launched(what);
}

int64_t flygemm_moe_balance_scratch(int32_t tokens, int32_t experts, int32_t sequences) {
  if (tokens < 0 || tokens > kMaxTokens || experts < 1 || experts > kMaxExperts || sequences < 1) return -1;
  const int chunk = balance_chunk(tokens);
  const int64_t slots = ((int64_t)tokens + chunk - 1) / chunk + sequences, B = sequences > 1 ? sequences : 0;
  return 2 * slots * 64 * row_pack(experts) * 4 + round16(slots * 4) + round16(B * 8) + round16(B * experts * 4) + round16(B * 4);
}

int flygemm_moe_balance(float* loss, int32_t* counts, float* aux, void* scratch, const void* logits, int64_t row_stride,
                        const void* topk_ids, const uint8_t* token_mask, const int32_t* cu_seqlens, int32_t tokens,
                        int32_t experts, int32_t topk, int32_t sequences, int32_t dtype, int32_t scoring,
                        int32_t ids_64bit, void* stream) {
  const char* what = "moe_balance";
  int rc = check_router(what, row_stride, tokens, experts, dtype, scoring);
  if (rc) return rc;
  if (topk < 1) return fail(hipErrorInvalidValue, "%s: topk=%d", what, topk);
  if (sequences < 1 || (!cu_seqlens && sequences != 1))
    return fail(hipErrorInvalidValue, "%s: sequences=%d", what, sequences);
  if (tokens < 1) return fail(hipErrorInvalidValue, "%s: no tokens", what);
  const int chunk = balance_chunk(tokens);
  // a thread's place among a chunk's ids goes up to a step behind the last
  if ((int64_t)chunk * topk > 0x7fffffffL - kPartThreads) return fail(hipErrorInvalidValue, "%s: topk=%d too large", what, topk);
  if (!loss || !counts || !aux || !scratch || !logits || !topk_ids)
    return fail(hipErrorInvalidValue, "%s: null tensor pointer", what);
  if ((uintptr_t)scratch & 15) return fail(hipErrorInvalidValue, "%s: scratch needs 16-byte alignment", what);
  const int64_t chunks = ((int64_t)tokens + chunk - 1) / chunk, slots = chunks + sequences, E = experts;
  char* s = (char*)scratch;
  auto take = [&](int64_t bytes) {
    char* at = s;
    s += round16(bytes);
    return at;
  };
  BalArgs a{};
  a.loss = loss, a.counts = counts, a.aux = aux;
  a.psum = (float*)take(slots * 64 * row_pack(experts) * 4);
  a.pcnt = (int32_t*)take(slots * 64 * row_pack(experts) * 4);
  a.pn = (int32_t*)take(slots * 4);
  if (sequences > 1) {
    a.seq_loss = (double*)take((int64_t)sequences * 8);
    a.seq_cnt = (int32_t*)take((int64_t)sequences * E * 4);
    a.seq_n = (int32_t*)take((int64_t)sequences * 4);
  }
  a.x = logits, a.ids = topk_ids, a.mask = token_mask, a.cu = cu_seqlens, a.stride = row_stride;
  a.T = tokens, a.E = experts, a.k = topk, a.B = sequences, a.chunk = chunk, a.ids64 = ids_64bit != 0;
  a.sigmoid = scoring == FLYGEMM_SCORE_SIGMOID, a.vec = packs_fit(logits, row_stride, experts, dtype);
  hipStream_t st = (hipStream_t)stream;
  by_row(dtype, experts, [&](auto t, auto v) {
    hipLaunchKernelGGL((moe_balance_part_kernel<decltype(t), decltype(v)::value>), dim3((unsigned)chunks),
                       dim3(kPartThreads), 0, st, a);
  });
  if ((rc = launched(what))) return rc;
  by_row(FLYGEMM_QIN_F32, experts, [&](auto, auto v) {
    hipLaunchKernelGGL((moe_balance_sum_kernel<decltype(v)::value>), grid_of(sequences), dim3(kSumThreads), 0, st, a);
  });
  if ((rc = launched(what))) return rc;
  if (sequences > 1) {
    hipLaunchKernelGGL(moe_balance_finish_kernel, dim3(1), dim3(kThreads), 0, st, a);
    rc = launched(what);
  }
  return rc;
}

int flygemm_moe_balance_grad(void* dlogits, const float* dloss, const float* aux, const void* logits, int64_t row_stride,
                             const uint8_t* token_mask, const int32_t* cu_seqlens, int32_t tokens, int32_t experts,
                             int32_t sequences, int32_t dtype, int32_t scoring, void* stream) {
  const char* what = "moe_balance_grad";
  const int rc = check_router(what, row_stride, tokens, experts, dtype, scoring);
  if (rc) return rc;
  if (sequences < 1 || (!cu_seqlens && sequences != 1))
    return fail(hipErrorInvalidValue, "%s: sequences=%d", what, sequences);
  if (tokens == 0) return 0;
  if (!dlogits || !dloss || !aux || !logits) return fail(hipErrorInvalidValue, "%s: null tensor pointer", what);
  BalGradArgs a{dlogits, dloss, aux, logits, token_mask, cu_seqlens, row_stride, tokens, experts, sequences,
                scoring == FLYGEMM_SCORE_SIGMOID, packs_fit(logits, row_stride, experts, dtype),
                packs_fit(dlogits, experts, experts, dtype)};
  const dim3 grid = grid_of(((int64_t)tokens + kWaves * kGradRows - 1) / (kWaves * kGradRows));
  by_row(dtype, experts, [&](auto t, auto v) {
    hipLaunchKernelGGL((moe_balance_grad_kernel<decltype(t), decltype(v)::value>), grid, dim3(kThreads), 0,
                       (hipStream_t)stream, a);
  });
  return launched(what);
}

}  // extern "C"
