// Verification of drafted tokens against the target's probabilities, from given random numbers.
//
// p = softmax(logits / T); T <= 0 stands for the arg-max (lowest index of equal ones).
//  * a tree of drafts: every node's own token is the first i with cdf(i) > u[depth] (what this operator draws with that number from the one row), and
//    the walk goes from node 0 to the first child that carries the token, until there is none;
//  * a chain of drafts drawn from q: draft x_i is kept while u_i q_i(x_i) < p_i(x_i); the token after it comes from max(p - q, 0) of the
//    first draft that is not kept, or from p behind the last one.
// A draw is an index, and among 150,000 tokens running sums in 32 bits put one draw in forty (flat probabilities) to three hundred
// beside the token that the probabilities give.  Weights, sums and comparisons are therefore 64-bit.  Sums are taken in a fixed order: the same inputs give the same tokens.
//
// An exponential is 2^(k / 256) 2^n p(f): the nearest 256th of the exponent from a table, a polynomial of degree three for the rest (table-driven
// exponentials: P. T. P. Tang, ACM TOMS 15, 1989), within 2e-14 relatively where (maximum - x) / T is at most 40 and 1e-13 up to
// 690, since the argument itself is rounded.  The 64-bit pipe is what bounds the sums: eight operations a logit;
// 128 rows of 151936 logits take 28 us, 12 us of them reading.  (Degree five and 16 table entries 2 us more, the library's exponential 36.)
//
// 1. row_stats: the logits are read once; a warp a (part of the vocabulary, row) leaves the part's maximum, its first place and the sum of
//    exp((x - maximum) / T).
// 2. tree_pick: a draw needs its part of its row once more; the last CTA of a sequence to arrive walks the tree.
//    draft_rest: draws from max(p - q, 0) need the whole row at which the chain ends; the last CTA of a sequence draws.
// The arrivals are counted in workspace that the first kernel clears.
#include <algorithm>

#include "common.cuh"

namespace {

constexpr int kStep = 512;        // logits of a warp at a time; a part is a multiple of it
constexpr int kParts = 256;       // parts of a row at most
constexpr int kNT = 256;          // threads of a CTA
constexpr int kE = 16, kPE = 8;   // logits of a thread at a time, for the sums of the parts and for a draw
constexpr int kNodes = 64;

struct PartStat { double sum; float mx; int arg; };

struct VerifyArgs {
  const float* logits; int64_t lds, ldr;      // sequence / node stride
  const int64_t* tokens;                      // [R, C]
  const int64_t* anc;                         // tree: [R, C]
  const int* lengths;                         // chain: [R] tokens of the chain, the fed one included
  const float* q; int64_t ldqs, ldqr;         // chain: [R, C - 1, V]
  const float* temperature; const float* u; const float* u_draw;
  PartStat* stats;                            // [R * C, P]
  int* picks;                                 // tree: [R * C]
  double2* rest;                              // chain: [R, P] sums of max(p - q, 0) and of p
  unsigned* arrived;                          // [R]
  int* path; int* steps; int64_t* next;
  int64_t V, per;
  int R, C, P;
};

__device__ __forceinline__ bool row_used(const VerifyArgs& a, int r, int j) {
  return a.anc ? a.anc[(int64_t)r * a.C + j] != 0 : j < min(a.lengths[r], a.C);
}
// 2^(k / 16) and 2^(k / 256)
__device__ const double kRoots[2][16] = {
    {1.0, 1.0442737824274138, 1.0905077326652577, 1.1387886347566916, 1.189207115002721, 1.241857812073484, 1.2968395546510096, 1.3542555469368927,
     1.4142135623730951, 1.4768261459394993, 1.5422108254079407, 1.6104903319492543, 1.681792830507429, 1.7562521603732995, 1.8340080864093424, 1.9152065613971474},
    {1.0, 1.0027112750502025, 1.0054299011128027, 1.0081558981184175, 1.0108892860517005, 1.0136300849514894, 1.016378314910953, 1.019133996077738,
     1.0218971486541166, 1.0246677928971357, 1.0274459491187637, 1.030231637686041, 1.0330248790212284, 1.0358256936019572, 1.0386341019613787, 1.041450124688316}};
constexpr double kMagic = 6755399441055744.0;               // 1.5 2^52: adding it leaves the nearest whole number in the low word
__device__ __forceinline__ double exp_rest(double f) {      // 2^(f / 256), |f| <= 1/2
  return fma(fma(fma(3.308302983711395e-09, f, 3.6655661567589336e-06), f, 0.0027076061740622767), f, 0.9999999999999825);
}
// exp((x - mx) / T) for x <= mx with s256 = 256 log2(e) / T; 1 at the maximum whatever it is, 0 for NaN
__device__ __forceinline__ double weight(float x, float mx, double s256) {
  const double d = (double)x - (double)mx, m = fma(d, s256, kMagic), f = fma(d, s256, -(m - kMagic));
  const int n = __double2loint(m);
  const double p = exp_rest(f) * (kRoots[0][n >> 4 & 15] * kRoots[1][n & 15]);
  // (a comparison with NaN is false; less than 2^-1000 is nothing)
  return x == mx ? 1.0 : (d * s256 > -256000.0 ? __hiloint2double(__double2hiint(p) + ((n >> 8) << 20), __double2loint(p)) : 0.0);
}
// The same added to a sum, for finite mx and a floor about 2^-995 below it, where a logit below the floor, -inf or NaN counts as the floor,
// which is next to nothing: the table's root with its exponent moved and the sum make one multiplication and addition.
__device__ __forceinline__ void add_weight(double& sum, float x, float floor, double mx, double s256, const double* roots) {
  const double d = (double)fmaxf(x, floor) - mx, m = fma(d, s256, kMagic), f = fma(d, s256, -(m - kMagic));
  const int n = __double2loint(m), k = n & 255;
  const double r = roots[k];
  sum = fma(exp_rest(f), __hiloint2double(__double2hiint(r) + (n - k) * 4096, __double2loint(r)), sum);
}
__device__ __forceinline__ double scale256(float T) { return 369.3299304675746 / (double)T; }
__device__ __forceinline__ double warp_sum_d(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// inclusive prefix sums over the CTA; `red` holds a double a warp
template <int NT>
__device__ __forceinline__ double block_scan_d(double v, double* red, double* total) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double x = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += x;
  }
  __syncthreads();
  if (lane == 31) red[w] = v;
  __syncthreads();
  double before = 0.0, all = 0.0;
#pragma unroll 1
  for (int i = 0; i < NT / 32; ++i) {
    if (i < w) before += red[i];
    all += red[i];
  }
  *total = all;
  return before + v;
}

__device__ __forceinline__ void load_logits(const float* row, int64_t at, int64_t end, bool vec, float* x) {
#pragma unroll
  for (int i = 0; i < kPE / 4; ++i) {
    const int64_t c = at + 4 * i;
    if (vec && c + 4 <= end) {
      const float4 v = *reinterpret_cast<const float4*>(row + c);
      x[4 * i] = v.x; x[4 * i + 1] = v.y; x[4 * i + 2] = v.z; x[4 * i + 3] = v.w;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) x[4 * i + e] = c + e < end ? row[c + e] : __int_as_float(0x7fffffff);      // NaN: no weight
    }
  }
}

// The maximum of a step is the warp's before its first weight, so that a sum is scaled anew for a whole warp or not at all.  The next step's
// logits are on their way meanwhile.  (A maximum of its own for every thread, and half the instructions go into scaling: a pass over 128 rows
// 38.5 us instead of 37.2, over 64 rows of drafts 34.6 instead of 32.7.)
__global__ void __launch_bounds__(kNT, 4) row_stats_kernel(const VerifyArgs a) {
  __shared__ double roots[256];
  griddep_launch();
  griddep_wait();
  const int lane = threadIdx.x & 31, p = blockIdx.x * (kNT / 32) + (threadIdx.x >> 5), r = blockIdx.y / a.C, j = blockIdx.y % a.C;
  roots[threadIdx.x] = kRoots[0][threadIdx.x / 16] * kRoots[1][threadIdx.x % 16];
  if (p == 0 && j == 0 && lane == 0) a.arrived[r] = 0;
  __syncthreads();
  if (p >= a.P || !row_used(a, r, j)) return;
  const float* row = a.logits + r * a.lds + j * a.ldr;
  const bool vec = ((uintptr_t)row & 15) == 0;
  const float T = a.temperature[r];
  const double s256 = scale256(T);
  const int64_t b = p * a.per, e = min(a.V, b + a.per);
  auto place = [&](int64_t c, int i) { return c + (i / 4 * 32 + lane) * 4 + i % 4; };      // groups of four, lane by lane
  auto load = [&](int64_t c, float* x) {
    if (vec && c + kStep <= e) {
#pragma unroll
      for (int i = 0; i < kE / 4; ++i) {
        const uint4 v = ld_stream(row + c + (i * 32 + lane) * 4);
        x[4 * i] = __uint_as_float(v.x); x[4 * i + 1] = __uint_as_float(v.y); x[4 * i + 2] = __uint_as_float(v.z); x[4 * i + 3] = __uint_as_float(v.w);
      }
    } else {
#pragma unroll
      for (int i = 0; i < kE; ++i) x[i] = place(c, i) < e ? row[place(c, i)] : __int_as_float(0x7fffffff);      // NaN: no logit
    }
  };
  float mx = -INFINITY, next[kE];
  int arg = 0x7fffffff;                                     // the arg-max is wanted where nothing is drawn
  double sum = 0.0;
  load(b, next);
#pragma unroll 1
  for (int64_t c = b; c < e; c += kStep) {
    float x[kE];
#pragma unroll
    for (int i = 0; i < kE; ++i) x[i] = next[i];
    if (c + kStep < e) load(c + kStep, next);
    float cm = x[0];
#pragma unroll
    for (int i = 1; i < kE; ++i) cm = fmaxf(cm, x[i]);
    if (!(T > 0.f)) {
      if (cm > mx || arg == 0x7fffffff) {                   // (false for NaN alone)
#pragma unroll
        for (int i = kE - 1; i >= 0; --i)
          if (x[i] == cm) arg = (int)place(c, i);
        mx = fmaxf(mx, cm);
      }
      continue;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) cm = fmaxf(cm, __shfl_xor_sync(0xffffffffu, cm, o));
    if (cm > mx) {
      if (sum > 0.0) sum *= weight(mx, cm, s256);
      mx = cm;
    }
    const float floor = fmaxf(mx - 690.f * T, -3.4e38f);
    if (fabsf(mx) < INFINITY && 690.f * T >= fabsf(mx) * 0x1p-10f && T < 1e30f) {
      const double top = (double)mx;
      double part[2] = {0.0, 0.0};
#pragma unroll
      for (int i = 0; i < kE; ++i) add_weight(part[i & 1], x[i], floor, top, s256, roots);
      sum += part[0] + part[1];
    } else {                                                // infinite, so cold that the floor would be rounded onto the maximum, or so hot that it has weight
#pragma unroll 1
      for (int i = 0; i < kE; ++i)
        if (place(c, i) < e) sum += weight(row[place(c, i)], mx, s256);
    }
  }
  float all = mx;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) all = fmaxf(all, __shfl_xor_sync(0xffffffffu, all, o));
  arg = __reduce_min_sync(0xffffffffu, mx == all ? arg : 0x7fffffff);
  sum = warp_sum_d(sum);
  if (lane == 0) a.stats[(int64_t)blockIdx.y * a.P + p] = PartStat{sum, all, arg};
}

// maximum, its first place and the whole sum of a row, from its parts; every lane of the warp gets them
__device__ __forceinline__ void row_whole(const PartStat* st, int P, float T, float& mx, int& arg, double& total) {
  const int lane = threadIdx.x & 31;
  const double s256 = scale256(T);
  mx = -INFINITY;
  arg = 0x7fffffff;
#pragma unroll 1
  for (int p = lane; p < P; p += 32)
    if (st[p].mx > mx || (st[p].mx == mx && st[p].arg < arg)) { mx = st[p].mx; arg = st[p].arg; }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float om = __shfl_xor_sync(0xffffffffu, mx, o);
    const int oa = __shfl_xor_sync(0xffffffffu, arg, o);
    if (om > mx || (om == mx && oa < arg)) { mx = om; arg = oa; }
  }
  total = 0.0;
  if (T > 0.f)
#pragma unroll 1
    for (int p = lane; p < P; p += 32) total += st[p].sum * weight(st[p].mx, mx, s256);
  total = warp_sum_d(total);
}

// The part that holds the target, given each part's own weight and the sum up to it (a thread a part): the first one whose sum exceeds
// it, else the last one with any weight; what comes before it goes to `before`.
__device__ __forceinline__ int pick_part(double mine, double incl, double target, double* before) {
  __shared__ int part;
  __shared__ double before_s;
  const int p = threadIdx.x;
  if (p == 0) part = 0;
  __syncthreads();
  if (mine > 0.0) atomicMax(&part, p);
  __syncthreads();
  if (mine > 0.0 && incl > target) atomicMin(&part, p);
  __syncthreads();
  if (p == part) before_s = incl - mine;
  __syncthreads();
  *before = before_s;
  return part;
}

// First place of [b, e) where the running sum of the weights, begun at `before`, exceeds `target`; the last place with any weight where
// none does.  w.all(at, x): the weights of kE consecutive places; w.one(at): of one.
template <typename W>
__device__ __forceinline__ int64_t pick_range(const W& w, int64_t b, int64_t e, double before, double target) {
  __shared__ double red[kNT / 32];
  __shared__ int who;
  __shared__ long long found, last;
  const int lane = threadIdx.x & 31;
  if (threadIdx.x == 0) { who = kNT; found = -1; last = -1; }
  __syncthreads();
#pragma unroll 1
  for (int64_t c = b; c < e; c += kNT * kPE) {
    double x[kPE], s = 0.0, total;
    const int64_t at = c + threadIdx.x * kPE;
    w.all(at, e, x);
    int end = -1;
#pragma unroll
    for (int i = 0; i < kPE; ++i) {
      s += x[i];
      if (x[i] > 0.0) end = i;
    }
    if (end >= 0) atomicMax(&last, (long long)(at + end));
    const double incl = before + block_scan_d<kNT>(s, red, &total);
    if (s > 0.0 && incl > target) atomicMin(&who, (int)threadIdx.x);
    __syncthreads();
    if (who / 32 == (int)threadIdx.x / 32) {                // the warp of the thread whose places reach the target: a lane a place
      const double from = __shfl_sync(0xffffffffu, incl - s, who & 31);
      const int64_t place = c + who * kPE + lane;
      const double mine = lane < kPE && place < e ? w.one(place) : 0.0;
      double run = mine;
#pragma unroll
      for (int o = 1; o < kPE; o <<= 1) {
        const double y = __shfl_up_sync(0xffffffffu, run, o);
        if (lane >= o) run += y;
      }
      const unsigned some = __ballot_sync(0xffffffffu, mine > 0.0), over = __ballot_sync(0xffffffffu, mine > 0.0 && from + run > target);
      // roundings aside, the target is reached before the last place with any weight
      if (lane == 0) found = c + who * kPE + (over ? __ffs(over) - 1 : 31 - __clz(some));
    }
    __syncthreads();
    if (found >= 0) return found;
    before += total;
  }
  return last;
}

struct RowWeights {                  // exp((logit - mx) / T)
  const float* row;
  bool vec;
  float mx; double s256;
  __device__ __forceinline__ void all(int64_t at, int64_t end, double* x) const {
    float f[kPE];
    load_logits(row, at, end, vec, f);
#pragma unroll
    for (int i = 0; i < kPE; ++i) x[i] = weight(f[i], mx, s256);
  }
  __device__ __forceinline__ double one(int64_t at) const { return weight(row[at], mx, s256); }
};

// Whether this CTA is the last of `all` to arrive for sequence r; what the others have written before is visible to it then.
__device__ __forceinline__ bool last_of(const VerifyArgs& a, int r, unsigned all) {
  __shared__ bool last;
  __syncthreads();
  if (threadIdx.x == 0) {
    __threadfence();
    last = atomicAdd(a.arrived + r, 1u) == all - 1;
    __threadfence();
  }
  __syncthreads();
  return last;
}

__device__ __forceinline__ void tree_walk(const VerifyArgs& a, int r);

// A node's own token (thread 0's).
__device__ __forceinline__ int node_token(const VerifyArgs& a, int r, int j) {
  __shared__ double red[kNT / 32];
  const PartStat* st = a.stats + ((int64_t)r * a.C + j) * a.P;
  const float T = a.temperature[r];
  float mx;
  int arg;
  double total, whole, before;
  row_whole(st, a.P, T, mx, arg, total);
  if (!(T > 0.f) || !(total > 0.0)) return arg < a.V ? arg : 0;
  const double s256 = scale256(T);
  const int depth = __popcll((uint64_t)a.anc[(int64_t)r * a.C + j] & ~(~0ull << j)), p = threadIdx.x;
  const double mine = p < a.P ? st[p].sum * weight(st[p].mx, mx, s256) : 0.0, incl = block_scan_d<kNT>(mine, red, &whole);
  const double target = (double)a.u[(int64_t)r * a.C + depth] * whole;
  const int part = pick_part(mine, incl, target, &before);
  const float* row = a.logits + r * a.lds + j * a.ldr;
  const int64_t b = part * a.per, pick = pick_range(RowWeights{row, ((uintptr_t)row & 15) == 0, mx, s256}, b, min(a.V, b + a.per), before, target);
  return pick < 0 ? 0 : (int)pick;                          // (a part that is picked has weight: never)
}

__global__ void __launch_bounds__(kNT) tree_pick_kernel(const VerifyArgs a) {
  griddep_launch();
  griddep_wait();
  const int r = blockIdx.x / a.C, j = blockIdx.x % a.C;
  if (row_used(a, r, j)) {
    const int token = node_token(a, r, j);
    if (threadIdx.x == 0) a.picks[blockIdx.x] = token;
  }
  if (last_of(a, r, a.C)) tree_walk(a, r);
}

// Node 0, then the first child that carries the token drawn at the node reached; children come after their parents.
__device__ __forceinline__ void tree_walk(const VerifyArgs& a, int r) {
  __shared__ int parent[kNodes];
  __shared__ int64_t token[kNodes], pick[kNodes];
  const int j = threadIdx.x;
  if (j < a.C) {
    const uint64_t on = (uint64_t)a.anc[(int64_t)r * a.C + j], up = on & ~(~0ull << j);
    parent[j] = on != 0 && up != 0 ? 63 - __clzll((long long)up) : -1;
    token[j] = a.tokens[(int64_t)r * a.C + j];
    pick[j] = on != 0 ? __ldcg(a.picks + (int64_t)r * a.C + j) : -1;
    a.path[(int64_t)r * a.C + j] = -1;
  }
  __syncthreads();
  if (j != 0) return;
  int n = 0, cur = 0;
  if (pick[0] >= 0) {
    a.path[(int64_t)r * a.C] = 0;
    n = 1;
#pragma unroll 1
    for (int i = 1; i < a.C; ++i)
      if (parent[i] == cur && token[i] == pick[cur]) {
        a.path[(int64_t)r * a.C + n++] = i;
        cur = i;
      }
  }
  a.steps[r] = n;
  a.next[r] = n ? pick[cur] : -1;
}

// How many drafts of the chain are kept, and of the row at which they end its maximum, arg-max and whole sum.
struct ChainEnd { int at; float mx; int arg; double total; };
template <int NT>
__device__ __forceinline__ ChainEnd chain_end(const VerifyArgs& a, int r, int n) {
  __shared__ float mx_s[kNodes];
  __shared__ int arg_s[kNodes], ok_s[kNodes];
  __shared__ double total_s[kNodes];
  const float T = a.temperature[r];
#pragma unroll 1
  for (int i = threadIdx.x >> 5; i < n; i += NT / 32) {
    float mx;
    int arg;
    double total;
    row_whole(a.stats + ((int64_t)r * a.C + i) * a.P, a.P, T, mx, arg, total);
    if ((threadIdx.x & 31) == 0) { mx_s[i] = mx; arg_s[i] = arg; total_s[i] = total; }
  }
  __syncthreads();
  const int i = threadIdx.x;
  if (i < n) {
    bool ok = false;
    if (i < n - 1) {
      const int64_t x = a.tokens[(int64_t)r * a.C + i + 1];
      if (x >= 0 && x < a.V) {
        const double u = a.u[(int64_t)r * a.C + i + 1], qx = a.q[r * a.ldqs + i * a.ldqr + x];
        const double px = T > 0.f ? weight(a.logits[r * a.lds + i * a.ldr + x], mx_s[i], scale256(T)) / total_s[i] : (x == arg_s[i] ? 1.0 : 0.0);
        ok = u * qx < px;
      }
    }
    ok_s[i] = ok;
  }
  __syncthreads();
  int at = 0;
#pragma unroll 1
  while (at < n - 1 && ok_s[at]) ++at;
  return ChainEnd{at, mx_s[at], arg_s[at], total_s[at]};
}

struct RestWeights {                 // p and max(p - q, 0) of the row at which a chain ends
  const float* row; const float* q;
  bool vec, qvec, rest;              // rest: all and one give max(p - q, 0), else p
  float mx; double s256, inv_total;
  __device__ __forceinline__ void both(int64_t at, int64_t end, double* left, double* p) const {
    float f[kPE], g[kPE];
    load_logits(row, at, end, vec, f);
#pragma unroll
    for (int i = 0; i < kPE; ++i) g[i] = 0.f;
    if (q) load_logits(q, at, end, qvec, g);
#pragma unroll
    for (int i = 0; i < kPE; ++i) {
      p[i] = __dmul_rn(weight(f[i], mx, s256), inv_total);      // not fused with the difference: one() has the same values
      left[i] = fmax(p[i] - (double)g[i], 0.0);             // (places behind the end: 0 - NaN, and fmax gives 0)
    }
  }
  __device__ __forceinline__ void all(int64_t at, int64_t end, double* x) const {
    double p[kPE];
    both(at, end, x, p);
    if (!rest) {
#pragma unroll
      for (int i = 0; i < kPE; ++i) x[i] = p[i];
    }
  }
  __device__ __forceinline__ double one(int64_t at) const {
    const double p = __dmul_rn(weight(row[at], mx, s256), inv_total);
    return rest && q ? fmax(p - (double)q[at], 0.0) : p;
  }
};
__device__ __forceinline__ RestWeights rest_weights(const VerifyArgs& a, int r, int n, const ChainEnd& c) {
  RestWeights w;
  w.rest = true;
  w.row = a.logits + r * a.lds + c.at * a.ldr;
  w.q = c.at < n - 1 ? a.q + r * a.ldqs + c.at * a.ldqr : nullptr;
  w.vec = ((uintptr_t)w.row & 15) == 0;
  w.qvec = ((uintptr_t)w.q & 15) == 0;
  w.mx = c.mx;
  w.s256 = scale256(a.temperature[r]);
  w.inv_total = 1.0 / c.total;
  return w;
}

__global__ void __launch_bounds__(kNT) draft_rest_kernel(const VerifyArgs a) {
  __shared__ double red[2][kNT / 32];
  griddep_launch();
  griddep_wait();
  const int p = blockIdx.x, r = blockIdx.y, n = min(a.lengths[r], a.C), tid = threadIdx.x;
  if (n < 1) {
    if (p == 0 && tid == 0) { a.steps[r] = 0; a.next[r] = -1; }
    return;
  }
  const ChainEnd c = chain_end<kNT>(a, r, n);
  if (p == 0 && tid == 0) a.steps[r] = c.at + 1;
  if (!(a.temperature[r] > 0.f) || !(c.total > 0.0)) {
    if (p == 0 && tid == 0) a.next[r] = c.arg < a.V ? c.arg : 0;
    return;
  }
  RestWeights w = rest_weights(a, r, n, c);
  const int64_t b = p * a.per, e = min(a.V, b + a.per);
  double rest = 0.0, all = 0.0;
#pragma unroll 1
  for (int64_t at = b + tid * kPE; at < e; at += kNT * kPE) {
    double x[kPE], y[kPE];
    w.both(at, e, x, y);
#pragma unroll
    for (int i = 0; i < kPE; ++i) { rest += x[i]; all += y[i]; }
  }
  rest = warp_sum_d(rest);
  all = warp_sum_d(all);
  if ((tid & 31) == 0) { red[0][tid >> 5] = rest; red[1][tid >> 5] = all; }
  __syncthreads();
  if (tid == 0) {
    rest = all = 0.0;
    for (int i = 0; i < kNT / 32; ++i) { rest += red[0][i]; all += red[1][i]; }
    a.rest[(int64_t)r * a.P + p] = make_double2(rest, all);
  }
  if (!last_of(a, r, a.P)) return;
  const double2 mine2 = tid < a.P ? __ldcg(a.rest + (int64_t)r * a.P + tid) : make_double2(0.0, 0.0);
  double whole, before;
  double incl = block_scan_d<kNT>(mine2.x, red[0], &whole), mine = mine2.x;
  w.rest = whole > 0.0;                           // nothing left over: drafts drawn from q are always kept then, up to rounding
  if (!w.rest) {
    mine = mine2.y;
    incl = block_scan_d<kNT>(mine, red[0], &whole);
  }
  const double target = (double)a.u_draw[r] * whole;
  const int part = pick_part(mine, incl, target, &before);
  const int64_t b1 = part * a.per, pick = pick_range(w, b1, min(a.V, b1 + a.per), before, target);
  if (tid == 0) a.next[r] = pick < 0 ? 0 : pick;
}

// Logits of a part: two steps of a warp where there are few rows, four where there are enough warps without; more where a row would have
// more than kParts.
int parts_of(int64_t rows, int64_t V, int64_t* per) {
  const int64_t least = (V + (int64_t)kParts * kStep - 1) / ((int64_t)kParts * kStep);
  *per = std::max<int64_t>(least, rows * V < 148ll * 32 * 2048 ? 2 : 4) * kStep;
  return (int)((V + *per - 1) / *per);
}

}  // namespace

// bytes of workspace of a call
CB_EXPORT int64_t cb_verify_scratch(int64_t R, int64_t C, int64_t V) {
  int64_t per;
  const int64_t P = parts_of(R * C, V, &per);
  return R * C * P * (int64_t)sizeof(PartStat) + R * P * (int64_t)sizeof(double2) + R * C * (int64_t)sizeof(int) + R * (int64_t)sizeof(unsigned);
}

CB_EXPORT int cb_verify_tree(const void* logits, int64_t lds, int64_t ldr, const void* tokens, const void* anc, const void* temperature,
                             const void* u, void* path, void* steps, void* next, void* scratch, int64_t R, int64_t C, int64_t V, void* stream) {
  if (!logits || !tokens || !anc || !temperature || !u || !path || !steps || !next || !scratch) return CB_ERR_ARG;
  if (R < 1 || C < 1 || C > kNodes || V < 1 || V > 0x7fffffff || R * C > 65535) return CB_ERR_SHAPE;
  VerifyArgs a = {};
  a.logits = (const float*)logits; a.lds = lds; a.ldr = ldr; a.tokens = (const int64_t*)tokens; a.anc = (const int64_t*)anc;
  a.temperature = (const float*)temperature; a.u = (const float*)u; a.path = (int*)path; a.steps = (int*)steps; a.next = (int64_t*)next;
  a.V = V; a.R = (int)R; a.C = (int)C; a.P = parts_of(R * C, V, &a.per);
  a.stats = (PartStat*)scratch;
  a.picks = (int*)(a.stats + R * C * a.P);
  a.arrived = (unsigned*)(a.picks + R * C);
  cudaStream_t st = (cudaStream_t)stream;
  cudaError_t e = cb_launch(row_stats_kernel, dim3((unsigned)((a.P + kNT / 32 - 1) / (kNT / 32)), (unsigned)(R * C)), dim3(kNT), 0, st, a);
  if (e == cudaSuccess) e = cb_launch_second(tree_pick_kernel, dim3((unsigned)(R * C)), dim3(kNT), 0, st, a);
  return (int)e;
}

CB_EXPORT int cb_verify_drafts(const void* logits, int64_t lds, int64_t ldr, const void* tokens, const void* lengths, const void* q, int64_t ldqs,
                               int64_t ldqr, const void* temperature, const void* u, const void* u_draw, void* steps, void* next, void* scratch,
                               int64_t R, int64_t C, int64_t V, void* stream) {
  if (!logits || !tokens || !lengths || (!q && C > 1) || !temperature || !u || !u_draw || !steps || !next || !scratch) return CB_ERR_ARG;
  if (R < 1 || C < 1 || C > kNodes || V < 1 || V > 0x7fffffff || R * C > 65535) return CB_ERR_SHAPE;
  VerifyArgs a = {};
  a.logits = (const float*)logits; a.lds = lds; a.ldr = ldr; a.tokens = (const int64_t*)tokens; a.lengths = (const int*)lengths;
  a.q = (const float*)q; a.ldqs = ldqs; a.ldqr = ldqr; a.temperature = (const float*)temperature; a.u = (const float*)u;
  a.u_draw = (const float*)u_draw; a.steps = (int*)steps; a.next = (int64_t*)next;
  a.V = V; a.R = (int)R; a.C = (int)C; a.P = parts_of(R * C, V, &a.per);
  a.stats = (PartStat*)scratch;
  a.rest = (double2*)(a.stats + R * C * a.P);
  a.arrived = (unsigned*)(a.rest + R * a.P);
  cudaStream_t st = (cudaStream_t)stream;
  cudaError_t e = cb_launch(row_stats_kernel, dim3((unsigned)((a.P + kNT / 32 - 1) / (kNT / 32)), (unsigned)(R * C)), dim3(kNT), 0, st, a);
  if (e == cudaSuccess) e = cb_launch_second(draft_rest_kernel, dim3((unsigned)a.P, (unsigned)R), dim3(kNT), 0, st, a);
  return (int)e;
}
