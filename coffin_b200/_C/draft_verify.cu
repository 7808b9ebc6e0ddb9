// Verification of drafted tokens against the target's probabilities, from given random numbers.
//
// p = softmax(logits / T); T <= 0 stands for the arg-max (lowest index of equal ones).
//  * a tree of drafts: every node's own token is the first i with cdf(i) > u[depth] (what plain sampling draws with that number), and
//    the walk goes from node 0 to the first child that carries the token, until there is none;
//  * a chain of drafts drawn from q: draft x_i is kept while u_i q_i(x_i) < p_i(x_i); the token after it comes from max(p - q, 0) of the
//    first draft that is not kept, or from p behind the last one.
// A draw is an index, and among 150,000 tokens a running sum in 32 bits puts one in about thirty draws beside the token that the
// probabilities give.  Weights, sums and comparisons are therefore 64-bit.  Sums are taken in a fixed order: the same inputs give the same tokens.
//
// 1. row_stats: the logits are read once; a CTA a (part of the vocabulary, row) leaves the part's maximum, its first place and the sum of
//    exp((x - maximum) / T).
// 2. tree_pick / draft_rest: a draw needs its part of the row once more (draws from max(p - q, 0) the whole row of the node they end at).
// 3. tree_walk / draft_pick: the path and the token after it.
#include "common.cuh"

namespace {

constexpr int kPart = 4096;       // logits of a part at least (a multiple of it, so that a row has at most kParts)
constexpr int kParts = 256;
constexpr int kNT = 256, kE = 16; // threads of a CTA, consecutive logits of a thread
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
  int* path; int* steps; int64_t* next;
  int64_t V, per;
  int R, C, P;
};

__device__ __forceinline__ bool row_used(const VerifyArgs& a, int r, int j) {
  return a.anc ? a.anc[(int64_t)r * a.C + j] != 0 : j < min(a.lengths[r], a.C);
}
// exp((x - mx) / T), 1 at the maximum whatever it is, 0 for NaN
__device__ __forceinline__ double weight(float x, float mx, double inv_t) {
  if (x == mx) return 1.0;
  const double w = exp(((double)x - (double)mx) * inv_t);
  return w >= 0.0 ? w : 0.0;
}
__device__ __forceinline__ double warp_sum_d(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// inclusive prefix sums over the CTA; `red` holds a double a warp
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
  for (int i = 0; i < kNT / 32; ++i) {
    if (i < w) before += red[i];
    all += red[i];
  }
  *total = all;
  return before + v;
}

__device__ __forceinline__ void load_logits(const float* row, int64_t at, int64_t end, bool vec, float* x) {
#pragma unroll
  for (int i = 0; i < kE / 4; ++i) {
    const int64_t c = at + 4 * i;
    if (vec && c + 4 <= end) {
      const float4 v = *reinterpret_cast<const float4*>(row + c);
      x[4 * i] = v.x; x[4 * i + 1] = v.y; x[4 * i + 2] = v.z; x[4 * i + 3] = v.w;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) x[4 * i + e] = c + e < end ? row[c + e] : -INFINITY;
    }
  }
}

__global__ void __launch_bounds__(kNT) row_stats_kernel(const VerifyArgs a) {
  __shared__ float mx_s[kNT / 32];
  __shared__ int arg_s[kNT / 32];
  __shared__ double sum_s[kNT / 32];
  griddep_launch();
  griddep_wait();
  const int p = blockIdx.x, r = blockIdx.y / a.C, j = blockIdx.y % a.C, lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  if (!row_used(a, r, j)) return;
  const float* row = a.logits + r * a.lds + j * a.ldr;
  const bool vec = ((uintptr_t)row & 15) == 0;
  const float T = a.temperature[r];
  const double inv_t = 1.0 / (double)T;
  const int64_t b = p * a.per, e = min(a.V, b + a.per);
  float mx = -INFINITY;
  int arg = 0x7fffffff;
  double sum = 0.0;
  for (int64_t c = b; c < e; c += kPart) {
    // lane-strided groups of four: the order of a sum is not the order of the row here
    float x[kE];
#pragma unroll
    for (int i = 0; i < kE / 4; ++i) {
      const int64_t at = c + (i * kNT + threadIdx.x) * 4;
      if (vec && at + 4 <= e) {
        const float4 v = *reinterpret_cast<const float4*>(row + at);
        x[4 * i] = v.x; x[4 * i + 1] = v.y; x[4 * i + 2] = v.z; x[4 * i + 3] = v.w;
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) x[4 * i + k] = at + k < e ? row[at + k] : -INFINITY;
      }
    }
    float cm = -INFINITY;
    int ca = 0x7fffffff;
#pragma unroll
    for (int i = 0; i < kE; ++i) {
      const int64_t at = c + (i / 4 * kNT + threadIdx.x) * 4 + i % 4;
      if (at < e && (x[i] > cm || ca == 0x7fffffff) && x[i] == x[i]) { cm = x[i]; ca = (int)at; }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const float om = __shfl_xor_sync(0xffffffffu, cm, o);
      const int oa = __shfl_xor_sync(0xffffffffu, ca, o);
      if (om > cm || (om == cm && oa < ca)) { cm = om; ca = oa; }
    }
    __syncthreads();
    if (lane == 0) { mx_s[w] = cm; arg_s[w] = ca; }
    __syncthreads();
    for (int i = 0; i < kNT / 32; ++i)
      if (mx_s[i] > cm || (mx_s[i] == cm && arg_s[i] < ca)) { cm = mx_s[i]; ca = arg_s[i]; }
    if (cm > mx || (cm == mx && ca < arg)) {
      if (T > 0.f && sum > 0.0) sum *= weight(mx, cm, inv_t);
      mx = cm;
      arg = ca;
    }
    if (T > 0.f) {
#pragma unroll
      for (int i = 0; i < kE; ++i)
        if (c + (i / 4 * kNT + threadIdx.x) * 4 + i % 4 < e) sum += weight(x[i], mx, inv_t);
    }
  }
  sum = warp_sum_d(sum);
  if (lane == 0) sum_s[w] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    double s = 0.0;
    for (int i = 0; i < kNT / 32; ++i) s += sum_s[i];
    a.stats[(int64_t)blockIdx.y * a.P + p] = PartStat{s, mx, arg};
  }
}

// maximum, its first place and the whole sum of a row, from its parts; every lane of the warp gets them
__device__ __forceinline__ void row_whole(const PartStat* st, int P, float T, float& mx, int& arg, double& total) {
  const int lane = threadIdx.x & 31;
  const double inv_t = 1.0 / (double)T;
  mx = -INFINITY;
  arg = 0x7fffffff;
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
    for (int p = lane; p < P; p += 32) total += st[p].sum * weight(st[p].mx, mx, inv_t);
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

// First place of [b, e) where the running sum of w(i), begun at `before`, exceeds `target`; the last place with any weight where none does.
template <typename W>
__device__ __forceinline__ int64_t pick_range(W w, int64_t b, int64_t e, double before, double target) {
  __shared__ double red[kNT / 32];
  __shared__ int who;
  __shared__ long long found, last;
  if (threadIdx.x == 0) { who = kNT; found = -1; last = -1; }
  __syncthreads();
  for (int64_t c = b; c < e; c += kPart) {
    double x[kE], s = 0.0, total;
    const int64_t at = c + threadIdx.x * kE;
    w(at, e, x);
    int64_t end = -1;
#pragma unroll
    for (int i = 0; i < kE; ++i) {
      s += x[i];
      if (x[i] > 0.0) end = at + i;
    }
    if (end >= 0) atomicMax(&last, (long long)end);
    const double incl = before + block_scan_d(s, red, &total);
    if (incl > target) atomicMin(&who, (int)threadIdx.x);
    __syncthreads();
    if (who == (int)threadIdx.x) {
      double run = incl - s;
      int64_t pick = end;                         // roundings aside, the sum is exceeded before the end
#pragma unroll
      for (int i = kE - 1; i >= 0; --i) {         // first place that exceeds the target: sums from the front
        double upto = run;
        for (int k = 0; k <= i; ++k) upto += x[k];
        if (upto > target && x[i] > 0.0) pick = at + i;
      }
      found = pick;
    }
    __syncthreads();
    if (found >= 0) return found;
    before += total;
  }
  return last;
}

// A node's own token.
__global__ void __launch_bounds__(kNT) tree_pick_kernel(const VerifyArgs a) {
  __shared__ double red[kNT / 32];
  double before;
  griddep_launch();
  griddep_wait();
  const int r = blockIdx.x / a.C, j = blockIdx.x % a.C;
  if (!row_used(a, r, j)) return;
  const PartStat* st = a.stats + (int64_t)blockIdx.x * a.P;
  const float T = a.temperature[r];
  float mx;
  int arg;
  double total;
  row_whole(st, a.P, T, mx, arg, total);
  if (!(T > 0.f) || !(total > 0.0)) {
    if (threadIdx.x == 0) a.picks[blockIdx.x] = arg < a.V ? arg : 0;
    return;
  }
  const double inv_t = 1.0 / (double)T;
  const int depth = __popcll((uint64_t)a.anc[(int64_t)r * a.C + j] & ~(~0ull << j));
  const int p = threadIdx.x;
  const double mine = p < a.P ? st[p].sum * weight(st[p].mx, mx, inv_t) : 0.0;
  double whole;
  const double incl = block_scan_d(mine, red, &whole);
  const double target = (double)a.u[(int64_t)r * a.C + depth] * whole;
  const int part = pick_part(mine, incl, target, &before);
  const float* row = a.logits + r * a.lds + j * a.ldr;
  const bool vec = ((uintptr_t)row & 15) == 0;
  const int64_t b = part * a.per, e = min(a.V, b + a.per);
  const int64_t pick = pick_range([&](int64_t at, int64_t end, double* x) {
    float f[kE];
    load_logits(row, at, end, vec, f);
#pragma unroll
    for (int i = 0; i < kE; ++i) x[i] = at + i < end ? weight(f[i], mx, inv_t) : 0.0;
  }, b, e, before, target);
  if (threadIdx.x == 0) a.picks[blockIdx.x] = pick < 0 ? arg : (int)pick;
}

// Node 0, then the first child that carries the token drawn at the node reached; children come after their parents.
__global__ void __launch_bounds__(kNodes) tree_walk_kernel(const VerifyArgs a) {
  __shared__ int parent[kNodes];
  __shared__ int64_t token[kNodes], pick[kNodes];
  griddep_launch();
  griddep_wait();
  const int r = blockIdx.x, j = threadIdx.x;
  if (j < a.C) {
    const uint64_t on = (uint64_t)a.anc[(int64_t)r * a.C + j], up = on & ~(~0ull << j);
    parent[j] = on != 0 && up != 0 ? 63 - __clzll((long long)up) : -1;
    token[j] = a.tokens[(int64_t)r * a.C + j];
    pick[j] = on != 0 ? a.picks[(int64_t)r * a.C + j] : -1;
    a.path[(int64_t)r * a.C + j] = -1;
  }
  __syncthreads();
  if (j != 0) return;
  int n = 0, cur = 0;
  if (pick[0] >= 0) {
    a.path[(int64_t)r * a.C] = 0;
    n = 1;
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
__device__ __forceinline__ ChainEnd chain_end(const VerifyArgs& a, int r, int n) {
  __shared__ float mx_s[kNodes];
  __shared__ int arg_s[kNodes], ok_s[kNodes];
  __shared__ double total_s[kNodes];
  const float T = a.temperature[r];
  for (int i = threadIdx.x >> 5; i < n; i += kNT / 32) {
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
        const double px = T > 0.f ? weight(a.logits[r * a.lds + i * a.ldr + x], mx_s[i], 1.0 / (double)T) / total_s[i] : (x == arg_s[i] ? 1.0 : 0.0);
        ok = u * qx < px;
      }
    }
    ok_s[i] = ok;
  }
  __syncthreads();
  int at = 0;
  while (at < n - 1 && ok_s[at]) ++at;
  return ChainEnd{at, mx_s[at], arg_s[at], total_s[at]};
}

struct RestWeights {                 // p and max(p - q, 0) of the row at which a chain ends
  const float* row; const float* q;
  bool vec, qvec;
  float mx; double inv_t, inv_total;
  __device__ __forceinline__ void operator()(int64_t at, int64_t end, double* rest, double* all) const {
    float f[kE], g[kE];
    load_logits(row, at, end, vec, f);
    if (q) load_logits(q, at, end, qvec, g);
#pragma unroll
    for (int i = 0; i < kE; ++i) {
      const double p = at + i < end ? weight(f[i], mx, inv_t) * inv_total : 0.0;
      all[i] = p;
      rest[i] = q && at + i < end ? fmax(p - (double)g[i], 0.0) : p;
    }
  }
};
__device__ __forceinline__ RestWeights rest_weights(const VerifyArgs& a, int r, int n, const ChainEnd& c) {
  RestWeights w;
  w.row = a.logits + r * a.lds + c.at * a.ldr;
  w.q = c.at < n - 1 ? a.q + r * a.ldqs + c.at * a.ldqr : nullptr;
  w.vec = ((uintptr_t)w.row & 15) == 0;
  w.qvec = ((uintptr_t)w.q & 15) == 0;
  w.mx = c.mx;
  w.inv_t = 1.0 / (double)a.temperature[r];
  w.inv_total = 1.0 / c.total;
  return w;
}

__global__ void __launch_bounds__(kNT) draft_rest_kernel(const VerifyArgs a) {
  __shared__ double red[2][kNT / 32];
  griddep_launch();
  griddep_wait();
  const int p = blockIdx.x, r = blockIdx.y, n = min(a.lengths[r], a.C);
  if (n < 1 || !(a.temperature[r] > 0.f)) return;
  const ChainEnd c = chain_end(a, r, n);
  const RestWeights w = rest_weights(a, r, n, c);
  const int64_t b = p * a.per, e = min(a.V, b + a.per);
  double rest = 0.0, all = 0.0;
  for (int64_t at = b + threadIdx.x * kE; at < e; at += kPart) {
    double x[kE], y[kE];
    w(at, e, x, y);
#pragma unroll
    for (int i = 0; i < kE; ++i) { rest += x[i]; all += y[i]; }
  }
  rest = warp_sum_d(rest);
  all = warp_sum_d(all);
  if ((threadIdx.x & 31) == 0) { red[0][threadIdx.x >> 5] = rest; red[1][threadIdx.x >> 5] = all; }
  __syncthreads();
  if (threadIdx.x == 0) {
    rest = all = 0.0;
    for (int i = 0; i < kNT / 32; ++i) { rest += red[0][i]; all += red[1][i]; }
    a.rest[(int64_t)r * a.P + p] = make_double2(rest, all);
  }
}

__global__ void __launch_bounds__(kNT) draft_pick_kernel(const VerifyArgs a) {
  __shared__ double red[kNT / 32];
  double before;
  griddep_launch();
  griddep_wait();
  const int r = blockIdx.x, n = min(a.lengths[r], a.C), p = threadIdx.x;
  if (n < 1) {
    if (p == 0) { a.steps[r] = 0; a.next[r] = -1; }
    return;
  }
  const ChainEnd c = chain_end(a, r, n);
  if (p == 0) a.steps[r] = c.at + 1;
  if (!(a.temperature[r] > 0.f) || !(c.total > 0.0)) {
    if (p == 0) a.next[r] = c.arg < a.V ? c.arg : 0;
    return;
  }
  const double2 mine2 = p < a.P ? a.rest[(int64_t)r * a.P + p] : make_double2(0.0, 0.0);
  double whole;
  double incl = block_scan_d(mine2.x, red, &whole);
  const bool rest = whole > 0.0;                  // nothing left over: drafts drawn from q are always kept then, up to rounding
  double mine = mine2.x;
  if (!rest) {
    mine = mine2.y;
    incl = block_scan_d(mine, red, &whole);
  }
  const double target = (double)a.u_draw[r] * whole;
  const int part = pick_part(mine, incl, target, &before);
  const RestWeights w = rest_weights(a, r, n, c);
  const int64_t b = part * a.per, e = min(a.V, b + a.per);
  const int64_t pick = pick_range([&](int64_t at, int64_t end, double* x) {
    double left[kE], all[kE];
    w(at, end, left, all);
#pragma unroll
    for (int i = 0; i < kE; ++i) x[i] = rest ? left[i] : all[i];
  }, b, e, before, target);
  if (p == 0) a.next[r] = pick < 0 ? c.arg : pick;
}

int parts_of(int64_t V, int64_t* per) {
  *per = ((V + kParts - 1) / kParts + kPart - 1) / kPart * kPart;
  return (int)((V + *per - 1) / *per);
}

}  // namespace

// bytes of workspace of a call
CB_EXPORT int64_t cb_verify_scratch(int64_t R, int64_t C, int64_t V) {
  int64_t per;
  const int64_t P = parts_of(V, &per);
  return R * C * P * (int64_t)sizeof(PartStat) + R * P * (int64_t)sizeof(double2) + R * C * (int64_t)sizeof(int);
}

CB_EXPORT int cb_verify_tree(const void* logits, int64_t lds, int64_t ldr, const void* tokens, const void* anc, const void* temperature,
                             const void* u, void* path, void* steps, void* next, void* scratch, int64_t R, int64_t C, int64_t V, void* stream) {
  if (!logits || !tokens || !anc || !temperature || !u || !path || !steps || !next || !scratch) return CB_ERR_ARG;
  if (R < 1 || C < 1 || C > kNodes || V < 1 || V > 0x7fffffff || R * C > 65535) return CB_ERR_SHAPE;
  VerifyArgs a = {};
  a.logits = (const float*)logits; a.lds = lds; a.ldr = ldr; a.tokens = (const int64_t*)tokens; a.anc = (const int64_t*)anc;
  a.temperature = (const float*)temperature; a.u = (const float*)u; a.path = (int*)path; a.steps = (int*)steps; a.next = (int64_t*)next;
  a.V = V; a.R = (int)R; a.C = (int)C; a.P = parts_of(V, &a.per);
  a.stats = (PartStat*)scratch;
  a.picks = (int*)(a.stats + R * C * a.P);
  cudaStream_t st = (cudaStream_t)stream;
  cudaError_t e = cb_launch(row_stats_kernel, dim3((unsigned)a.P, (unsigned)(R * C)), dim3(kNT), 0, st, a);
  if (e == cudaSuccess) e = cb_launch(tree_pick_kernel, dim3((unsigned)(R * C)), dim3(kNT), 0, st, a);
  if (e == cudaSuccess) e = cb_launch(tree_walk_kernel, dim3((unsigned)R), dim3(kNodes), 0, st, a);
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
  a.V = V; a.R = (int)R; a.C = (int)C; a.P = parts_of(V, &a.per);
  a.stats = (PartStat*)scratch;
  a.rest = (double2*)(a.stats + R * C * a.P);
  cudaStream_t st = (cudaStream_t)stream;
  cudaError_t e = cb_launch(row_stats_kernel, dim3((unsigned)a.P, (unsigned)(R * C)), dim3(kNT), 0, st, a);
  if (e == cudaSuccess) e = cb_launch(draft_rest_kernel, dim3((unsigned)a.P, (unsigned)R), dim3(kNT), 0, st, a);
  if (e == cudaSuccess) e = cb_launch(draft_pick_kernel, dim3((unsigned)R), dim3(kNT), 0, st, a);
  return (int)e;
}
