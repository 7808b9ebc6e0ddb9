// The gated delta rule over a tree of drafted tokens.
//
// A chain is stepped token by token; in a tree every branch would need a state of its own.  Unrolled along the path of a node, with
// g = log alpha, c_j = the sum of g over the path of j (itself included) and S0 the sequence's state,
//   d_j = beta_j (v_j - e^{c_j} S0^T k_j - sum_{i above j} e^{c_j - c_i} (k_j.k_i) d_i)
//   o_j = e^{c_j} S0^T q_j + sum_{i above j or j} e^{c_j - c_i} (q_j.k_i) d_i,     out_j = rmsnorm(o_j) * w * silu(z_j) (or sigmoid)
// so the state is read once whatever the shape of the tree, and the nodes meet in two masked Gram matrices.  q, k, v come from the causal
// convolution along the path: its older taps are the node's ancestors, behind them the ring.  State and ring stay as they were; k, d and
// alpha of every node are recorded and the raw rows kept, from which a commit replays the accepted path (tree_commit.cu).
//
// 1. rows: a warp a (node, head) convolves, norms q and k and leaves them, and v, as fp32 rows by head.  (Within the kernel below it would be
//    repeated for every value head of a key head and every group of columns, which only few nodes are worth.)
// 2. nodes: a CTA owns DVS columns of one head's state; the DV / DVS CTAs of a head are a cluster, share out the Gram matrices and
//    exchange the sums of squares of the norm.  (1 - A)^-1 of the strictly lower matrix A of the first equation is built from inverted 8 x 8
//    blocks by doubling, so that what follows are small dense products.
// Everything is fp32, as the recorded updates are; the products with the state are most of it (2 C DK DV multiplications a head: 4 x 64
// nodes of 48 heads 0.8 GFLOP).  Sums of g along a path are 64-bit, since differences of them are exponents.  Coefficients off a node's path
// are exactly 0 and skipped, so that a node's values do not reach its siblings whatever they are.  A CTA runs through the code once, and
// at small sizes fetching it is what takes the time: loops are kept rolled (66 KB of code unrolled: 18 us for four nodes).
#include "sm100.cuh"

namespace {

constexpr int kRing = 16, kMaxNodes = 64, kThreads = 256, kFuse = 8;

struct GdnTreeArgs {
  const bf16* proj; int64_t ldp;          // [R * C, ldp]: q | k | v | z | b | a
  const float* conv_w;                    // [conv, 4], oldest tap first
  const float* A_log; const float* dt_bias; const float* norm_w;
  const bf16* ring;                       // [slots, 16, conv]
  const float* state;                     // [slots, nv, dk, dv]
  const int* slots; const int* positions; // [R]
  const int64_t* anc;                     // [R, C]
  bf16* out; int64_t ldo;                 // [R * C, nv * dv]
  float* record;                          // [R, C, nv, dk + dv + 1]
  bf16* raw;                              // [R, C, conv]
  float* rows;                            // [R, 2 nk + nv, C, d]: q heads, k heads, v heads
  int R, C, Cp, nk, nv, rep, nslots, gate_sigmoid;
  float eps;
};

__device__ __forceinline__ uint64_t path_word(const GdnTreeArgs& a, int r, int j) {
  const uint64_t on = (uint64_t)a.anc[(int64_t)r * a.C + j];
  return on ? (on & (~0ull >> (63 - j))) | 1ull << j : 0;    // a path ends at its node
}
__device__ __forceinline__ bool unused(const GdnTreeArgs& a, int r) {
  return a.slots[r] < 0 || a.slots[r] >= a.nslots || a.positions[r] < 0;
}

// ---- rows -----------------------------------------------------------------------------------
// Four (two) channels a lane of head u's row at node j: convolved along the path `on`, SiLU, q and k normed.  `raw` says whether to keep the raw row.
template <int D>
__device__ __forceinline__ void tree_row(const GdnTreeArgs& a, int r, int j, uint64_t on, int u, bool raw, float (&y)[D / 32]) {
  constexpr int E = D / 32;
  const int lane = threadIdx.x & 31, conv = (2 * a.nk + a.nv) * D, c = u * D + lane * E, pos = a.positions[r] + __popcll(on) - 1;
  const bf16* ring = a.ring + (int64_t)a.slots[r] * kRing * conv + c;
  const bf16* rows = a.proj + (int64_t)r * a.C * a.ldp + c;
  uint32_t x[4][E / 2];
  uint64_t up = on;
#pragma unroll
  for (int b = 0; b < 4; ++b) {                              // the node, its parent, ...; behind the root the ring
    const int node = up ? 63 - __clzll((long long)up) : -1;
    if (up) up &= ~(1ull << node);
    const bf16* from = node >= 0 ? rows + (int64_t)node * a.ldp : (pos >= b ? ring + (int64_t)((pos - b) & (kRing - 1)) * conv : nullptr);
#pragma unroll
    for (int e = 0; e < E / 2; ++e) x[b][e] = 0;
    if (from) {
      if (E == 4) *reinterpret_cast<uint2*>(x[b]) = *reinterpret_cast<const uint2*>(from);
      else x[b][0] = *reinterpret_cast<const uint32_t*>(from);
    }
  }
  float4 w[E];
#pragma unroll
  for (int e = 0; e < E; ++e) w[e] = *reinterpret_cast<const float4*>(a.conv_w + (int64_t)(c + e) * 4);
  if (raw) {
    bf16* to = a.raw + ((int64_t)r * a.C + j) * conv + c;
    if (E == 4) *reinterpret_cast<uint2*>(to) = *reinterpret_cast<const uint2*>(x[0]);
    else *reinterpret_cast<uint32_t*>(to) = x[0][0];
  }
  float ss = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const auto f = [&](int b) { return __uint_as_float(e & 1 ? x[b][e / 2] & 0xffff0000u : x[b][e / 2] << 16); };
    float v = w[e].x * f(3);
    v = fmaf(w[e].y, f(2), v);
    v = fmaf(w[e].z, f(1), v);
    v = fmaf(w[e].w, f(0), v);
    y[e] = v / (1.f + expf(-v));
    ss = fmaf(y[e], y[e], ss);
  }
  if (u < 2 * a.nk) {
    float f = rsqrtf(warp_sum(ss) + 1e-6f);
    if (u < a.nk) f *= D == 128 ? 0.08838834764831845f : 0.125f;      // D^-0.5
#pragma unroll
    for (int e = 0; e < E; ++e) y[e] *= f;
  }
}

template <int D>
__global__ void __launch_bounds__(kThreads) gdn_tree_rows_kernel(const GdnTreeArgs a) {
  constexpr int E = D / 32;
  griddep_launch();
  griddep_wait();
  const int heads = 2 * a.nk + a.nv, lane = threadIdx.x & 31;
  const int u = blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5), j = blockIdx.y, r = blockIdx.z;
  if (u >= heads) return;
  const uint64_t on = path_word(a, r, j);
  if (on == 0 || unused(a, r)) return;
  float y[E];
  tree_row<D>(a, r, j, on, u, true, y);
  float* to = a.rows + (((int64_t)r * heads + u) * a.C + j) * D + lane * E;
  if (E == 4) *reinterpret_cast<float4*>(to) = *reinterpret_cast<const float4*>(y);
  else *reinterpret_cast<float2*>(to) = *reinterpret_cast<const float2*>(y);
}

// ---- nodes ----------------------------------------------------------------------------------
// The products with the state: a warp keeps DK / SL channels of all DVS columns in registers, DVS / 32 columns a lane, and multiplies every
// vector of its share with them (the vector's channels are the same for all lanes); the SL partial products meet in shared memory, BV
// vectors at a time.  (What is left of it is bound by the loads of the vectors, 16 bytes a lane whether the lanes differ or not.)
template <int DK, int DVS>
struct TreeState {
  static constexpr int WC = DVS / 32, SL = WC == 4 ? 8 : 4, VG = kThreads / 32 / SL, KR = DK / SL, BV = WC == 4 ? 8 : 32;
};

// With many nodes and a whole head a CTA, tiles of eight vectors by eight columns a thread from shared memory are the better way: no partial
// products, and 16 multiplications for a load of 16 bytes.  (192 heads of 64 nodes 106.7 -> 94.5 us, of 48 nodes 76.5 -> 75.1, 240 heads of 40 nodes 67.0 -> 69.9.)
template <int DK, int DVS, bool TILE>
struct TreeSmem {                         // floats
  static constexpr int LK = DK + 4;       // rows a quarter warp reads lie in different banks
  int kn, qn, d, o, z, P, A, B, D, total; // z as bf16; A, B, D (and the doubling's scratch in D's place) follow the partial products in their place
  __host__ __device__ explicit TreeSmem(int Cp) {
    kn = 0;
    qn = kn + Cp * LK;
    d = qn + Cp * LK;
    o = d + Cp * DVS;
    z = o + Cp * DVS;
    P = A = z + Cp * DVS / 2;
    B = A + Cp * (Cp + 4);
    D = B + Cp * (Cp + 4);
    const int scratch = Cp * DVS > 32 * 36 ? Cp * DVS : 32 * 36;
    const int bv = 2 * Cp < TreeState<DK, DVS>::BV ? 2 * Cp : TreeState<DK, DVS>::BV;
    const int a = P + (TILE ? DK * DVS : TreeState<DK, DVS>::SL * bv * DVS), b = D + scratch;
    total = a > b ? a : b;
  }
};

// x[j][.] += sum_{i < i1} m[j][i] y[i][.] for RT rows j and four columns; coefficients 0 are skipped
template <int RT>
__device__ __forceinline__ void rows_times(float (&x)[RT][4], const float* m, int ldm, const float* y, int ldy, int i1) {
#pragma unroll 1
  for (int i = 0; i < i1; i += 4) {
    float4 w[RT], v[4];
#pragma unroll
    for (int j = 0; j < RT; ++j) w[j] = *reinterpret_cast<const float4*>(m + j * ldm + i);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = *reinterpret_cast<const float4*>(y + (i + e) * ldy);
#pragma unroll
    for (int j = 0; j < RT; ++j) {
      const float f[4] = {w[j].x, w[j].y, w[j].z, w[j].w};
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (f[e] != 0.f) {
          x[j][0] = fmaf(f[e], v[e].x, x[j][0]);
          x[j][1] = fmaf(f[e], v[e].y, x[j][1]);
          x[j][2] = fmaf(f[e], v[e].z, x[j][2]);
          x[j][3] = fmaf(f[e], v[e].w, x[j][3]);
        }
    }
  }
}

template <int NS>
__device__ __forceinline__ void sync_all() {
  if (NS > 1) sm100::cluster_sync_all();
  else __syncthreads();
}

template <int DK, int DV, int DVS, bool TILE, bool FUSE>
__global__ void __launch_bounds__(kThreads) gdn_tree_kernel(const GdnTreeArgs a) {
  constexpr int NS = DV / DVS, LK = TreeSmem<DK, DVS, TILE>::LK;
  extern __shared__ __align__(16) float sm[];
  __shared__ uint64_t anc_s[kMaxNodes];
  __shared__ double c_s[kMaxNodes];
  __shared__ __align__(16) float g_s[kMaxNodes];
  __shared__ float beta_s[kMaxNodes], dec_s[kMaxNodes], ss_s[kMaxNodes];
  griddep_launch();
  griddep_wait();
  const int cg = blockIdx.x, h = blockIdx.y, r = blockIdx.z, kh = h / a.rep, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int C = a.C, Cp = a.Cp, LA = Cp + 4, heads = 2 * a.nk + a.nv;
  const TreeSmem<DK, DVS, TILE> off(Cp);
  float *kn = sm + off.kn, *qn = sm + off.qn, *d = sm + off.d, *o = sm + off.o, *A = sm + off.A, *B = sm + off.B, *P = sm + off.P, *D = sm + off.D;
  bf16* zs = reinterpret_cast<bf16*>(sm + off.z);
  const int conv = 2 * a.nk * DK + a.nv * DV, col0 = cg * DVS;
  auto copy16 = [](void* to, const void* from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(sm100::smem_u32(to)), "l"(from));
  };
  // All that is read from memory is requested at once.  Rows without a node hold anything; they meet coefficients 0 alone.
  const int slot = a.slots[r], pos0 = a.positions[r];
  uint64_t on = 0;
  float xb = 0.f, xa = 0.f;
  if (tid < C) {
    const bf16* row = a.proj + ((int64_t)r * C + tid) * a.ldp + conv + a.nv * DV;
    on = path_word(a, r, tid);
    xb = __bfloat162float(row[h]);
    xa = __bfloat162float(row[a.nv + h]);
  }
  const float rate = a.A_log[h], dtb = a.dt_bias[h];
  if (!FUSE) {
    const float* q = a.rows + ((int64_t)r * heads + kh) * C * DK;
    const float* k = q + (int64_t)a.nk * C * DK;
    const float* v = a.rows + ((int64_t)r * heads + 2 * a.nk + h) * C * DV + col0;
#pragma unroll 1
    for (int i = tid; i < C * DK / 4; i += kThreads) {
      const int j = i / (DK / 4), c = i % (DK / 4) * 4;
      copy16(kn + j * LK + c, k + j * DK + c);
      copy16(qn + j * LK + c, q + j * DK + c);
    }
#pragma unroll 1
    for (int i = tid; i < C * DVS / 4; i += kThreads) {
      const int j = i / (DVS / 4), c = i % (DVS / 4) * 4;
      copy16(d + j * DVS + c, v + (int64_t)j * DV + c);
    }
  }
  {
    const bf16* z = a.proj + (int64_t)r * C * a.ldp + conv + h * DV + col0;
#pragma unroll 1
    for (int i = tid; i < C * DVS / 8; i += kThreads) {
      const int j = i / (DVS / 8), c = i % (DVS / 8) * 8;
      copy16(zs + j * DVS + c, z + j * a.ldp + c);
    }
  }
  if (slot < 0 || slot >= a.nslots || pos0 < 0) {            // an unused row: the same for the whole cluster
    asm volatile("cp.async.wait_all;" ::: "memory");
    return;
  }
  constexpr int WC = TreeState<DK, DVS>::WC, SL = TreeState<DK, DVS>::SL, VG = TreeState<DK, DVS>::VG, KR = TreeState<DK, DVS>::KR, BV = TreeState<DK, DVS>::BV;
  const int sl = warp % SL;
  float st[TILE ? 1 : KR][WC];
  const float* head = a.state + ((int64_t)slot * a.nv + h) * DK * DV + col0;
  if (TILE) {
#pragma unroll 1
    for (int i = tid; i < DK * DVS / 4; i += kThreads) copy16(P + i * 4, head + (int64_t)(i / (DVS / 4)) * DV + i % (DVS / 4) * 4);
  } else {
    const float* sp = head + sl * KR * DV + lane * WC;
#pragma unroll
    for (int k = 0; k < KR; ++k) {
      float* x = st[TILE ? 0 : k];
      if (WC == 4) *reinterpret_cast<float4*>(x) = *reinterpret_cast<const float4*>(sp + k * DV);
      else if (WC == 2) *reinterpret_cast<float2*>(x) = *reinterpret_cast<const float2*>(sp + k * DV);
      else x[0] = sp[k * DV];
    }
  }
  if (FUSE) {                                                // a warp a row of q, k or v
#pragma unroll 1
    for (int i = warp; i < 3 * C; i += kThreads / 32) {
      const int j = i / 3, which = i % 3, u = which == 0 ? kh : which == 1 ? a.nk + kh : 2 * a.nk + h;
      const uint64_t path = path_word(a, r, j);
      if (path == 0) continue;
      float y[DK / 32];
      tree_row<DK>(a, r, j, path, u, cg == 0 && (which == 2 || h % a.rep == 0), y);
      const int c = lane * (DK / 32) - (which == 2 ? col0 : 0);        // (DK = DV)
      float* to = which == 0 ? qn + j * LK + c : which == 1 ? kn + j * LK + c : d + j * DVS + c;
      if (c >= 0 && (which < 2 || c < DVS)) {
        if (DK == 128) *reinterpret_cast<float4*>(to) = *reinterpret_cast<const float4*>(y);
        else *reinterpret_cast<float2*>(to) = *reinterpret_cast<const float2*>(y);
      }
    }
  }
  if (tid < Cp) {
    const float x = xa + dtb;
    anc_s[tid] = on;
    const float g = -expf(rate) * (x > 20.f ? x : log1pf(expf(x)));
    g_s[tid] = !on ? 0.f : g < -1e4f ? -1e4f : g;             // exp of less is 0 all the same
    beta_s[tid] = 1.f / (1.f + expf(-xb));
  }
  __syncthreads();
  if (tid < Cp) {
    double c[4] = {};
#pragma unroll 1
    for (int i = 0; on; i += 4, on >>= 4) {
      const float4 g = *reinterpret_cast<const float4*>(g_s + i);
      if (on & 1) c[0] += (double)g.x;
      if (on & 2) c[1] += (double)g.y;
      if (on & 4) c[2] += (double)g.z;
      if (on & 8) c[3] += (double)g.w;
    }
    const double sum = (c[0] + c[1]) + (c[2] + c[3]);
    c_s[tid] = sum;
    dec_s[tid] = expf((float)sum);
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  __syncthreads();
  // ---- S0^T k and S0^T q (vector v < Cp: row of kn, then of qn)
  if (TILE) {
    // 16 groups of columns 4 g + {0..3} and 64 + 4 g + {0..3}, 16 of vectors v0 + 16 n
    const int c4 = tid % 16 * 4, v0 = tid / 16;
    float acc[8][8];
#pragma unroll
    for (int n = 0; n < 8; ++n)
#pragma unroll
      for (int c = 0; c < 8; ++c) acc[n][c] = 0.f;
    const float* vec[8];
#pragma unroll
    for (int n = 0; n < 8; ++n) {
      const int v = min(v0 + 16 * n, 2 * Cp - 1);
      vec[n] = v < Cp ? kn + v * LK : qn + (v - Cp) * LK;
    }
#pragma unroll 1
    for (int k = 0; k < DK; k += 4) {
      float4 s[4][2];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[e][0] = *reinterpret_cast<const float4*>(P + (k + e) * DVS + c4);
        s[e][1] = *reinterpret_cast<const float4*>(P + (k + e) * DVS + c4 + DVS / 2);
      }
#pragma unroll
      for (int n = 0; n < 8; ++n) {
        const float4 x = *reinterpret_cast<const float4*>(vec[n] + k);
        const float f[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            acc[n][4 * u] = fmaf(f[e], s[e][u].x, acc[n][4 * u]);
            acc[n][4 * u + 1] = fmaf(f[e], s[e][u].y, acc[n][4 * u + 1]);
            acc[n][4 * u + 2] = fmaf(f[e], s[e][u].z, acc[n][4 * u + 2]);
            acc[n][4 * u + 3] = fmaf(f[e], s[e][u].w, acc[n][4 * u + 3]);
          }
      }
    }
#pragma unroll
    for (int n = 0; n < 8; ++n) {
      const int v = v0 + 16 * n, j = v < Cp ? v : v - Cp;
      if (v >= 2 * Cp) continue;
      const float f = dec_s[j], b = beta_s[j];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        float4* x = reinterpret_cast<float4*>((v < Cp ? d : o) + j * DVS + c4 + u * (DVS / 2));
        float4 y = make_float4(f * acc[n][4 * u], f * acc[n][4 * u + 1], f * acc[n][4 * u + 2], f * acc[n][4 * u + 3]);
        if (v < Cp) {
          const float4 w = *x;
          y = make_float4(b * (w.x - y.x), b * (w.y - y.y), b * (w.z - y.z), b * (w.w - y.w));
        }
        *x = y;
      }
    }
  } else {
#pragma unroll 1
  for (int b0 = 0; b0 < 2 * Cp; b0 += BV) {
    const int here = min(BV, 2 * Cp - b0);
#pragma unroll 1
    for (int v0 = (warp / SL) * 2; v0 < here; v0 += 2 * VG) {        // two vectors at a time (their number is even)
      const int v = b0 + v0;
      const float* x = (v < Cp ? kn + v * LK : qn + (v - Cp) * LK) + sl * KR;
      float acc[2][WC];
#pragma unroll
      for (int c = 0; c < WC; ++c) acc[0][c] = acc[1][c] = 0.f;
#pragma unroll
      for (int k = 0; k < KR; k += 4) {
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          const float4 f = *reinterpret_cast<const float4*>(x + n * LK + k);
#pragma unroll
          for (int c = 0; c < WC; ++c) {
            acc[n][c] = fmaf(f.x, st[TILE ? 0 : k][c], acc[n][c]);
            acc[n][c] = fmaf(f.y, st[TILE ? 0 : k + 1][c], acc[n][c]);
            acc[n][c] = fmaf(f.z, st[TILE ? 0 : k + 2][c], acc[n][c]);
            acc[n][c] = fmaf(f.w, st[TILE ? 0 : k + 3][c], acc[n][c]);
          }
        }
      }
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        float* to = P + (sl * here + v0 + n) * DVS + lane * WC;
        if (WC == 4) *reinterpret_cast<float4*>(to) = *reinterpret_cast<const float4*>(acc[n]);
        else if (WC == 2) *reinterpret_cast<float2*>(to) = *reinterpret_cast<const float2*>(acc[n]);
        else to[0] = acc[n][0];
      }
    }
    __syncthreads();
#pragma unroll 1
    for (int i = tid; i < here * DVS / 4; i += kThreads) {
      float4 s = *reinterpret_cast<const float4*>(P + i * 4);
#pragma unroll
      for (int n = 1; n < SL; ++n) {
        const float4 p = *reinterpret_cast<const float4*>(P + n * here * DVS + i * 4);
        s.x += p.x; s.y += p.y; s.z += p.z; s.w += p.w;
      }
      const int v = b0 + i / (DVS / 4), j = v < Cp ? v : v - Cp, c = i % (DVS / 4) * 4;
      const float f = dec_s[j], b = beta_s[j];
      float4* x = reinterpret_cast<float4*>((v < Cp ? d : o) + j * DVS + c);
      if (v < Cp) {
        const float4 w = *x;
        *x = make_float4(b * (w.x - f * s.x), b * (w.y - f * s.y), b * (w.z - f * s.z), b * (w.w - f * s.w));
      } else *x = make_float4(f * s.x, f * s.y, f * s.z, f * s.w);
    }
    if (b0 + BV < 2 * Cp) __syncthreads();
  }
  }
  sync_all<NS>();                                            // the partial products' place is free, in every CTA of the cluster
  // ---- Gram matrices: A_ji = -beta_j e^{c_j - c_i} k_j.k_i above j, B_ji = e^{c_j - c_i} q_j.k_i above j and at j; 0 elsewhere.  Units of
  // 4 x 4 on and below the diagonal, four threads (a quarter of the channels each) a unit; the CTAs of a cluster take every NS-th unit.
  {
    const int nb = Cp / 4, units = nb * (nb + 1) / 2, part = tid & 3;
    const unsigned four = 0xfu << (lane & 28);
#pragma unroll 1
    for (int u = tid; u < Cp * nb; u += kThreads)            // above the diagonal blocks A is 0; B is not read there
      if (u % nb > u / nb / 4) *reinterpret_cast<float4*>(A + u / nb * LA + u % nb * 4) = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
    for (int u = (tid >> 2) * NS + cg; u < units; u += kThreads / 4 * NS) {        // the four threads of a unit stay together
      const int jb = (int)((sqrtf((float)(8 * u + 1)) - 1.f) * 0.5f), j0 = jb * 4, i0 = (u - jb * (jb + 1) / 2) * 4;      // exact: u <= 135
      float g[2][4][4];                                      // k_j.k_i, q_j.k_i
#pragma unroll
      for (int x = 0; x < 4; ++x)
#pragma unroll
        for (int y = 0; y < 4; ++y) g[0][x][y] = g[1][x][y] = 0.f;
#pragma unroll 1
      for (int k = part * 4; k < DK; k += 16) {              // quarters interleaved by 16 bytes: the four threads read neighbours
        float4 ki[4];
#pragma unroll
        for (int y = 0; y < 4; ++y) ki[y] = *reinterpret_cast<const float4*>(kn + (i0 + y) * LK + k);
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const float4 kj = *reinterpret_cast<const float4*>(kn + (j0 + x) * LK + k), qj = *reinterpret_cast<const float4*>(qn + (j0 + x) * LK + k);
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            g[0][x][y] = fmaf(kj.x, ki[y].x, fmaf(kj.y, ki[y].y, fmaf(kj.z, ki[y].z, fmaf(kj.w, ki[y].w, g[0][x][y]))));
            g[1][x][y] = fmaf(qj.x, ki[y].x, fmaf(qj.y, ki[y].y, fmaf(qj.z, ki[y].z, fmaf(qj.w, ki[y].w, g[1][x][y]))));
          }
        }
      }
      // the four quarters are added so that thread x of the four ends up with row x: first pairs of rows, then rows
      const int j = j0 + part;
      const bool hi = part & 2, odd = part & 1;
      float row[2][4];
#pragma unroll
      for (int w = 0; w < 2; ++w)
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          const float s0 = __shfl_xor_sync(four, hi ? g[w][0][y] : g[w][2][y], 2), s1 = __shfl_xor_sync(four, hi ? g[w][1][y] : g[w][3][y], 2);
          const float a0 = (hi ? g[w][2][y] : g[w][0][y]) + s0, a1 = (hi ? g[w][3][y] : g[w][1][y]) + s1;
          row[w][y] = (odd ? a1 : a0) + __shfl_xor_sync(four, odd ? a0 : a1, 1);
        }
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        const int i = i0 + y;
        const bool on = anc_s[j] >> i & 1;
        const float f = on ? expf((float)(c_s[j] - c_s[i])) : 0.f;
        row[0][y] = on && i != j ? -beta_s[j] * f * row[0][y] : 0.f;
        row[1][y] = on ? f * row[1][y] : 0.f;
      }
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        float* to = (w ? B : A) + j * LA + i0;
        if (NS == 1) *reinterpret_cast<float4*>(to) = make_float4(row[w][0], row[w][1], row[w][2], row[w][3]);
        else {
#pragma unroll
          for (int n = 0; n < NS; ++n)
            asm volatile("st.shared::cluster.v4.f32 [%0], {%1,%2,%3,%4};" ::"r"(sm100::map_to_cta(sm100::smem_u32(to), n)), "f"(row[w][0]), "f"(row[w][1]),
                         "f"(row[w][2]), "f"(row[w][3]) : "memory");
        }
      }
    }
  }
  sync_all<NS>();
  // ---- M = (1 - A)^-1 in A's place: 4 x 4 blocks on the diagonal, a thread a column, then M21 = M22 A21 M11 by doubling
  if (tid < Cp) {
    const int i = tid % 4;
    float* x = A + (tid / 4 * 4) * LA + tid / 4 * 4;         // strictly lower: x10, x20, x21, x30, x31, x32
    const float x10 = x[LA], x20 = x[2 * LA], x21 = x[2 * LA + 1], x30 = x[3 * LA], x31 = x[3 * LA + 1], x32 = x[3 * LA + 2];
    __syncwarp(Cp - warp * 32 >= 32 ? 0xffffffffu : (1u << (Cp - warp * 32)) - 1);      // all four have read before one writes
    auto times = [](float f, float y) { return f != 0.f && y != 0.f ? f * y : 0.f; };
    const float m0 = i == 0 ? 1.f : 0.f;
    const float m1 = i == 1 ? 1.f : times(x10, m0);
    const float m2 = i == 2 ? 1.f : times(x20, m0) + times(x21, m1);
    const float m3 = i == 3 ? 1.f : times(x30, m0) + times(x31, m1) + times(x32, m2);
    x[i] = m0;
    x[LA + i] = m1;
    x[2 * LA + i] = m2;
    x[3 * LA + i] = m3;
  }
  __syncthreads();
#pragma unroll 1
  for (int n = 4; n < Cp; n *= 2) {                          // pairs of n x n blocks: rows [p + n, p + 2 n), columns [p, p + n)
    const int q = n / 4, units = n * q;                      // a row and four columns a thread
    const int u = tid % units, p = tid / units * 2 * n, x0 = u / q, y0 = u % q * 4;
    const bool mine = p + n < Cp && x0 < Cp - p - n;
    float* low = A + (p + n + x0) * LA + p;                  // this row of the lower block, first column of the pair
    float* t = D + tid / units * n * (n + 4);                // [n][n + 4] a pair: A21 M11
#pragma unroll 1
    for (int s = 0; s < 2; ++s) {
      float x[1][4] = {};
      if (mine) rows_times(x, s ? low + n : low, 0, s ? t + y0 : A + p * LA + p + y0, s ? n + 4 : LA, s ? x0 / 4 * 4 + 4 : n);
      __syncthreads();                                       // A21 has been read before it is written
      if (mine) *reinterpret_cast<float4*>(s ? low + y0 : t + x0 * (n + 4) + y0) = make_float4(x[0][0], x[0][1], x[0][2], x[0][3]);
      __syncthreads();
    }
  }
  // ---- updates D = M W and outputs O += B D with their squares, four rows and four columns a thread
#pragma unroll 1
  for (int pass = 0; pass < 2; ++pass) {
#pragma unroll 1
    for (int u = tid; u < Cp / 4 * (DVS / 4); u += kThreads) {
      const int c4 = u % (DVS / 4) * 4, j0 = u / (DVS / 4) * 4;
      float x[4][4] = {};
      if (pass) {
#pragma unroll
        for (int e = 0; e < 4; ++e) *reinterpret_cast<float4*>(x[e]) = *reinterpret_cast<const float4*>(o + (j0 + e) * DVS + c4);
      }
      rows_times(x, (pass ? B : A) + j0 * LA, LA, (pass ? D : d) + c4, DVS, j0 + 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) *reinterpret_cast<float4*>((pass ? o : D) + (j0 + e) * DVS + c4) = make_float4(x[e][0], x[e][1], x[e][2], x[e][3]);
      if (pass) {                                            // DVS / 4 neighbouring lanes hold a row's columns, all of them or none
        const unsigned lanes = DVS == 128 ? 0xffffffffu : ((1u << (DVS / 4)) - 1) << (lane / (DVS / 4) * (DVS / 4));
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float ss = fmaf(x[e][0], x[e][0], fmaf(x[e][1], x[e][1], fmaf(x[e][2], x[e][2], x[e][3] * x[e][3])));
#pragma unroll
          for (int w = DVS / 8; w > 0; w >>= 1) ss += __shfl_xor_sync(lanes, ss, w);
          if (c4 == 0) ss_s[j0 + e] = ss;
        }
      }
    }
    __syncthreads();
  }
  // ---- norm over the head's columns, gate, record
  sync_all<NS>();
  if (tid < C) {
    float ss = ss_s[tid];
    if (NS > 1) {
      ss = 0.f;
#pragma unroll
      for (int n = 0; n < NS; ++n) {                         // the same order in every CTA
        float v;
        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(sm100::map_to_cta(sm100::smem_u32(ss_s + tid), n)) : "memory");
        ss += v;
      }
    }
    dec_s[tid] = rsqrtf(ss * (1.f / DV) + a.eps);
    if (cg == 0 && anc_s[tid]) a.record[(((int64_t)r * C + tid) * a.nv + h) * (DK + DV + 1) + DK + DV] = expf(g_s[tid]);
  }
  if (NS > 1) sm100::cluster_sync_all();                     // nobody leaves while its sums may still be read
  else __syncthreads();
  const float4 nw = *reinterpret_cast<const float4*>(a.norm_w + col0 + tid % (DVS / 4) * 4);
#pragma unroll 1
  for (int i = tid; i < C * (DVS / 4); i += kThreads) {
    const int j = i / (DVS / 4), c = i % (DVS / 4) * 4;      // the same columns in every turn
    if (!anc_s[j]) continue;
    const int64_t row = (int64_t)r * C + j;
    const float4 x = *reinterpret_cast<const float4*>(o + j * DVS + c), u = *reinterpret_cast<const float4*>(D + j * DVS + c);
    const uint2 zb = *reinterpret_cast<const uint2*>(zs + j * DVS + c);
    const float z[4] = {__uint_as_float(zb.x << 16), __uint_as_float(zb.x & 0xffff0000u), __uint_as_float(zb.y << 16), __uint_as_float(zb.y & 0xffff0000u)};
    float y[4] = {x.x * nw.x, x.y * nw.y, x.z * nw.z, x.w * nw.w};
    const float f = dec_s[j];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float s = 1.f / (1.f + expf(-z[e]));
      y[e] *= f * (a.gate_sigmoid ? s : z[e] * s);
    }
    bf16* out = a.out + row * a.ldo + h * DV + col0 + c;
    *reinterpret_cast<uint2*>(out) = make_uint2(pack_bf162(y[0], y[1]), pack_bf162(y[2], y[3]));
    float* rec = a.record + (row * a.nv + h) * (DK + DV + 1) + DK + col0 + c;
    rec[0] = u.x; rec[1] = u.y; rec[2] = u.z; rec[3] = u.w;
  }
  constexpr int KS = DK / NS;                                // the CTAs of a cluster share the copy of the keys
#pragma unroll 4
  for (int i = tid; i < C * KS; i += kThreads) {
    const int j = i / KS, c = cg * KS + i % KS;
    if (anc_s[j]) a.record[(((int64_t)r * C + j) * a.nv + h) * (DK + DV + 1) + c] = kn[j * LK + c];
  }
}

template <int DK, int DV, int DVS, bool FUSE, bool TILE = false>
int launch_gdn_tree(const GdnTreeArgs& a, int R, cudaStream_t st) {
  auto kern = gdn_tree_kernel<DK, DV, DVS, TILE, FUSE>;
  const size_t smem = TreeSmem<DK, DVS, TILE>(a.Cp).total * sizeof(float);
  static SmemLimit limit;
  std::lock_guard<std::mutex> lock(limit.held);
  cudaError_t e = limit.set(kern, smem);
  if (e != cudaSuccess) return (int)e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(DV / DVS, (unsigned)a.nv, (unsigned)R);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (g_cb_use_pdl || !FUSE) {                               // (behind the rows, it is the second kernel of the operator)
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (DV / DVS > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = DV / DVS;
    attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
    ++n;
  }
  cfg.attrs = attr;
  cfg.numAttrs = (unsigned)n;
  if (g_cb_trace_names) cb_trace_name((const void*)kern);
  return (int)cudaLaunchKernelEx(&cfg, kern, a);
}

}  // namespace

CB_EXPORT int cb_gdn_tree(const void* proj, int64_t ldp, const void* conv_w, const void* A_log, const void* dt_bias, const void* norm_w,
                          const void* ring, const void* state, const void* slots, const void* positions, const void* anc, void* out, int64_t ldo,
                          void* record, void* raw, void* rows, int64_t nslots, int64_t R, int64_t C, int64_t nk, int64_t nv, int64_t dk, int64_t dv, float eps,
                          int64_t gate_sigmoid, void* stream) {
  if (!proj || !conv_w || !A_log || !dt_bias || !norm_w || !ring || !state || !slots || !positions || !anc || !out || !record || !raw) return CB_ERR_ARG;
  if (R < 1 || R > 65535 || C < 1 || C > kMaxNodes || nk < 1 || nv < 1 || nv % nk || nv > 65535 || ldp % 8 || ldo % 4 || ((uintptr_t)out & 7) || ((uintptr_t)norm_w & 15) ||
      (((uintptr_t)proj | (uintptr_t)ring | (uintptr_t)state | (uintptr_t)raw | (uintptr_t)rows | (uintptr_t)conv_w) & 15)) return CB_ERR_SHAPE;
  GdnTreeArgs a{(const bf16*)proj, ldp, (const float*)conv_w, (const float*)A_log, (const float*)dt_bias, (const float*)norm_w, (const bf16*)ring,
                (const float*)state, (const int*)slots, (const int*)positions, (const int64_t*)anc, (bf16*)out, ldo, (float*)record, (bf16*)raw, (float*)rows,
                (int)R, (int)C, (int)((C + 7) / 8 * 8), (int)nk, (int)nv, (int)(nv / nk), (int)nslots, (int)gate_sigmoid, eps};
  cudaStream_t st = (cudaStream_t)stream;
  if (!((dk == 128 && dv == 128) || (dk == 64 && dv == 64))) return CB_ERR_SHAPE;
  // Few nodes: the rows in the kernel that uses them, repeated for the value heads of a key head, a launch less.  us of a pass with a kernel
  // of their own / without: 4 nodes, 32 heads 11.5 / 11.2, 8 x 4 nodes 16.1 / 14.4, 8 x 8 nodes 16.8 / 16.5, 4 x 12 nodes, 48 heads 22.9 / 24.4,
  // 8 x 16 nodes 25.7 / 27.3; a call's host time 18 / 14.
  const bool fuse = C <= kFuse;
  if (!fuse && !rows) return CB_ERR_ARG;
  if (!fuse) {
    const dim3 grid((unsigned)((2 * nk + nv + kThreads / 32 - 1) / (kThreads / 32)), (unsigned)C, (unsigned)R);
    cudaError_t e = dk == 128 ? cb_launch(gdn_tree_rows_kernel<128>, grid, dim3(kThreads), 0, st, a) : cb_launch(gdn_tree_rows_kernel<64>, grid, dim3(kThreads), 0, st, a);
    if (e != cudaSuccess) return (int)e;
  }
  // A head's columns are split over a cluster while all CTAs still run at once.  us of 1 / 2 / 4 CTAs a head: 16 nodes, 32 heads 21.1 / 18.0 /
  // 17.9, 128 heads 23.9 / 20.9 / 32.6, 256 heads 25.6 / 35.4 / 47.2; 64 nodes, 32 heads 49.9 / 36.0 / 30.3, 192 heads 93 (tiles) / 106.4 / 156.4.
  // Up to eight nodes the exchange costs more than it saves: 4 nodes, 32 heads 11.8 / 12.8 / 13.3 (128-wide heads; those of 64 have two CTAs throughout).
  const int64_t room = 148 / (R * nv);
  const int ns = fuse || room < 2 ? 1 : (room < 4 ? 2 : 4);
  if (fuse) return dk == 128 ? launch_gdn_tree<128, 128, 128, true>(a, (int)R, st) : launch_gdn_tree<64, 64, 32, true>(a, (int)R, st);
  if (dk == 64) return launch_gdn_tree<64, 64, 32, false>(a, (int)R, st);              // two CTAs a head
  if (ns == 1 && C > 48) return launch_gdn_tree<128, 128, 128, false, true>(a, (int)R, st);
  return ns == 1 ? launch_gdn_tree<128, 128, 128, false>(a, (int)R, st) : ns == 2 ? launch_gdn_tree<128, 128, 64, false>(a, (int)R, st) : launch_gdn_tree<128, 128, 32, false>(a, (int)R, st);
}
