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
// A CTA owns DVS columns of one head's state (columns are independent but for the norm, whose sums of squares the CTAs of a cluster
// exchange).  Everything is fp32; sums of g along a path are 64-bit, since differences of them are exponents.  Entries of the Gram
// matrices off a node's path are never multiplied, so a node's values do not reach its siblings whatever they are.
#include "sm100.cuh"

namespace {

constexpr int kRing = 16, kMaxNodes = 64, kThreads = 256;

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
  int C, Cp, nk, nv, rep, nslots, gate_sigmoid;
  float eps;
};

template <int DK, int DVS>
struct TreeSmem {                         // floats
  static constexpr int LK = DK + 4;       // rows a quarter warp reads lie in different banks
  int kn, qn, d, o, A, B, S, total;
  __host__ __device__ explicit TreeSmem(int Cp) {
    kn = 0;
    qn = kn + Cp * LK;
    d = qn + Cp * LK;
    o = d + Cp * DVS;
    A = o + Cp * DVS;
    B = A + Cp * (Cp + 4);
    S = B + Cp * (Cp + 4);
    total = S + DK * DVS;
  }
};

// x_j += sum_i m[j][i] d_i over the nodes i < i1 for eight nodes j0 .. j0 + 7 of one column; places with m = 0 are off the path
template <int DVS>
__device__ __forceinline__ void add_nodes(float* x, const float* m, int ldm, const float* d, int j0, int i1, int col) {
  for (int i = 0; i < i1; i += 4) {
    float4 w[8];
    bool any = false;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      w[j] = *reinterpret_cast<const float4*>(m + (j0 + j) * ldm + i);
      any = any || w[j].x != 0.f || w[j].y != 0.f || w[j].z != 0.f || w[j].w != 0.f;
    }
    if (!any) continue;
    float dv[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) dv[e] = d[(i + e) * DVS + col];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float f[4] = {w[j].x, w[j].y, w[j].z, w[j].w};
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (f[e] != 0.f) x[j] = fmaf(f[e], dv[e], x[j]);
    }
  }
}

template <int DK, int DV, int DVS, int NVT>
__global__ void __launch_bounds__(kThreads) gdn_tree_kernel(const GdnTreeArgs a) {
  constexpr int NS = DV / DVS, LK = TreeSmem<DK, DVS>::LK, NCH = (2 * DK + DVS) / 8;
  extern __shared__ __align__(16) float sm[];
  __shared__ uint64_t anc_s[kMaxNodes];
  __shared__ int up_s[kMaxNodes][3], depth_s[kMaxNodes];
  __shared__ double c_s[kMaxNodes];
  __shared__ float g_s[kMaxNodes], beta_s[kMaxNodes], ss_s[kMaxNodes];
  griddep_launch();
  griddep_wait();
  const int cg = blockIdx.x, h = blockIdx.y, r = blockIdx.z, kh = h / a.rep, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int slot = a.slots[r], pos0 = a.positions[r], C = a.C, Cp = a.Cp, LA = Cp + 4;
  if (slot < 0 || slot >= a.nslots || pos0 < 0) return;      // the same for the whole cluster
  const TreeSmem<DK, DVS> off(Cp);
  float *kn = sm + off.kn, *qn = sm + off.qn, *d = sm + off.d, *o = sm + off.o, *A = sm + off.A, *B = sm + off.B, *S = sm + off.S;
  const int kdim = a.nk * DK, conv = 2 * kdim + a.nv * DV, col0 = cg * DVS;

  // this CTA's columns of the state, on their way while the convolution runs
  {
    const float* sp = a.state + ((int64_t)slot * a.nv + h) * DK * DV + col0;
    for (int i = tid; i < DK * DVS / 4; i += kThreads) {
      const int k = i / (DVS / 4), c = i % (DVS / 4) * 4;
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(sm100::smem_u32(S + k * DVS + c)), "l"(sp + (int64_t)k * DV + c));
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
  if (tid < Cp) {
    uint64_t on = 0;
    if (tid < C) {
      on = (uint64_t)a.anc[(int64_t)r * C + tid];
      on = on ? (on & (~0ull >> (63 - tid))) | 1ull << tid : 0;
    }
    anc_s[tid] = on;
    depth_s[tid] = __popcll(on) - 1;
    uint64_t up = on & ~(1ull << tid);
#pragma unroll
    for (int b = 0; b < 3; ++b) {
      up_s[tid][b] = up ? 63 - __clzll((long long)up) : -1;
      if (up) up &= ~(1ull << up_s[tid][b]);
    }
    float g = 0.f, beta = 0.f;
    if (on) {
      const bf16* row = a.proj + ((int64_t)r * C + tid) * a.ldp + conv + a.nv * DV;
      const float x = __bfloat162float(row[a.nv + h]) + a.dt_bias[h];
      g = fmaxf(-expf(a.A_log[h]) * (x > 20.f ? x : log1pf(expf(x))), -1e4f);      // exp of less is 0 all the same
      beta = 1.f / (1.f + expf(-__bfloat162float(row[h])));
    }
    g_s[tid] = g;
    beta_s[tid] = beta;
  }
  __syncthreads();
  if (tid < Cp) {
    double c = 0.0;
    for (uint64_t on = anc_s[tid]; on; on &= on - 1) c += (double)g_s[__ffsll((long long)on) - 1];
    c_s[tid] = c;
  }
  // ---- convolution + SiLU: eight channels a thread, its weights in registers
  if (tid < kThreads / NCH * NCH) {
    const int ch = tid % NCH, x0 = ch * 8;
    int c;                                                   // channel in the projection row
    bool own;                                                // whose raw rows this CTA keeps
    float* to;
    int ldt;
    if (x0 < DK) { c = kh * DK + x0; own = h % a.rep == 0 && cg == 0; to = qn + x0; ldt = LK; }
    else if (x0 < 2 * DK) { c = kdim + kh * DK + x0 - DK; own = h % a.rep == 0 && cg == 0; to = kn + x0 - DK; ldt = LK; }
    else { c = 2 * kdim + h * DV + col0 + x0 - 2 * DK; own = true; to = d + x0 - 2 * DK; ldt = DVS; }
    float w[8][4];
#pragma unroll
    for (int i = 0; i < 8; ++i) *reinterpret_cast<float4*>(w[i]) = *reinterpret_cast<const float4*>(a.conv_w + (int64_t)(c + i) * 4);
    const bf16* ring = a.ring + (int64_t)slot * kRing * conv + c;
    const bf16* rows = a.proj + (int64_t)r * C * a.ldp + c;
    for (int j = tid / NCH; j < Cp; j += kThreads / NCH) {
      float y[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = 0.f;
      if (anc_s[j]) {
#pragma unroll
        for (int b = 3; b >= 0; --b) {                       // oldest tap first
          const int node = b == 0 ? j : up_s[j][b - 1], pos = pos0 + depth_s[j] - b;
          uint4 x = make_uint4(0, 0, 0, 0);
          if (node >= 0) x = *reinterpret_cast<const uint4*>(rows + (int64_t)node * a.ldp);
          else if (pos >= 0) x = *reinterpret_cast<const uint4*>(ring + (int64_t)(pos & (kRing - 1)) * conv);
          if (b == 0 && own) *reinterpret_cast<uint4*>(a.raw + ((int64_t)r * C + j) * conv + c) = x;
          float f[8];
          bf16x8_to_float(x, f);
#pragma unroll
          for (int i = 0; i < 8; ++i) y[i] = fmaf(w[i][3 - b], f[i], y[i]);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = y[i] / (1.f + expf(-y[i]));
      }
      *reinterpret_cast<float4*>(to + j * ldt) = make_float4(y[0], y[1], y[2], y[3]);
      *reinterpret_cast<float4*>(to + j * ldt + 4) = make_float4(y[4], y[5], y[6], y[7]);
    }
  }
  __syncthreads();
  // ---- norms of q and k
  for (int j = warp; j < 2 * Cp; j += kThreads / 32) {
    float* x = j < Cp ? kn + j * LK : qn + (j - Cp) * LK;
    float ss = 0.f;
    for (int i = lane; i < DK; i += 32) ss = fmaf(x[i], x[i], ss);
    float f = 1.f / sqrtf(warp_sum(ss) + 1e-6f);
    if (j >= Cp) f *= 1.f / sqrtf((float)DK);
    for (int i = lane; i < DK; i += 32) x[i] *= f;
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  __syncthreads();
  // ---- S0^T k and S0^T q: four columns and NVT of the 2 Cp vectors a thread (row v < Cp of kn, then of qn)
  {
    constexpr int CG = DVS / 4, VL = kThreads / CG;
    const int c4 = tid % CG * 4, v0 = tid / CG;
    float acc[NVT][4];
#pragma unroll
    for (int n = 0; n < NVT; ++n) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.f;
#pragma unroll 1
    for (int k = 0; k < DK; k += 4) {
      float4 s[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) s[e] = *reinterpret_cast<const float4*>(S + (k + e) * DVS + c4);
#pragma unroll
      for (int n = 0; n < NVT; ++n) {
        const int v = v0 + n * VL;
        if (v < 2 * Cp) {
          const float4 x = *reinterpret_cast<const float4*>((v < Cp ? kn + v * LK : qn + (v - Cp) * LK) + k);
          const float f[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            acc[n][0] = fmaf(f[e], s[e].x, acc[n][0]);
            acc[n][1] = fmaf(f[e], s[e].y, acc[n][1]);
            acc[n][2] = fmaf(f[e], s[e].z, acc[n][2]);
            acc[n][3] = fmaf(f[e], s[e].w, acc[n][3]);
          }
        }
      }
    }
#pragma unroll
    for (int n = 0; n < NVT; ++n) {
      const int v = v0 + n * VL, j = v < Cp ? v : v - Cp;
      if (v >= 2 * Cp) continue;
      const float f = (float)exp(c_s[j]), b = beta_s[j];
      float* x = (v < Cp ? d : o) + j * DVS + c4;
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = v < Cp ? b * (x[e] - f * acc[n][e]) : f * acc[n][e];
    }
  }
  // ---- Gram matrices: A_ji = -beta_j e^{c_j - c_i} k_j.k_i above j, B_ji = e^{c_j - c_i} q_j.k_i above j and at j; 0 elsewhere
  for (int t = tid; t < Cp * Cp / 4; t += kThreads) {        // two rows j, two columns i a thread
    const int half = Cp / 2, i0 = t % half, j0 = t / half;
    float kk[2][2] = {}, qk[2][2] = {};
    const bool low = j0 + half >= i0;
    if (low) {
      for (int k = 0; k < DK; k += 4) {
        float4 x[2], y[2], z[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          x[e] = *reinterpret_cast<const float4*>(kn + (i0 + e * half) * LK + k);
          y[e] = *reinterpret_cast<const float4*>(kn + (j0 + e * half) * LK + k);
          z[e] = *reinterpret_cast<const float4*>(qn + (j0 + e * half) * LK + k);
        }
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int v = 0; v < 2; ++v) {
            kk[u][v] += y[u].x * x[v].x + y[u].y * x[v].y + y[u].z * x[v].z + y[u].w * x[v].w;
            qk[u][v] += z[u].x * x[v].x + z[u].y * x[v].y + z[u].z * x[v].z + z[u].w * x[v].w;
          }
      }
    }
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int v = 0; v < 2; ++v) {
        const int j = j0 + u * half, i = i0 + v * half;
        const bool on = anc_s[j] >> i & 1;
        const float f = on ? (float)exp(c_s[j] - c_s[i]) : 0.f;
        A[j * LA + i] = on && i != j ? -beta_s[j] * f * kk[u][v] : 0.f;
        B[j * LA + i] = on ? f * qk[u][v] : 0.f;
      }
  }
  __syncthreads();
  // ---- d: blocks of eight nodes; what comes from earlier blocks first, then eight steps within the block.  o follows with the d's of
  // its own block.
  for (int j0 = 0; j0 < Cp; j0 += 8) {
    if (tid < DVS) {
      float x[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = d[(j0 + j) * DVS + tid];
      add_nodes<DVS>(x, A, LA, d, j0, j0, tid);
#pragma unroll
      for (int j = 1; j < 8; ++j)
#pragma unroll
        for (int i = 0; i < j; ++i) {
          const float f = A[(j0 + j) * LA + j0 + i];
          if (f != 0.f) x[j] = fmaf(f, x[i], x[j]);
        }
#pragma unroll
      for (int j = 0; j < 8; ++j) d[(j0 + j) * DVS + tid] = x[j];
    }
  }
  __syncthreads();
  for (int t = tid; t < Cp / 8 * DVS; t += kThreads) {
    const int col = t % DVS, j0 = t / DVS * 8;
    float x[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = o[(j0 + j) * DVS + col];
    add_nodes<DVS>(x, B, LA, d, j0, j0 + 8, col);
#pragma unroll
    for (int j = 0; j < 8; ++j) o[(j0 + j) * DVS + col] = x[j];
  }
  __syncthreads();
  // ---- norm over the head's columns, gate, record
  for (int j = warp; j < C; j += kThreads / 32) {
    float ss = 0.f;
    for (int i = lane; i < DVS; i += 32) ss = fmaf(o[j * DVS + i], o[j * DVS + i], ss);
    ss = warp_sum(ss);
    if (lane == 0) ss_s[j] = ss;
  }
  if (NS > 1) sm100::cluster_sync_all();
  else __syncthreads();
  for (int j = warp; j < C; j += kThreads / 32) {
    if (!anc_s[j]) continue;
    float ss = 0.f;
    if (NS > 1) {
#pragma unroll
      for (int n = 0; n < NS; ++n) {                         // the same order in every CTA
        float v;
        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(sm100::map_to_cta(sm100::smem_u32(ss_s + j), n)) : "memory");
        ss += v;
      }
    } else ss = ss_s[j];
    const float f = 1.f / sqrtf(ss / (float)DV + a.eps);
    const int64_t row = (int64_t)r * C + j;
    const bf16* z = a.proj + row * a.ldp + conv + h * DV + col0;
    float* rec = a.record + (row * a.nv + h) * (DK + DV + 1);
    for (int i = lane; i < DVS; i += 32) {
      const float x = __bfloat162float(z[i]), s = 1.f / (1.f + expf(-x));
      a.out[row * a.ldo + h * DV + col0 + i] = __float2bfloat16(o[j * DVS + i] * f * a.norm_w[col0 + i] * (a.gate_sigmoid ? s : x * s));
      rec[DK + col0 + i] = d[j * DVS + i];
    }
    if (cg == 0) {
      for (int i = lane; i < DK; i += 32) rec[i] = kn[j * LK + i];
      if (lane == 0) rec[DK + DV] = expf(g_s[j]);
    }
  }
  if (NS > 1) sm100::cluster_sync_all();                     // nobody leaves while its sums may still be read
}

template <int DK, int DV, int DVS, int NVT>
int launch_gdn_tree(const GdnTreeArgs& a, int R, cudaStream_t st) {
  auto kern = gdn_tree_kernel<DK, DV, DVS, NVT>;
  const size_t smem = TreeSmem<DK, DVS>(a.Cp).total * sizeof(float);
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return (int)e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(DV / DVS, (unsigned)a.nv, (unsigned)R);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = DV / DVS; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = g_cb_use_pdl ? 2 : 1;
  if (g_cb_trace_names) cb_trace_name((const void*)kern);
  return (int)cudaLaunchKernelEx(&cfg, kern, a);
}

template <int DK, int DV, int DVS>
int pick_nodes(const GdnTreeArgs& a, int R, cudaStream_t st) {
  constexpr int VL = kThreads / (DVS / 4);                   // vectors side by side
  const int need = (2 * a.Cp + VL - 1) / VL;
  if (need <= 1) return launch_gdn_tree<DK, DV, DVS, 1>(a, R, st);
  if (need <= 2) return launch_gdn_tree<DK, DV, DVS, 2>(a, R, st);
  if (need <= 4) return launch_gdn_tree<DK, DV, DVS, 4>(a, R, st);
  if (need <= 8) return launch_gdn_tree<DK, DV, DVS, 8>(a, R, st);
  return need <= 16 ? launch_gdn_tree<DK, DV, DVS, 16>(a, R, st) : CB_ERR_SHAPE;
}

}  // namespace

CB_EXPORT int cb_gdn_tree(const void* proj, int64_t ldp, const void* conv_w, const void* A_log, const void* dt_bias, const void* norm_w,
                          const void* ring, const void* state, const void* slots, const void* positions, const void* anc, void* out, int64_t ldo,
                          void* record, void* raw, int64_t nslots, int64_t R, int64_t C, int64_t nk, int64_t nv, int64_t dk, int64_t dv, float eps,
                          int64_t gate_sigmoid, void* stream) {
  if (!proj || !conv_w || !A_log || !dt_bias || !norm_w || !ring || !state || !slots || !positions || !anc || !out || !record || !raw) return CB_ERR_ARG;
  if (R < 1 || R > 65535 || C < 1 || C > kMaxNodes || nk < 1 || nv % nk || nv > 65535 || ldp % 8 ||
      (((uintptr_t)proj | (uintptr_t)ring | (uintptr_t)state | (uintptr_t)raw | (uintptr_t)conv_w) & 15)) return CB_ERR_SHAPE;
  GdnTreeArgs a{(const bf16*)proj, ldp, (const float*)conv_w, (const float*)A_log, (const float*)dt_bias, (const float*)norm_w, (const bf16*)ring,
                (const float*)state, (const int*)slots, (const int*)positions, (const int64_t*)anc, (bf16*)out, ldo, (float*)record, (bf16*)raw,
                (int)C, (int)((C + 7) / 8 * 8), (int)nk, (int)nv, (int)(nv / nk), (int)nslots, (int)gate_sigmoid, eps};
  cudaStream_t st = (cudaStream_t)stream;
  if (dk == 128 && dv == 128) return pick_nodes<128, 128, 64>(a, (int)R, st);
  if (dk == 64 && dv == 64) return pick_nodes<64, 64, 32>(a, (int)R, st);
  return CB_ERR_SHAPE;
}
