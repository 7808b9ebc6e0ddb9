// Attention of a tree of drafted tokens over a paged cache.
//
// A sequence has pos0 cached tokens and C <= 64 nodes behind them; node j's key and value lie at position pos0 + j, and the word
// anc[j] has bit i set where node i is an ancestor of j or j itself (0: no node, its row stays as it was).  Every node sees the whole
// cache and its own path:
//   o_j = sum_s p_js v_s / sum_s p_js,  p_js = 2^(scale q_j.k_s - m_j),  s < pos0 or s - pos0 in anc_j;  out = o_j * sigmoid(gate_j).
// The cache needs no mask but at its end, so it is a dense product of C * (nh / nkv) rows a kv head against all keys, split along the
// keys.  The nodes' own keys are few and sparse: a warp walks the set bits of a row and merges the partial sums of the splits.  A key
// that is not on a node's path is never multiplied, whatever it holds.
#include "sm100.cuh"

namespace {

constexpr int kPage = 64;
constexpr int kMaxNodes = 64;

struct TreeAttnArgs {
  const bf16* q;                          // [R * C, nh, hd] normed and rotated
  const bf16* gate; int64_t ldg;          // gate of head h at gate[row * ldg + h * 2 * hd + hd + d] (null: none)
  const void* kpool; const void* vpool;   // [slots, nkv, hd] bf16, or int8 with a scale a (slot, kv head)
  const float* kscale; const float* vscale;
  const int* tables; int64_t ldbt;        // [R, ldbt] pages
  int width, pages;                       // entries of a table; pages of the pool
  const int* positions;                   // [R] cached tokens (< 0: unused row)
  const int64_t* anc;                     // [R, C]
  bf16* out; int64_t ldo;                 // [R * C, nh * hd]
  float* part_o;                          // [R, nkv, nsplit, C * rep, hd] unnormalised sums
  float* part_ml;                         // the same rows: (maximum, sum)
  int R, C, nh, nkv, rep, nsplit;
  float scale_log2;                       // hd^-0.5 * log2(e)
};

// keys [0, n) of the cache that the table covers
__device__ __forceinline__ int cached_keys(const TreeAttnArgs& a, int r) {
  return min(a.positions[r], a.width * kPage);
}
// first slot of a page, or -1 where the table names none of the pool's
__device__ __forceinline__ int64_t page_slot(const TreeAttnArgs& a, const int* table, int page) {
  if (page >= a.width) return -1;
  const int id = table[page];
  return (unsigned)id < (unsigned)a.pages ? (int64_t)id * kPage : -1;
}

__device__ __forceinline__ void tree_ldsm(uint32_t* r, const void* p) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(sm100::smem_u32(p)));
}
__device__ __forceinline__ void tree_ldsm_t(uint32_t* r, const void* p) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(sm100::smem_u32(p)));
}
__device__ __forceinline__ void tree_mma(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// eight int8 -> eight bf16, exact
__device__ __forceinline__ uint4 q8_to_bf16(uint2 w) {
  float f[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[i] = (float)(int8_t)(w.x >> (8 * i) & 0xff);
    f[4 + i] = (float)(int8_t)(w.y >> (8 * i) & 0xff);
  }
  return float_to_bf16x8(f);
}

// One 64-key tile of one kv head into shared memory; rows behind the cache's end are zero.
template <int HD, bool Q8>
__device__ __forceinline__ void load_tile(bf16* Ks, bf16* Vs, float* ks, float* vs, const TreeAttnArgs& a, int64_t slot0, int kvh, int valid, int tid) {
  constexpr int LD = HD + 8, CPR = HD / 8;
  for (int idx = tid; idx < kPage * CPR; idx += 128) {
    const int r = idx / CPR, c = idx % CPR;
    uint4 k = make_uint4(0, 0, 0, 0), v = k;
    if (r < valid) {
      const int64_t at = ((slot0 + r) * a.nkv + kvh) * HD + c * 8;
      if (Q8) {
        k = q8_to_bf16(*reinterpret_cast<const uint2*>((const int8_t*)a.kpool + at));
        v = q8_to_bf16(*reinterpret_cast<const uint2*>((const int8_t*)a.vpool + at));
      } else {
        k = *reinterpret_cast<const uint4*>((const bf16*)a.kpool + at);
        v = *reinterpret_cast<const uint4*>((const bf16*)a.vpool + at);
      }
    }
    *reinterpret_cast<uint4*>(Ks + r * LD + c * 8) = k;
    *reinterpret_cast<uint4*>(Vs + r * LD + c * 8) = v;
  }
  if (Q8 && tid < kPage) {
    const int64_t row = (slot0 + tid) * a.nkv + kvh;
    ks[tid] = tid < valid ? a.kscale[row] : 0.f;
    vs[tid] = tid < valid ? a.vscale[row] : 0.f;
  }
}

// The cache: 64 rows (node, head of the group) a CTA, four warps of 16, one split of the pages.  The keys' scales of an int8 pool
// multiply the scores, the values' the weights, so both products take the codes as they are.
template <int HD, bool Q8>
__global__ void __launch_bounds__(128) tree_cache_kernel(const TreeAttnArgs a) {
  constexpr int LD = HD + 8, CPR = HD / 8;
  extern __shared__ __align__(16) unsigned char smem_raw[];
  bf16* Qs = reinterpret_cast<bf16*>(smem_raw);
  bf16* Ks = Qs + 64 * LD;
  bf16* Vs = Ks + 64 * LD;
  __shared__ float ks[kPage], vs[kPage];
  griddep_launch();
  griddep_wait();
  const int split = blockIdx.x, kvh = blockIdx.y % a.nkv, row0 = (blockIdx.y / a.nkv) * 64, r = blockIdx.z;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, tq = lane & 3;
  const int rows = a.C * a.rep, keys = cached_keys(a, r);
  const int64_t pr0 = (((int64_t)r * a.nkv + kvh) * a.nsplit + split) * rows;
  const int tiles = (max(keys, 0) + kPage - 1) / kPage, per = (tiles + a.nsplit - 1) / a.nsplit;
  const int t0 = split * per, t1 = min(tiles, t0 + per);
  if (t0 >= t1) {
    for (int i = tid; i < 64 && row0 + i < rows; i += 128) {
      a.part_ml[(pr0 + row0 + i) * 2] = -INFINITY;
      a.part_ml[(pr0 + row0 + i) * 2 + 1] = 0.f;
    }
    return;
  }
  const int* table = a.tables + (int64_t)r * a.ldbt;
  for (int idx = tid; idx < 64 * CPR; idx += 128) {
    const int i = idx / CPR, c = idx % CPR, row = row0 + i;
    uint4 v = make_uint4(0, 0, 0, 0);
    if (row < rows)
      v = *reinterpret_cast<const uint4*>(a.q + (((int64_t)r * a.C + row / a.rep) * a.nh + kvh * a.rep + row % a.rep) * HD + c * 8);
    *reinterpret_cast<uint4*>(Qs + i * LD + c * 8) = v;
  }
  float o[HD / 8][4];
#pragma unroll
  for (int n = 0; n < HD / 8; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
  float mrow[2] = {-INFINITY, -INFINITY}, lrow[2] = {0.f, 0.f};
  for (int kt = t0; kt < t1; ++kt) {
    const int64_t slot0 = page_slot(a, table, kt);
    const int valid = slot0 < 0 ? 0 : min(kPage, keys - kt * kPage);
    __syncthreads();
    load_tile<HD, Q8>(Ks, Vs, ks, vs, a, slot0, kvh, valid, tid);
    __syncthreads();
    if (valid == 0 || row0 + warp * 16 >= rows) continue;
    float s[8][4];
#pragma unroll
    for (int n = 0; n < 8; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll 4
    for (int kk = 0; kk < HD / 16; ++kk) {
      uint32_t af[4];
      tree_ldsm(af, Qs + (warp * 16 + (lane & 15)) * LD + kk * 16 + (lane >> 4) * 8);
#pragma unroll
      for (int np = 0; np < 4; ++np) {
        uint32_t b[4];
        tree_ldsm(b, Ks + (np * 16 + (lane & 7) + ((lane >> 4) << 3)) * LD + kk * 16 + ((lane >> 3) & 1) * 8);
        tree_mma(s[2 * np], af, b[0], b[1]);
        tree_mma(s[2 * np + 1], af, b[2], b[3]);
      }
    }
    float mnew[2] = {mrow[0], mrow[1]};
#pragma unroll
    for (int n = 0; n < 8; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int key = n * 8 + tq * 2 + (e & 1);
        const float f = Q8 ? a.scale_log2 * ks[key] : a.scale_log2;
        s[n][e] = key < valid ? s[n][e] * f : -INFINITY;
        mnew[e >> 1] = fmaxf(mnew[e >> 1], s[n][e]);
      }
    float corr[2], msafe[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      mnew[i] = fmaxf(mnew[i], __shfl_xor_sync(0xffffffffu, mnew[i], 1));
      mnew[i] = fmaxf(mnew[i], __shfl_xor_sync(0xffffffffu, mnew[i], 2));
      msafe[i] = mnew[i] == -INFINITY ? 0.f : mnew[i];
      corr[i] = exp2f(mrow[i] - msafe[i]);
      mrow[i] = mnew[i];
    }
    uint32_t pf[4][4];
    float lsum[2] = {0.f, 0.f};
#pragma unroll
    for (int n = 0; n < 8; ++n) {
      float p[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        p[e] = exp2f(s[n][e] - msafe[e >> 1]);
        lsum[e >> 1] += p[e];
        if (Q8) p[e] *= vs[n * 8 + tq * 2 + (e & 1)];
      }
      pf[n >> 1][(n & 1) * 2] = pack_bf162(p[0], p[1]);          // weights rounded to bf16, half a step 2^-9; their sum is not
      pf[n >> 1][(n & 1) * 2 + 1] = pack_bf162(p[2], p[3]);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) lrow[i] = lrow[i] * corr[i] + lsum[i];
#pragma unroll
    for (int n = 0; n < HD / 8; ++n) {
      o[n][0] *= corr[0]; o[n][1] *= corr[0]; o[n][2] *= corr[1]; o[n][3] *= corr[1];
    }
#pragma unroll
    for (int kk = 0; kk < 4; ++kk)
#pragma unroll
      for (int np = 0; np < HD / 16; ++np) {
        uint32_t b[4];
        tree_ldsm_t(b, Vs + (kk * 16 + (lane & 15)) * LD + np * 16 + (lane >> 4) * 8);
        tree_mma(o[2 * np], pf[kk], b[0], b[1]);
        tree_mma(o[2 * np + 1], pf[kk], b[2], b[3]);
      }
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    lrow[i] += __shfl_xor_sync(0xffffffffu, lrow[i], 1);
    lrow[i] += __shfl_xor_sync(0xffffffffu, lrow[i], 2);
    const int row = row0 + warp * 16 + g + i * 8;
    if (row >= rows) continue;
    float* po = a.part_o + (pr0 + row) * HD;
#pragma unroll
    for (int n = 0; n < HD / 8; ++n)
      *reinterpret_cast<float2*>(po + n * 8 + tq * 2) = make_float2(o[n][i * 2], o[n][i * 2 + 1]);
    if (tq == 0) *reinterpret_cast<float2*>(a.part_ml + (pr0 + row) * 2) = make_float2(mrow[i], lrow[i]);
  }
}

// A warp a (node, head): the node's path, then the splits' partial sums, the gate and the store.  Lanes own hd / 32 channels.
template <int HD, bool Q8>
__global__ void __launch_bounds__(256) tree_finish_kernel(const TreeAttnArgs a) {
  constexpr int EPL = HD / 32;
  griddep_launch();
  griddep_wait();
  const int64_t task = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (task >= (int64_t)a.R * a.C * a.nh) return;
  const int h = (int)(task % a.nh), j = (int)(task / a.nh % a.C), r = (int)(task / ((int64_t)a.nh * a.C));
  const int pos0 = a.positions[r];
  uint64_t on = (uint64_t)a.anc[(int64_t)r * a.C + j];
  if (on == 0 || pos0 < 0) return;
  on = (on & (~0ull >> (63 - j))) | 1ull << j;              // a path ends at its node
  const int kvh = h / a.rep;
  const int* table = a.tables + (int64_t)r * a.ldbt;
  const int64_t row = (int64_t)r * a.C + j;
  float q[EPL], o[EPL], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int e = 0; e < EPL; ++e) {
    q[e] = __bfloat162float(a.q[(row * a.nh + h) * HD + lane * EPL + e]) * a.scale_log2;
    o[e] = 0.f;
  }
  while (on) {
    const int i = __ffsll((long long)on) - 1;
    on &= on - 1;
    const int p = pos0 + i;
    const int64_t slot0 = page_slot(a, table, p / kPage);
    if (slot0 < 0) continue;
    const int64_t kr = (slot0 + p % kPage) * a.nkv + kvh;
    float k[EPL], v[EPL];
#pragma unroll
    for (int e = 0; e < EPL; ++e) {
      const int64_t at = kr * HD + lane * EPL + e;
      k[e] = Q8 ? (float)((const int8_t*)a.kpool)[at] * a.kscale[kr] : __bfloat162float(((const bf16*)a.kpool)[at]);
      v[e] = Q8 ? (float)((const int8_t*)a.vpool)[at] * a.vscale[kr] : __bfloat162float(((const bf16*)a.vpool)[at]);
    }
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < EPL; ++e) s = fmaf(q[e], k[e], s);
    s = warp_sum(s);
    const float mn = fmaxf(m, s), ms = mn == -INFINITY ? 0.f : mn, c = exp2f(m - ms), w = exp2f(s - ms);
    m = mn;
    l = l * c + w;
#pragma unroll
    for (int e = 0; e < EPL; ++e) o[e] = o[e] * c + w * v[e];
  }
  const int rows = a.C * a.rep;
  for (int sp = 0; sp < a.nsplit; ++sp) {
    const int64_t pr = (((int64_t)r * a.nkv + kvh) * a.nsplit + sp) * rows + j * a.rep + h % a.rep;
    const float2 ml = *reinterpret_cast<const float2*>(a.part_ml + pr * 2);
    if (ml.x == -INFINITY) continue;                        // nothing in this split (its sums were not written)
    const float mn = fmaxf(m, ml.x), c = exp2f(m - mn), w = exp2f(ml.x - mn);
    m = mn;
    l = l * c + ml.y * w;
#pragma unroll
    for (int e = 0; e < EPL; ++e) o[e] = o[e] * c + w * a.part_o[pr * HD + lane * EPL + e];
  }
  const float inv = l > 0.f ? 1.f / l : 0.f;
  const bf16* gp = a.gate ? a.gate + row * a.ldg + (int64_t)h * 2 * HD + HD + lane * EPL : nullptr;
  bf16* op = a.out + row * a.ldo + (int64_t)h * HD + lane * EPL;
#pragma unroll
  for (int e = 0; e < EPL; ++e) op[e] = __float2bfloat16(o[e] * inv * (gp ? sigmoid_f(__bfloat162float(gp[e])) : 1.f));
}

template <int HD, bool Q8>
int launch_tree(const TreeAttnArgs& a, cudaStream_t st) {
  const size_t smem = (size_t)3 * 64 * (HD + 8) * sizeof(bf16);
  auto kern = tree_cache_kernel<HD, Q8>;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return (int)e;
  const int rows = a.C * a.rep;
  const dim3 grid((unsigned)a.nsplit, (unsigned)(a.nkv * ((rows + 63) / 64)), (unsigned)a.R);
  e = cb_launch(kern, grid, dim3(128), smem, st, a);
  if (e != cudaSuccess) return (int)e;
  const int64_t tasks = (int64_t)a.R * a.C * a.nh;
  return (int)cb_launch(tree_finish_kernel<HD, Q8>, dim3((unsigned)((tasks + 7) / 8)), dim3(256), 0, st, a);
}

}  // namespace

CB_EXPORT int cb_attn_tree(const void* q, const void* gate, int64_t ldg, const void* kpool, const void* vpool, int64_t slots,
                           const void* kscale, const void* vscale, const void* tables, int64_t ldbt, int64_t width, const void* positions,
                           const void* anc, void* out, int64_t ldo, void* part, int64_t R, int64_t C, int64_t nh, int64_t nkv, int64_t hd,
                           int64_t nsplit, void* stream) {
  if (!q || !kpool || !vpool || !tables || !positions || !anc || !out || !part) return CB_ERR_ARG;
  if ((kscale == nullptr) != (vscale == nullptr)) return CB_ERR_ARG;
  if (R < 1 || R > 65535 || C < 1 || C > kMaxNodes || nkv < 1 || nh % nkv || nsplit < 1 || width < 1) return CB_ERR_SHAPE;
  TreeAttnArgs a{(const bf16*)q, (const bf16*)gate, ldg, kpool, vpool, (const float*)kscale, (const float*)vscale, (const int*)tables, ldbt,
                 (int)width, (int)(slots / kPage), (const int*)positions, (const int64_t*)anc, (bf16*)out, ldo,
                 (float*)part + 2 * R * nh * C * nsplit, (float*)part, (int)R, (int)C, (int)nh, (int)nkv, (int)(nh / nkv), (int)nsplit,
                 1.4426950408889634f / sqrtf((float)hd)};
  cudaStream_t st = (cudaStream_t)stream;
  if (hd == 256) return kscale ? launch_tree<256, true>(a, st) : launch_tree<256, false>(a, st);
  if (hd == 128) return kscale ? launch_tree<128, true>(a, st) : launch_tree<128, false>(a, st);
  if (hd == 64) return kscale ? launch_tree<64, true>(a, st) : launch_tree<64, false>(a, st);
  return CB_ERR_SHAPE;
}
