// Commit of an accepted path: what a tree of drafted tokens left behind becomes the sequence's own.
//
// Nodes of a tree keep their keys and values at position pos0 + node; the path's rows move to pos0 + step.  path[i] >= i (parents come
// before children), so a row is never written before it is read if all reads of a batch of steps come before its writes.  The
// recurrent states advance by the recorded rank-one updates of the path, S <- alpha S + k d^T, and the convolution ring takes the
// path's raw rows.  All layers go in one launch; both kernels are bound by the bytes they move.
#include "common.cuh"

namespace {

constexpr int kPage = 64, kRing = 16;

struct KvCommitArgs {
  unsigned char* pool[2];                 // [L, slots, row_bytes]: keys, values
  float* scale[2];                        // int8: [L, slots, nkv] (null: none)
  const int* tables; int64_t ldbt;
  const int* positions; const int* path; const int* steps;
  int64_t slots;
  int width, C, nkv, chunks;              // chunks: 16-byte pieces of a row
};

__global__ void __launch_bounds__(256) kv_tree_commit_kernel(const KvCommitArgs a) {
  griddep_launch();
  griddep_wait();
  const int r = blockIdx.y, l = blockIdx.z, pos0 = a.positions[r], n = min(a.steps[r], a.C);
  if (pos0 < 0 || n < 2) return;
  const int* table = a.tables + (int64_t)r * a.ldbt;
  const int* path = a.path + (int64_t)r * a.C;
  auto slot = [&](unsigned p) -> int64_t {                  // a position behind the cache may pass 2^31
    if (p / kPage >= (unsigned)a.width) return -1;
    const int64_t s = (int64_t)table[p / kPage] * kPage + p % kPage;
    return s >= 0 && s < a.slots ? s : -1;
  };
  const int t = blockIdx.x * blockDim.x + threadIdx.x, which = t & 1, c = t >> 1;
  const bool scales = c >= a.chunks;
  if (scales && (c - a.chunks >= a.nkv || !a.scale[which])) return;
  constexpr int B = 8;
  for (int i0 = 1; i0 < n; i0 += B) {
    uint4 v[B];
    int64_t to[B];
#pragma unroll
    for (int i = 0; i < B; ++i) {
      const int step = i0 + i, node = step < n ? path[step] : -1;
      to[i] = -1;
      if (node <= step || node >= a.C) continue;           // in place already (or no node)
      const int64_t from = slot((unsigned)pos0 + node);
      to[i] = from < 0 ? -1 : slot((unsigned)pos0 + step);
      if (to[i] < 0) continue;
      if (scales) v[i].x = __float_as_uint(a.scale[which][(l * a.slots + from) * a.nkv + c - a.chunks]);
      else v[i] = *reinterpret_cast<const uint4*>(a.pool[which] + ((l * a.slots + from) * a.chunks + c) * 16);
    }
#pragma unroll
    for (int i = 0; i < B; ++i) {
      if (to[i] < 0) continue;
      if (scales) a.scale[which][(l * a.slots + to[i]) * a.nkv + c - a.chunks] = __uint_as_float(v[i].x);
      else *reinterpret_cast<uint4*>(a.pool[which] + ((l * a.slots + to[i]) * a.chunks + c) * 16) = v[i];
    }
  }
}

struct GdnCommitArgs {
  float* state;                           // [L, slots, nv, dk, dv]
  bf16* ring;                             // [L, slots, 16, conv]
  const float* record;                    // [L, R, C, nv, dk + dv + 1]: k, d, alpha
  const bf16* raw;                        // [L, R, C, conv]
  const int* from; const int* to;         // [R] slots (< 0: unused row)
  const int* positions; const int* path; const int* steps;
  int slots, R, C, nv, conv, ring_blocks;
};

// A CTA takes one head's state: a warp a few rows of it, four columns a lane, in registers.  The path's records come through shared memory,
// kSteps at a time.  8 sequences of 32 heads in 24 layers, five steps: 805 MB of states in 181 us.  (Records read from global memory by every
// thread: 215 us.)
constexpr int kSteps = 16;

template <int D>
__global__ void __launch_bounds__(D * D / 32) gdn_tree_commit_kernel(const GdnCommitArgs a) {
  constexpr int LANES = D / 4, ROWS = 8, REC = 2 * D + 1, NT = D * D / 32;       // a thread: ROWS rows, four columns
  __shared__ __align__(16) float k_s[kSteps][D], d_s[kSteps][D];
  __shared__ float alpha_s[kSteps];
  griddep_launch();
  griddep_wait();
  const int r = blockIdx.y, l = blockIdx.z, src = a.from[r], dst = a.to[r], n = min(a.steps[r], a.C), pos0 = a.positions[r], tid = threadIdx.x;
  if (src < 0 || dst < 0 || src >= a.slots || dst >= a.slots || pos0 < 0 || n < 0) return;
  const int* path = a.path + (int64_t)r * a.C;
  const int64_t row = (int64_t)l * a.R + r;
  if ((int)blockIdx.x >= a.nv) {                            // ring: entry e holds the last position that is e modulo 16
    const bf16* in = a.ring + ((int64_t)l * a.slots + src) * kRing * a.conv;
    bf16* out = a.ring + ((int64_t)l * a.slots + dst) * kRing * a.conv;
    const int last = pos0 + n - 1, per = a.conv / 8;
#pragma unroll 4
    for (int i = (blockIdx.x - a.nv) * NT + tid; i < kRing * per; i += a.ring_blocks * NT) {
      const int e = i / per, c = i % per * 8, step = last - ((last - e) & (kRing - 1)) - pos0;
      const int node = step >= 0 && step < n ? path[step] : -1;
      if (node >= 0 && node < a.C) *reinterpret_cast<uint4*>(out + (int64_t)e * a.conv + c) = *reinterpret_cast<const uint4*>(a.raw + (row * a.C + node) * a.conv + c);
      else if (src != dst) *reinterpret_cast<uint4*>(out + (int64_t)e * a.conv + c) = *reinterpret_cast<const uint4*>(in + (int64_t)e * a.conv + c);
    }
    return;
  }
  if (n == 0 && src == dst) return;
  const int h = blockIdx.x, k0 = tid / LANES * ROWS, c = tid % LANES * 4;
  const int64_t at = (int64_t)h * D * D + k0 * D + c;
  const float* sp = a.state + ((int64_t)l * a.slots + src) * a.nv * D * D + at;
  float4 s[ROWS];
#pragma unroll
  for (int i = 0; i < ROWS; ++i) s[i] = *reinterpret_cast<const float4*>(sp + i * D);
#pragma unroll 1
  for (int t0 = 0; t0 < n; t0 += kSteps) {
    const int here = min(kSteps, n - t0);
    if (t0) __syncthreads();
#pragma unroll 1
    for (int i = tid; i < here * REC; i += NT) {
      const int t = i / REC, x = i % REC, node = path[t0 + t];
      const bool ok = node >= 0 && node < a.C;              // no node: nothing is added, nothing decays
      const float v = ok ? a.record[((row * a.C + node) * a.nv + h) * REC + x] : (x == 2 * D ? 1.f : 0.f);
      if (x < D) k_s[t][x] = v;
      else if (x < 2 * D) d_s[t][x - D] = v;
      else alpha_s[t] = v;
    }
    __syncthreads();
#pragma unroll 1
    for (int t = 0; t < here; ++t) {
      const float4 d = *reinterpret_cast<const float4*>(d_s[t] + c);
      const float alpha = alpha_s[t];
#pragma unroll
      for (int i = 0; i < ROWS; i += 4) {
        const float4 k = *reinterpret_cast<const float4*>(k_s[t] + k0 + i);
        const float f[4] = {k.x, k.y, k.z, k.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float4& x = s[i + e];
          x.x = fmaf(f[e], d.x, alpha * x.x);
          x.y = fmaf(f[e], d.y, alpha * x.y);
          x.z = fmaf(f[e], d.z, alpha * x.z);
          x.w = fmaf(f[e], d.w, alpha * x.w);
        }
      }
    }
  }
  float* op = a.state + ((int64_t)l * a.slots + dst) * a.nv * D * D + at;
#pragma unroll
  for (int i = 0; i < ROWS; ++i) *reinterpret_cast<float4*>(op + i * D) = s[i];
}

}  // namespace

CB_EXPORT int cb_kv_tree_commit(void* kpool, void* vpool, void* kscale, void* vscale, const void* tables, int64_t ldbt, int64_t width,
                                const void* positions, const void* path, const void* steps, int64_t L, int64_t slots, int64_t row_bytes,
                                int64_t nkv, int64_t R, int64_t C, void* stream) {
  if (!kpool || !vpool || !tables || !positions || !path || !steps || (kscale == nullptr) != (vscale == nullptr)) return CB_ERR_ARG;
  if (row_bytes % 16 || row_bytes < 16 || L < 1 || L > 65535 || R < 1 || R > 65535 || C < 1 || width < 1 || (((uintptr_t)kpool | (uintptr_t)vpool) & 15)) return CB_ERR_SHAPE;
  KvCommitArgs a{{(unsigned char*)kpool, (unsigned char*)vpool}, {(float*)kscale, (float*)vscale}, (const int*)tables, ldbt, (const int*)positions,
                 (const int*)path, (const int*)steps, slots, (int)width, (int)C, (int)nkv, (int)(row_bytes / 16)};
  const int64_t threads = 2 * (row_bytes / 16 + (kscale ? nkv : 0));
  return (int)cb_launch(kv_tree_commit_kernel, dim3((unsigned)((threads + 255) / 256), (unsigned)R, (unsigned)L), dim3(256), 0, (cudaStream_t)stream, a);
}

CB_EXPORT int cb_gdn_tree_commit(void* state, void* ring, const void* record, const void* raw, const void* from, const void* to,
                                 const void* positions, const void* path, const void* steps, int64_t L, int64_t slots, int64_t R, int64_t C,
                                 int64_t nv, int64_t dk, int64_t dv, int64_t conv, void* stream) {
  if (!state || !ring || !record || !raw || !from || !to || !positions || !path || !steps) return CB_ERR_ARG;
  if (L < 1 || L > 65535 || R < 1 || R > 65535 || C < 1 || conv % 8 || (((uintptr_t)state | (uintptr_t)ring | (uintptr_t)raw) & 15)) return CB_ERR_SHAPE;
  const int ring_blocks = 4;
  GdnCommitArgs a{(float*)state, (bf16*)ring, (const float*)record, (const bf16*)raw, (const int*)from, (const int*)to, (const int*)positions,
                  (const int*)path, (const int*)steps, (int)slots, (int)R, (int)C, (int)nv, (int)conv, ring_blocks};
  const dim3 grid((unsigned)(nv + ring_blocks), (unsigned)R, (unsigned)L);
  if (dk == 128 && dv == 128) return (int)cb_launch(gdn_tree_commit_kernel<128>, grid, dim3(512), 0, (cudaStream_t)stream, a);
  if (dk == 64 && dv == 64) return (int)cb_launch(gdn_tree_commit_kernel<64>, grid, dim3(128), 0, (cudaStream_t)stream, a);
  return CB_ERR_SHAPE;
}
