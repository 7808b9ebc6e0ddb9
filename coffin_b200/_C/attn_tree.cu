// Attention of a tree of drafted tokens over a paged cache.
//
// A sequence has pos0 cached tokens and C <= 64 nodes behind them; node j's key and value lie at position pos0 + j, and the word
// anc[j] has bit i set where node i is an ancestor of j or j itself (0: no node, its row stays as it was).  Every node sees the whole
// cache and its own path:
//   o_j = sum_s p_js v_s / sum_s p_js,  p_js = 2^(scale q_j.k_s - m_j),  s < pos0 or s - pos0 in anc_j;  out = o_j * sigmoid(gate_j).
// The cache needs no mask but at its end, so it is a dense product of C * (nh / nkv) rows a kv head against all keys.  The nodes' own
// keys are few and sparse: a warp walks the set bits of a row and merges the partial sums of the cache.  A key that is not on a node's
// path is never multiplied, whatever it holds, and values behind the cache's end are cleared before they are.
//
// Cache kernel: an item is (sequence, kv head, 128 rows); the pages of all items form one list that the CTAs, one an SM, cut into even
// pieces, whatever the lengths.  A CTA walks the segments of its piece; each leaves unnormalised sums, maxima and sums of weights in
// slot (CTA + item), which is different for any two segments because one of the two grows from segment to segment.
//   warp 0       TMA: K and V pages into rings (a page of a kv head is a [64 x hd] box of the pool, hd / 64 swizzled [64 x 128 B] blocks)
//   warp 1, 10   tcgen05.mma (one thread each): S = Q K^T with Q in tensor memory into one of two accumulators; O += P V
//   warps 2-9    the segment's Q rows into tensor memory, then the softmax, two threads a row, and the sums out of tensor memory.  The
//                reference maximum of a row is raised, and O rescaled, only when its maximum has grown by more than 2^8.
//   warps 11-14  int8 pools, in TMA's place: pages as codes into registers a page ahead, as exact bf16 into the rings.  The keys' scales
//                multiply the scores, the values' the weights.
// Every wait is bounded by 2 s and reports through the status word; tensor memory is freed on every path.
#include "sm100.cuh"

namespace {
using namespace sm100;

constexpr int kPage = 64, kRows = 128, kMaxNodes = 64;

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
  float* part_o;                          // [ctas + items, used rows, hd] unnormalised sums
  float* part_ml;                         // the same rows: (reference maximum, sum)
  int R, C, nh, nkv, rep, tiles, used, ctas;   // tiles: of 128 rows a (sequence, kv head); used: rows of a slot
  float scale_log2;                       // hd^-0.5 * log2(e)
  int* status;
};

__device__ __forceinline__ int cached_keys(const TreeAttnArgs& a, int r) { return max(0, min(a.positions[r], a.width * kPage)); }
__device__ __forceinline__ int cached_pages(const TreeAttnArgs& a, int r) { return (cached_keys(a, r) + kPage - 1) / kPage; }
// first slot of a page, or -1 where the table names none of the pool's
__device__ __forceinline__ int64_t page_slot(const TreeAttnArgs& a, int r, int page) {
  if (page >= a.width) return -1;
  const int id = a.tables[(int64_t)r * a.ldbt + page];
  return (unsigned)id < (unsigned)a.pages ? (int64_t)id * kPage : -1;
}
// The list of all items' pages, cut into even pieces: piece b is [b T / G, (b + 1) T / G).
__device__ __forceinline__ int64_t piece_start(int64_t b, int64_t T, int G) { return b * T / G; }
__device__ __forceinline__ int piece_of(int64_t g, int64_t T, int G) { return (int)(((g + 1) * G - 1) / T); }
// pages of one item of every sequence before `r`, and of all sequences (a warp)
__device__ __forceinline__ void page_sums(const TreeAttnArgs& a, int r, int64_t* before, int64_t* all) {
  const int lane = threadIdx.x & 31;
  int64_t b = 0, t = 0;
  for (int i = lane; i < a.R; i += 32) {
    const int n = cached_pages(a, i);
    t += n;
    if (i < r) b += n;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    b += __shfl_xor_sync(0xffffffffu, b, o);
    t += __shfl_xor_sync(0xffffffffu, t, o);
  }
  *before = b;
  *all = t;
}

// Segments of a CTA's piece, one after the other.
struct Segments {
  int64_t g, end, start;                  // next page of the list, end of the piece, first page of sequence r
  int r, n;                               // sequence, pages of one of its items
  int kvh, tile, p0, p1, item;            // the segment: pages [p0, p1) of an item
  __device__ __forceinline__ bool next(const TreeAttnArgs& a) {
    if (g >= end) return false;
    const int per = a.nkv * a.tiles;
    while (g >= start + (int64_t)n * per) {
      start += (int64_t)n * per;
      n = cached_pages(a, ++r);
    }
    const int64_t at = g - start;
    const int it = (int)(at / n);
    p0 = (int)(at - (int64_t)it * n);
    p1 = (int)min((int64_t)n, p0 + (end - g));
    kvh = it / a.tiles;
    tile = it % a.tiles;
    item = r * per + it;
    g += p1 - p0;
    return true;
  }
};

__device__ __forceinline__ uint64_t tree_now() {
  uint64_t t;
  asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
  return t;
}
__device__ __forceinline__ bool tree_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  if (mbar_try(bar, parity)) return true;
  const uint64_t t0 = tree_now();
  for (;;) {
    for (int i = 0; i < 128; ++i)
      if (mbar_try(bar, parity)) return true;
    if (*abort_flag) return false;
    if (tree_now() - t0 > 2000000000ull) return false;
  }
}
__device__ __forceinline__ float tree_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// four int8 codes (as x + 128 in a word) -> two words of bf16, exact
__device__ __forceinline__ uint2 codes_to_bf16(uint32_t w) {
  float f[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) f[i] = __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7650 + i)) - 8388736.f;
  return make_uint2(pack_bf162(f[0], f[1]), pack_bf162(f[2], f[3]));
}

// Stages of the rings.  int8: the next page waits in registers, and the scales need room too.
template <int HD, bool Q8> struct TreeRing { static constexpr int stages = HD == 256 ? (Q8 ? 2 : 3) : HD == 128 ? 4 : 6; };

template <int HD, bool Q8>
__global__ void __launch_bounds__(Q8 ? 480 : 352, 1)
tree_cache_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const TreeAttnArgs a) {
  constexpr int NC = HD / 64, ST = TreeRing<HD, Q8>::stages;
  constexpr int KC = kPage * 128, KV_BYTES = kPage * HD * 2, P_BYTES = kRows * kPage * 2;
  constexpr uint32_t TMEM_COLS = 2 * kPage + HD + HD / 2 <= 256 ? 256 : 512;
  constexpr uint32_t IDESC_S = umma_idesc(kRows, kPage, 1, 1);
  constexpr uint32_t IDESC_O = umma_idesc(kRows, HD, 1, 1) | (1u << 16);     // B operand MN-major
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* Ks = smem_raw;                       // the swizzle wants 1024-byte blocks; there is no room to round up
  unsigned char* Vs = Ks + ST * KV_BYTES;
  unsigned char* Ps = Vs + ST * KV_BYTES;             // [2][P_BYTES]
  __shared__ uint64_t q_full, k_full[ST], v_full[ST], k_free[ST], v_free[ST], s_full[2], s_free[2], p_full[2], p_free[2], o_full, o_free,
      pair_bar[4];
  __shared__ float xch[2][2][kRows];                  // [page parity][half][row] maxima
  __shared__ float lx[kRows];
  __shared__ float scales[Q8 ? ST : 1][2][kPage];
  __shared__ Segments seg_s;
  __shared__ uint32_t tmem_base_s;
  __shared__ int abort_s;
  volatile int* abort_flag = &abort_s;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  griddep_launch();
  griddep_wait();
  if (smem_u32(smem_raw) & 1023) {
    if (threadIdx.x == 0) atomicCAS(a.status, 0, 89);
    return;
  }
  if (warp == 0) {
    int64_t none, all;
    page_sums(a, 0, &none, &all);
    const int per = a.nkv * a.tiles;
    const int64_t T = all * per, lo = piece_start(blockIdx.x, T, a.ctas), hi = piece_start(blockIdx.x + 1, T, a.ctas);
    int64_t start = 0;
    int r = 0;
    if (lo < hi)                                      // the sequence of the first page: 32 sequences at a time
      for (;; r += 32) {
        const int64_t n = r + lane < a.R ? (int64_t)cached_pages(a, r + lane) * per : 0;
        int64_t incl = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int64_t x = __shfl_up_sync(0xffffffffu, incl, o);
          if (lane >= o) incl += x;
        }
        const unsigned hit = __ballot_sync(0xffffffffu, start + incl > lo);
        if (hit) {
          const int f = __ffs(hit) - 1;
          start += __shfl_sync(0xffffffffu, incl - n, f);
          r += f;
          break;
        }
        start += __shfl_sync(0xffffffffu, incl, 31);
      }
    if (lane == 0) {
      seg_s.g = lo; seg_s.end = hi; seg_s.start = start; seg_s.r = r; seg_s.n = lo < hi ? cached_pages(a, r) : 0;
      abort_s = 0;
      mbar_init(&q_full, 8);
      mbar_init(&o_full, 1);
      mbar_init(&o_free, 8);
      for (int i = 0; i < ST; ++i) {
        mbar_init(&k_full[i], Q8 ? 128 : 1); mbar_init(&v_full[i], Q8 ? 128 : 1); mbar_init(&k_free[i], 1); mbar_init(&v_free[i], 1);
      }
      for (int i = 0; i < 2; ++i) {
        mbar_init(&s_full[i], 1); mbar_init(&s_free[i], 8); mbar_init(&p_full[i], 8); mbar_init(&p_free[i], 1);
      }
      for (int i = 0; i < 4; ++i) mbar_init(&pair_bar[i], 64);
      mbar_fence_init();
    }
  }
  __syncthreads();
  Segments seg = seg_s;
  if (seg.g >= seg.end) return;                       // no page for this CTA
  if (warp == 1) {
    tmem_alloc(&tmem_base_s, TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = tmem_base_s, tmem_o = tmem_base + 2 * kPage, tmem_q = tmem_o + HD;       // S0 | S1 | O | Q
  auto give_up = [&](int code) { atomicCAS(a.status, 0, code); abort_s = 1; };

  if (warp == 0) {
    // ------------------------------------ TMA producer ------------------------------------------
    if (!Q8 && lane == 0) {
      int n = 0;
      while (seg.next(a) && !*abort_flag)
        for (int p = seg.p0; p < seg.p1; ++p, ++n) {
          const int s = n % ST;
          const uint32_t ph = (n / ST) & 1;
          const int64_t slot0 = page_slot(a, seg.r, p);
          if (!tree_wait(&k_free[s], ph ^ 1, abort_flag)) { give_up(90); break; }
          if (slot0 < 0) mbar_arrive(&k_full[s]);     // no such page: its scores are masked, its values cleared
          else {
            mbar_expect_tx(&k_full[s], KV_BYTES);
            for (int c = 0; c < NC; ++c) tma_load_2d(Ks + s * KV_BYTES + c * KC, &tmK, &k_full[s], seg.kvh * HD + c * 64, (int)slot0);
          }
          if (!tree_wait(&v_free[s], ph ^ 1, abort_flag)) { give_up(91); break; }
          if (slot0 < 0) mbar_arrive(&v_full[s]);
          else {
            mbar_expect_tx(&v_full[s], KV_BYTES);
            for (int c = 0; c < NC; ++c) tma_load_2d(Vs + s * KV_BYTES + c * KC, &tmV, &v_full[s], seg.kvh * HD + c * 64, (int)slot0);
          }
        }
    }
  } else if (warp == 1) {
    // ------------------------------------ S = Q K^T ----------------------------------------------
    if (lane == 0) {
      int n = 0;
      bool ok = true;
      for (int sg = 0; ok && seg.next(a); ++sg) {
        if (!tree_wait(&q_full, sg & 1, abort_flag)) { give_up(92); break; }
        tc_fence_after();
        for (int p = seg.p0; p < seg.p1; ++p, ++n) {
          const int s = n % ST, sb = n & 1;
          if (!tree_wait(&k_full[s], (n / ST) & 1, abort_flag) || !tree_wait(&s_free[sb], ((n >> 1) & 1) ^ 1, abort_flag)) { give_up(93); ok = false; break; }
          tc_fence_after();
#pragma unroll
          for (int c = 0; c < NC; ++c) {
            const uint64_t kd = umma_desc_sw128(Ks + s * KV_BYTES + c * KC);
#pragma unroll
            for (int k = 0; k < 4; ++k) umma_f16_ta(tmem_base + sb * kPage, tmem_q + c * 32 + k * 8, kd + 2 * k, IDESC_S, (c | k) != 0);
          }
          umma_commit(&k_free[s]);
          umma_commit(&s_full[sb]);
        }
      }
    }
  } else if (warp == 10) {
    // ------------------------------------ O += P V -----------------------------------------------
    if (lane == 0) {
      int n = 0;
      bool ok = true;
      for (int sg = 0; ok && seg.next(a); ++sg) {
        if (!tree_wait(&o_free, (sg & 1) ^ 1, abort_flag)) { give_up(94); break; }
        for (int p = seg.p0; p < seg.p1; ++p, ++n) {
          const int s = n % ST, sb = n & 1;
          if (!tree_wait(&p_full[sb], (n >> 1) & 1, abort_flag) || !tree_wait(&v_full[s], (n / ST) & 1, abort_flag)) { give_up(95); ok = false; break; }
          tc_fence_after();
          const uint64_t pd = umma_desc_sw128(Ps + sb * P_BYTES);
          const uint64_t vd = umma_desc_mn_sw128(Vs + s * KV_BYTES, KC);
#pragma unroll
          for (int k = 0; k < 4; ++k) umma_f16(tmem_o, pd + 2 * k, vd + (uint64_t)(k * 16 * 128 >> 4), IDESC_O, p != seg.p0 || k != 0);
          umma_commit(&v_free[s]);
          umma_commit(&p_free[sb]);
        }
        if (ok) umma_commit(&o_full);
      }
    }
  } else if (Q8 && warp >= 11) {
    // ------------------------------------ int8 pages ---------------------------------------------
    // A thread holds 16 codes of each of kPage * HD / 16 / 128 places of K and of V; the next page's are requested before this one's
    // are converted.
    constexpr int PER = kPage * HD / 16 / 128;
    const int t = threadIdx.x - 352;
    uint4 kq[PER], vq[PER];
    float ksc = 0.f, vsc = 0.f;
    Segments ahead = seg;
    int ap = 0;
    bool have = false;
    auto fetch = [&]() {                              // the page after the last one fetched
      if (!have || ap >= ahead.p1) {
        if (!ahead.next(a)) { have = false; return; }
        ap = ahead.p0;
        have = true;
      }
      const int64_t slot0 = page_slot(a, ahead.r, ap);
      const int valid = slot0 < 0 ? 0 : min(kPage, cached_keys(a, ahead.r) - ap * kPage);
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const int idx = i * 128 + t, row = idx / (HD / 16), c = idx % (HD / 16);
        kq[i] = vq[i] = make_uint4(0, 0, 0, 0);
        if (row < valid) {
          const int64_t at = ((slot0 + row) * a.nkv + ahead.kvh) * HD + c * 16;
          kq[i] = ld_stream((const int8_t*)a.kpool + at);
          vq[i] = ld_stream((const int8_t*)a.vpool + at);
        }
      }
      if (t < kPage) {
        const int64_t row = (slot0 + t) * a.nkv + ahead.kvh;
        ksc = t < valid ? a.kscale[row] : 0.f;
        vsc = t < valid ? a.vscale[row] : 0.f;
      }
      ++ap;
    };
    auto store = [&](unsigned char* to, const uint4* q) {
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const int idx = i * 128 + t, row = idx / (HD / 16), c = idx % (HD / 16);
        unsigned char* at = to + (c / 4) * KC + row * 128;
        const int piece = (c % 4) * 2;
        const uint2 x = codes_to_bf16(q[i].x ^ 0x80808080u), y = codes_to_bf16(q[i].y ^ 0x80808080u);
        const uint2 z = codes_to_bf16(q[i].z ^ 0x80808080u), w = codes_to_bf16(q[i].w ^ 0x80808080u);
        *reinterpret_cast<uint4*>(at + ((piece ^ (row & 7)) << 4)) = make_uint4(x.x, x.y, y.x, y.y);
        *reinterpret_cast<uint4*>(at + (((piece + 1) ^ (row & 7)) << 4)) = make_uint4(z.x, z.y, w.x, w.y);
      }
    };
    fetch();
    int n = 0;
    bool ok = true;
    while (ok && seg.next(a))
      for (int p = seg.p0; p < seg.p1; ++p, ++n) {
        const int s = n % ST;
        const uint32_t ph = (n / ST) & 1;
        // both products of the stage's last page are done, so nobody reads its scales either
        if (!tree_wait(&k_free[s], ph ^ 1, abort_flag) || !tree_wait(&v_free[s], ph ^ 1, abort_flag)) { if (lane == 0) give_up(96); ok = false; break; }
        store(Ks + s * KV_BYTES, kq);
        store(Vs + s * KV_BYTES, vq);
        if (t < kPage) { scales[Q8 ? s : 0][0][t] = ksc; scales[Q8 ? s : 0][1][t] = vsc; }
        fence_async_smem();
        mbar_arrive(&k_full[s]);
        mbar_arrive(&v_full[s]);
        fetch();
      }
  } else if (warp < 10) {
    // ------------------------------------ softmax, sums -------------------------------------------
    const int q = warp & 3, hf = (warp - 2) >> 2, r = q * 32 + lane;
    const uint32_t lane_base = (uint32_t)(q * 32) << 16;
    int n = 0;
    uint32_t xph = 0;
    bool ok = true;
    for (int sg = 0; ok && seg.next(a); ++sg) {
      const int row = seg.tile * kRows + r, rows = a.C * a.rep;
      const bool idle = seg.tile * kRows + q * 32 >= rows;     // no row in this quadrant: its lanes only keep the barriers going
      const int keys = cached_keys(a, seg.r);
      if (!idle) {
        const int rr = min(row, rows - 1);
        const bf16* qrow = a.q + (((int64_t)seg.r * a.C + rr / a.rep) * a.nh + seg.kvh * a.rep + rr % a.rep) * HD;
#pragma unroll 1
        for (int i = hf; i < NC; i += 2) {
          uint32_t w[32];
#pragma unroll
          for (int v = 0; v < 8; ++v) {
            const uint4 x = *reinterpret_cast<const uint4*>(qrow + i * 64 + v * 8);
            w[4 * v] = x.x; w[4 * v + 1] = x.y; w[4 * v + 2] = x.z; w[4 * v + 3] = x.w;
          }
          tmem_st32(tmem_q + lane_base + i * 32, w);
        }
        tmem_st_wait();
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&q_full);
      float m_ref = -INFINITY, l = 0.f;
      for (int p = seg.p0; p < seg.p1; ++p, ++n) {
        const int sb = n & 1, s = n % ST;
        const uint32_t ph = (n >> 1) & 1;
        const int valid = page_slot(a, seg.r, p) < 0 ? 0 : min(kPage, keys - p * kPage);
        if (!tree_wait(&s_full[sb], ph, abort_flag)) { if (lane == 0) give_up(97); ok = false; break; }
        if (Q8 && !tree_wait(&k_full[s], (n / ST) & 1, abort_flag)) { if (lane == 0) give_up(97); ok = false; break; }
        tc_fence_after();
        uint32_t sv[32];
        if (!idle) {
          tmem_ld32(tmem_base + lane_base + sb * kPage + hf * 32, sv);
          tmem_ld_wait();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s_free[sb]);
        if (!idle) {
          float mx0 = -INFINITY, mx1 = -INFINITY;
          if (Q8) {
#pragma unroll
            for (int c = 0; c < 32; ++c) sv[c] = __float_as_uint(__uint_as_float(sv[c]) * (a.scale_log2 * scales[Q8 ? s : 0][0][hf * 32 + c]));
          } else {
#pragma unroll
            for (int c = 0; c < 32; ++c) sv[c] = __float_as_uint(__uint_as_float(sv[c]) * a.scale_log2);
          }
          if (valid < kPage) {
#pragma unroll
            for (int c = 0; c < 32; ++c)
              if (hf * 32 + c >= valid) sv[c] = __float_as_uint(-INFINITY);
          }
#pragma unroll
          for (int c = 0; c < 32; c += 2) {
            mx0 = fmaxf(mx0, __uint_as_float(sv[c]));
            mx1 = fmaxf(mx1, __uint_as_float(sv[c + 1]));
          }
          xch[sb][hf][r] = fmaxf(mx0, mx1);
        }
        mbar_arrive(&pair_bar[q]);
        if (!tree_wait(&pair_bar[q], xph, abort_flag)) { if (lane == 0) give_up(98); ok = false; break; }
        xph ^= 1;
        uint32_t pk[16];
        if (!idle) {
          const float mx = fmaxf(xch[sb][0][r], xch[sb][1][r]);
          if (p == seg.p0) m_ref = mx;
          else if (__any_sync(0xffffffffu, mx > m_ref + 8.f)) {
            // every product that wrote O has to be complete; the one of this page cannot start before P
            if (!tree_wait(&p_free[(n - 1) & 1], ((n - 1) >> 1) & 1, abort_flag)) { if (lane == 0) give_up(99); ok = false; break; }
            tc_fence_after();
            const float m_new = fmaxf(m_ref, mx), f = m_new == -INFINITY ? 1.f : tree_ex2(m_ref - m_new);
            m_ref = m_new;
            l *= f;
#pragma unroll 1
            for (int c0 = hf * (HD / 2); c0 < (hf + 1) * (HD / 2); c0 += 32) {
              uint32_t o[32];
              tmem_ld32(tmem_o + lane_base + c0, o);
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
              tmem_st32(tmem_o + lane_base + c0, o);
            }
            tmem_st_wait();
            tc_fence_before();
          }
          const float ms = m_ref == -INFINITY ? 0.f : m_ref;
          float l0 = 0.f, l1 = 0.f;
#pragma unroll
          for (int c = 0; c < 16; ++c) {
            float p0 = tree_ex2(__uint_as_float(sv[2 * c]) - ms), p1 = tree_ex2(__uint_as_float(sv[2 * c + 1]) - ms);
            l0 += p0; l1 += p1;
            if (Q8) { p0 *= scales[Q8 ? s : 0][1][hf * 32 + 2 * c]; p1 *= scales[Q8 ? s : 0][1][hf * 32 + 2 * c + 1]; }
            pk[c] = pack_bf162(p0, p1);               // weights rounded to bf16, half a step 2^-8; their sum is not
          }
          l += l0 + l1;
        }
        if (n >= 2 && !tree_wait(&p_free[sb], ((n - 2) >> 1) & 1, abort_flag)) { if (lane == 0) give_up(100); ok = false; break; }
        if (!idle) {
          unsigned char* prow = Ps + sb * P_BYTES + r * 128;
#pragma unroll
          for (int c = 0; c < 4; ++c)
            *reinterpret_cast<uint4*>(prow + (((hf * 4 + c) ^ (r & 7)) << 4)) = make_uint4(pk[4 * c], pk[4 * c + 1], pk[4 * c + 2], pk[4 * c + 3]);
        }
        if (!Q8 && valid < kPage) {                   // 0 times what lies behind the cache is not always 0: clear it
          if (!tree_wait(&v_full[s], (n / ST) & 1, abort_flag)) { if (lane == 0) give_up(101); ok = false; break; }
          const int per = (kPage - valid) * 8;        // 16-byte pieces of a chunk
          for (int i = (warp - 2) * 32 + lane; i < NC * per; i += 256)
            *reinterpret_cast<uint4*>(Vs + s * KV_BYTES + (i / per) * KC + valid * 128 + (i % per) * 16) = make_uint4(0, 0, 0, 0);
        }
        fence_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[sb]);
      }
      if (!ok) break;
      if (!tree_wait(&o_full, sg & 1, abort_flag)) { if (lane == 0) give_up(102); break; }
      tc_fence_after();
      if (hf == 1) lx[r] = l;
      mbar_arrive(&pair_bar[q]);
      if (!tree_wait(&pair_bar[q], xph, abort_flag)) { if (lane == 0) give_up(103); break; }
      xph ^= 1;
      if (!idle) {
        const int64_t at = ((int64_t)blockIdx.x + seg.item) * a.used + r;
        if (hf == 0 && row < rows) *reinterpret_cast<float2*>(a.part_ml + at * 2) = make_float2(m_ref, l + lx[r]);
#pragma unroll 1
        for (int c0 = hf * (HD / 2); c0 < (hf + 1) * (HD / 2); c0 += 32) {
          uint32_t o[32];
          tmem_ld32(tmem_o + lane_base + c0, o);
          tmem_ld_wait();
          if (row < rows) {
#pragma unroll
            for (int i = 0; i < 32; i += 4)
              *reinterpret_cast<uint4*>(a.part_o + at * HD + c0 + i) = make_uint4(o[i], o[i + 1], o[i + 2], o[i + 3]);
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&o_free);
    }
  }
  // ------------------------------------ teardown --------------------------------------------------
  tc_fence_before();
  __syncthreads();
  if (abort_s) {                                      // copies still in flight land before the shared memory is released
    const uint64_t t0 = tree_now();
    while (tree_now() - t0 < 2000000ull) __nanosleep(1000);
  }
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, TMEM_COLS);
  }
}

// A warp a (node, head): the node's path, then the partial sums of the cache, the gate and the store.  Lanes own hd / 32 channels.
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
    const int64_t slot0 = page_slot(a, r, p / kPage);
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
  int64_t before, all;
  page_sums(a, r, &before, &all);
  const int n = cached_pages(a, r);
  if (n > 0) {
    const int per = a.nkv * a.tiles, lrow = j * a.rep + h % a.rep, it = kvh * a.tiles + lrow / kRows, item = r * per + it;
    const int64_t T = all * per, g0 = before * per + (int64_t)it * n;
    const int b0 = piece_of(g0, T, a.ctas), b1 = piece_of(g0 + n - 1, T, a.ctas);
    for (int b = b0; b <= b1; ++b) {
      const int64_t at = (int64_t)(b + item) * a.used + lrow % kRows;
      if (piece_start(b, T, a.ctas) == piece_start(b + 1, T, a.ctas)) continue;      // fewer pages than pieces: an empty one
      const float2 ml = *reinterpret_cast<const float2*>(a.part_ml + at * 2);
      if (ml.x == -INFINITY) continue;                      // no key in these pages
      const float mn = fmaxf(m, ml.x), c = exp2f(m - mn), w = exp2f(ml.x - mn);
      m = mn;
      l = l * c + ml.y * w;
#pragma unroll
      for (int e = 0; e < EPL; ++e) o[e] = o[e] * c + w * a.part_o[at * HD + lane * EPL + e];
    }
  }
  const float inv = l > 0.f ? 1.f / l : 0.f;
  const bf16* gp = a.gate ? a.gate + row * a.ldg + (int64_t)h * 2 * HD + HD + lane * EPL : nullptr;
  bf16* op = a.out + row * a.ldo + (int64_t)h * HD + lane * EPL;
#pragma unroll
  for (int e = 0; e < EPL; ++e) op[e] = __float2bfloat16(o[e] * inv * (gp ? sigmoid_f(__bfloat162float(gp[e])) : 1.f));
}

template <int HD, bool Q8>
int launch_tree(const TreeAttnArgs& a, int64_t slots, cudaStream_t st) {
  CUtensorMap tmK = {}, tmV = {};
  if (!Q8) {
    int rc = cb_make_tmap_2d(&tmK, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, a.kpool, (uint64_t)slots, (uint64_t)a.nkv * HD, (uint64_t)a.nkv * HD, kPage, 64);
    if (!rc) rc = cb_make_tmap_2d(&tmV, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, a.vpool, (uint64_t)slots, (uint64_t)a.nkv * HD, (uint64_t)a.nkv * HD, kPage, 64);
    if (rc) return rc;
  }
  const size_t smem = (size_t)2 * TreeRing<HD, Q8>::stages * kPage * HD * 2 + 2 * kRows * kPage * 2;
  auto kern = tree_cache_kernel<HD, Q8>;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return (int)e;
  e = cb_launch(kern, dim3((unsigned)a.ctas), dim3(Q8 ? 480 : 352), smem, st, tmK, tmV, a);
  if (e != cudaSuccess) return (int)e;
  const int64_t tasks = (int64_t)a.R * a.C * a.nh;
  return (int)cb_launch(tree_finish_kernel<HD, Q8>, dim3((unsigned)((tasks + 7) / 8)), dim3(256), 0, st, a);
}

}  // namespace

// part: (ctas + R * nkv * tiles) * used * (hd + 2) floats, tiles = ceil(C * rep / 128), used = min(128, C * rep)
CB_EXPORT int cb_attn_tree(const void* q, const void* gate, int64_t ldg, const void* kpool, const void* vpool, int64_t slots,
                           const void* kscale, const void* vscale, const void* tables, int64_t ldbt, int64_t width, const void* positions,
                           const void* anc, void* out, int64_t ldo, void* part, int64_t ctas, int64_t R, int64_t C, int64_t nh, int64_t nkv,
                           int64_t hd, void* status, void* stream) {
  if (!q || !kpool || !vpool || !tables || !positions || !anc || !out || !part || !status) return CB_ERR_ARG;
  if ((kscale == nullptr) != (vscale == nullptr)) return CB_ERR_ARG;
  if (R < 1 || C < 1 || C > kMaxNodes || nkv < 1 || nh % nkv || ctas < 1 || ctas > 65535 || width < 1 || width > (1 << 24) || R * C * nh > (1ll << 30) || slots > 0x7fffffff ||
      ((uintptr_t)part & 15)) return CB_ERR_SHAPE;
  const int64_t rows = C * (nh / nkv), tiles = (rows + kRows - 1) / kRows, used = rows < kRows ? rows : kRows;
  const int64_t places = (ctas + R * nkv * tiles) * used;
  TreeAttnArgs a{(const bf16*)q, (const bf16*)gate, ldg, kpool, vpool, (const float*)kscale, (const float*)vscale, (const int*)tables, ldbt,
                 (int)width, (int)(slots / kPage), (const int*)positions, (const int64_t*)anc, (bf16*)out, ldo, (float*)part,
                 (float*)part + places * hd, (int)R, (int)C, (int)nh, (int)nkv, (int)(nh / nkv), (int)tiles, (int)used, (int)ctas,
                 1.4426950408889634f / sqrtf((float)hd), (int*)status};
  cudaStream_t st = (cudaStream_t)stream;
  if (hd == 256) return kscale ? launch_tree<256, true>(a, slots, st) : launch_tree<256, false>(a, slots, st);
  if (hd == 128) return kscale ? launch_tree<128, true>(a, slots, st) : launch_tree<128, false>(a, slots, st);
  if (hd == 64) return kscale ? launch_tree<64, true>(a, slots, st) : launch_tree<64, false>(a, slots, st);
  return CB_ERR_SHAPE;
}
