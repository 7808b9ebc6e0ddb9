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
// Cache kernel: an item is (sequence, kv head, 128 rows); the pages of all items form one list that the CTAs, one an SM, cut into pieces of
// the same length, whatever the sequences'.  A CTA walks the segments of its piece; each leaves unnormalised sums, maxima and sums of
// weights in slot (CTA + item), which is different for any two segments because one of the two grows from segment to segment.
// More than 128 rows a kv head: an item has 256, of which each CTA of a pair (cta_group::2) holds half.  Both bring half the bytes of every
// page, the even one issues the products, and what those threads wait for is signalled there by both.  (Two items of 128 rows bring every
// page twice: 2 x 64 nodes behind 65536 tokens 193 us, in pairs 149.)
// What bounds it: 8 x 16 nodes behind 517 to 16391 tokens, 280 MB in 52 us, 5.4 TB/s, the rest are the ends of the pieces and the merge; 2 x 64
// nodes behind 65536 tokens, 540 MB and 137 GFLOP in 119 us, tensor pipe 67 % busy; int8 pages, the chain of waits of a page (conversion, scores,
// softmax, values: 1.6 us, a page at a time; issue slots 33 % and tensor pipe 24 % busy).
//   warp 0       TMA: K and V pages into rings (a page of a kv head is a [64 x hd] box of the pool, hd / 64 swizzled [64 x 128 B] blocks)
//   warp 1, 10   tcgen05.mma (one thread each): S = Q K^T with Q in tensor memory into one of two accumulators; O += P V
//   warps 2-9    two groups of 128 threads, a thread a row: one takes the even pages, the other the odd ones, so that the exponentials of a
//                page run under the maxima of the next.  The reference maximum of a row goes from group to group through shared memory
//                ahead of the exponentials; it is raised, and O rescaled, only when the maximum has grown by more than 2^8.  Between
//                segments both groups put the next Q rows into tensor memory and take the sums out of it.
//   warps 11-18  int8 pools, in TMA's place: pages as codes by cp.async, two pages ahead, then as exact bf16 into the rings.  The keys'
//                scales multiply the scores, the values' the weights.
// Every wait is bounded by 2 s and reports through the status word; tensor memory is freed on every path.
#include "sm100.cuh"

namespace {
using namespace sm100;

constexpr int kPage = 64, kRows = 128, kMaxNodes = 64;
constexpr int kLoaders = 256;                         // threads that bring int8 pages

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
  float* part_o;                          // [workers + items, used rows, hd] unnormalised sums
  float* part_ml;                         // the same rows: (reference maximum, sum)
  int* part_pages;                        // what whole_pieces gave
  int R, C, nh, nkv, rep, span, tiles, used, workers;      // tiles: of `span` rows a (sequence, kv head); used: rows of a slot; workers: CTAs or pairs
  float scale_log2;                       // hd^-0.5 * log2(e)
  int* status;
};

__device__ __forceinline__ int cached_keys(const TreeAttnArgs& a, int r) { return max(0, min(a.positions[r], a.width * kPage)); }
__device__ __forceinline__ int pages_of(int pos0, int width) { return (max(0, min(pos0, width * kPage)) + kPage - 1) / kPage; }
__device__ __forceinline__ int cached_pages(const TreeAttnArgs& a, int r) { return pages_of(a.positions[r], a.width); }
// First slot of a page, or -1 where the table names none of the pool's.  Pages of nodes come from positions that may pass 2^31: unsigned.
__device__ __forceinline__ int64_t page_slot(const TreeAttnArgs& a, int r, unsigned page) {
  if (page >= (unsigned)a.width) return -1;
  const int id = a.tables[(int64_t)r * a.ldbt + page];
  return (unsigned)id < (unsigned)a.pages ? (int64_t)id * kPage : -1;
}
// The list of all items' T < 2^31 pages, cut into G even pieces (at most one a page), the first T % G of them a page longer.
__device__ __forceinline__ int piece_start(int b, int T, int G) { return b * (T / G) + min(b, T % G); }
__device__ __forceinline__ int piece_of(int g, int T, int G) {
  const int q = T / G, rest = T % G, longer = rest * (q + 1);
  return g < longer ? g / (q + 1) : rest + (g - longer) / q;
}
// Pages of a piece if no piece is to hold pages of two items: the smallest L for which ceil(n / L) pieces an item are no more than the
// workers.  0 where it is kSwitch pages or more above an even share: going from one item to the next costs a worker about as long as
// kSwitch pages (the sums leave tensor memory, the next Q enters it, and the chain of products starts anew).  us of a pass with whole
// pieces / with even ones: 8 x 16 nodes behind 517 to 16391 tokens 64 / 76, 4 x 23 behind up to 8191 (int8) 52 / 56, 2 x 64 behind 65536 133 / 140.
constexpr int kSwitch = 8;
__device__ __noinline__ int whole_pieces(const int* positions, int R, int width, int workers, int T, int per) {
  const int lane = threadIdx.x & 31, L = (T + workers - 1) / workers + lane;
  int pieces = 0;
#pragma unroll 1
  for (int r0 = 0; r0 < R; r0 += 32) {
    const int n = r0 + lane < R ? pages_of(positions[r0 + lane], width) : 0;
#pragma unroll 1
    for (int i = 0; i < min(32, R - r0); ++i) pieces += (__shfl_sync(0xffffffffu, n, i) + L - 1) / L;
  }
  const unsigned fits = __ballot_sync(0xffffffffu, lane < kSwitch && (int64_t)pieces * per <= workers);
  return fits ? __shfl_sync(0xffffffffu, L, __ffs(fits) - 1) : 0;
}

// Segments of a CTA's piece, one after the other.
struct Segments {
  int left;                               // pages of the piece to come
  int r, n, kvh, tile, item;              // sequence, pages of one of its items, item
  int p0, p1;                             // the segment: pages [p0, p1) of the item (at first, p1 is where the piece begins)
  __device__ __forceinline__ bool next(const TreeAttnArgs& a) {
    if (left <= 0) return false;
    while (p1 >= n) {
      p1 = 0;
      ++item;
      if (++tile == a.tiles) {
        tile = 0;
        if (++kvh == a.nkv) {
          kvh = 0;
          n = cached_pages(a, ++r);
        }
      }
    }
    p0 = p1;
    p1 = min(n, p0 + left);
    left -= p1 - p0;
    return true;
  }
};

// Bounded by the SM's own clock, 2 s at its highest rate (the global timer is read over the chip: dozens of warps that wait slow each other).
__device__ __noinline__ bool tree_wait_long(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  long long t0 = 0;
  for (;;) {
#pragma unroll 1
    for (int i = 0; i < 64; ++i)
      if (mbar_try(bar, parity)) return true;
    if (*abort_flag) return false;
    const long long now = clock64();
    if (t0 == 0) t0 = now;
    else if (now - t0 > 4000000000ll) return false;
  }
}
__device__ __forceinline__ bool tree_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  return mbar_try(bar, parity) || tree_wait_long(bar, parity, abort_flag);
}
__device__ __noinline__ void tree_give_up(int* status, volatile int* abort_flag, int code) {
  atomicCAS(status, 0, code);
  *abort_flag = 1;
}
__device__ __forceinline__ float tree_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// two at a time, in one instruction
__device__ __forceinline__ uint64_t pack2(float x, float y) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ void unpack2(uint64_t v, float& x, float& y) { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(v)); }
__device__ __forceinline__ uint64_t fma2(uint64_t x, uint64_t y, uint64_t z) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(x), "l"(y), "l"(z));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t x, uint64_t y) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(x), "l"(y));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t x, uint64_t y) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(x), "l"(y));
  return r;
}
// Four int8 codes -> four bf16, exact: 128 + (x & 127) is 0x4300 | (x & 127) as bf16, and 128 or (x < 0) 256 is 0x4300 | (x & 128).
__device__ __forceinline__ uint2 codes_to_bf16(uint32_t w) {
  uint2 v;
  uint32_t* o = &v.x;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t h = __byte_perm(w, 0, i ? 0x4342 : 0x4140);
    const uint32_t m = (h & 0x007f007fu) | 0x43004300u, c = (h & 0x00800080u) | 0x43004300u;
    const bf162 d = __hsub2(*reinterpret_cast<const bf162*>(&m), *reinterpret_cast<const bf162*>(&c));
    o[i] = *reinterpret_cast<const uint32_t*>(&d);
  }
  return v;
}

// Stages of the rings, and shared memory: rings of K and V, two tiles of P, int8: two pages of codes.  bf16 pages share one ring of
// twice as many tiles, in the order of their use: the scores of a page are multiplied while the page before is still in the softmax, so
// K of a page is requested before V of the page before it.  (With a ring each,
// a V tile waits for its turn in a place that a K tile could use.)
template <int HD, bool Q8, bool PAIR> struct TreeRing {
  static constexpr int half = Q8 && PAIR ? 2 : 1, stages = (HD == 256 ? (Q8 ? 2 : 3) : HD == 128 ? 4 : 6) * half;
  static constexpr size_t tile = (size_t)kPage * HD * 2 / half, bytes = 2 * stages * tile + 2 * kRows * kPage * 2 + (Q8 ? (size_t)2 * 2 * kPage * HD / half : 0);
};

// Places of step n's tiles in the order of the shared ring (the one before the last V stays empty).
__device__ __forceinline__ int unit_k(int n) { return n == 0 ? 0 : 2 * n - 1; }
__device__ __forceinline__ int unit_v(int n) { return 2 * n + 2; }

template <int HD, bool Q8, bool PAIR>
__global__ void __launch_bounds__(Q8 ? 352 + kLoaders : 352, 1)
tree_cache_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const TreeAttnArgs a) {
  // bf16 pairs take two pages a step: a page of K each, the two sides of one product of 128 keys (products of 64 keys take 46 cycles per 16
  // channels, of 128 keys 64 cycles), and half the channels of V of both.  An odd last page has a partner that is none.
  constexpr bool TWO = PAIR && !Q8;
  constexpr int HALF = PAIR ? 2 : 1, STEP = TWO ? 2 : 1, NC = HD / 64, VC = NC / HALF, ST = TreeRing<HD, Q8, PAIR>::stages, SPAN = kRows * HALF;
  // Scales of an int8 page are read until its accumulator is free.  K of page n is converted after the scores of page n - ST, and those
  // were multiplied after the accumulator of page n - ST - 2 was free.
  constexpr int SR = ST + 2;
  constexpr int KROWS = Q8 ? kPage / HALF : kPage, KC = KROWS * 128, VCB = kPage * 128;     // a tile's keys; 64 channels of them; of the values
  constexpr int KV_BYTES = (int)TreeRing<HD, Q8, PAIR>::tile, P_BYTES = kRows * kPage * 2;
  constexpr uint32_t TMEM_COLS = 2 * kPage + HD + HD / 2 <= 256 ? 256 : 512;
  constexpr uint32_t IDESC_S = umma_idesc(SPAN, STEP * kPage, 1, 1);
  constexpr uint32_t IDESC_O = umma_idesc(SPAN, HD, 1, 1) | (1u << 16);     // B operand MN-major
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* Ks = smem_raw;                       // the swizzle wants 1024-byte blocks; there is no room to round up
  unsigned char* Ps = Ks + 2 * ST * KV_BYTES;         // [2][P_BYTES]
  unsigned char* Cs = Ps + 2 * P_BYTES;               // int8: [2][K, V codes], each thread's own
  // bf16: k_full and k_free of all 2 ST places of the shared ring; int8: ST each of K and V
  __shared__ uint64_t q_full, k_full[2 * ST], k_free[2 * ST], s_full[2], s_free[2], p_full[2], p_free[2], o_full, o_free,
      m_done[4][2], pair_bar[4], sc_full[Q8 ? SR : 1];
  __shared__ float mref[kRows];                       // reference maxima
  __shared__ __align__(16) float scales[Q8 ? SR : 1][2][kPage];     // scale_log2 * key scales, value scales
  __shared__ Segments seg_s;
  __shared__ uint32_t tmem_base_s;
  __shared__ int abort_s;
  volatile int* abort_flag = &abort_s;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = PAIR ? cluster_ctarank() : 0;
  const bool lead = rank == 0;
  const int worker = blockIdx.x / HALF;
  if (smem_u32(smem_raw) & 1023) {
    if (threadIdx.x == 0) atomicCAS(a.status, 0, 89);
    return;
  }
  // Tensor memory is taken before a later kernel may start beside this one: one that took it first would wait for this kernel with it.
  if (warp == 1) {
    if (PAIR) { tmem_alloc_pair(&tmem_base_s, TMEM_COLS); tmem_relinquish_pair(); }
    else { tmem_alloc(&tmem_base_s, TMEM_COLS); tmem_relinquish(); }
  } else if (warp == 2) {
    if (lane == 0) {
      abort_s = 0;
      mbar_init(&q_full, 8 * HALF);
      mbar_init(&o_full, 1);
      mbar_init(&o_free, 8 * HALF);
      for (int i = 0; i < 2 * ST; ++i) { mbar_init(&k_full[i], Q8 ? kLoaders / 64 * HALF : lead ? HALF : 1); mbar_init(&k_free[i], 1); }
      for (int i = 0; i < 2; ++i) {
        mbar_init(&s_full[i], 1); mbar_init(&s_free[i], 4 * HALF); mbar_init(&p_full[i], 4 * HALF); mbar_init(&p_free[i], 1);
      }
      for (int i = 0; Q8 && i < SR; ++i) mbar_init(&sc_full[i], 2 * kPage);
      for (int i = 0; i < 4; ++i) { mbar_init(&m_done[i][0], 1); mbar_init(&m_done[i][1], 1); mbar_init(&pair_bar[i], 64); }
      mbar_fence_init();
    }
  }
  griddep_launch();
  griddep_wait();
  if (warp == 0) {
    int all = 0;
#pragma unroll 1
    for (int i = lane; i < a.R; i += 32) all += cached_pages(a, i);
    all = __reduce_add_sync(0xffffffffu, all);
    const int per = a.nkv * a.tiles, T = all * per, G = min(a.workers, T);
    const int L = T > G ? whole_pieces(a.positions, a.R, a.width, a.workers, T, per) : 0;      // (one page each: nothing to cut)
    if (blockIdx.x == 0 && lane == 0) *a.part_pages = L;
    // where the worker's piece begins and ends, in pages of the list or (whole pieces) as a number among all items' pieces
    const bool some = L ? true : worker < G;
    const int lo = L ? worker : some ? piece_start(worker, T, G) : 0, hi = L ? worker + 1 : some ? piece_start(worker + 1, T, G) : 0;
    int start = 0, r = 0;
    if (lo < hi)                                      // the sequence of the first page: 32 sequences at a time
#pragma unroll 1
      for (; r < a.R; r += 32) {
        const int np = r + lane < a.R ? cached_pages(a, r + lane) : 0, n = (L ? (np + L - 1) / L : np) * per;
        int incl = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int x = __shfl_up_sync(0xffffffffu, incl, o);
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
      seg_s.left = 0;
      if (lo < hi && r < a.R) {                       // (whole pieces: there may be fewer of them than workers)
        const int n = cached_pages(a, r), k = L ? (n + L - 1) / L : n, it = (lo - start) / k, i = lo - start - it * k;
        const int p = L ? piece_start(i, n, k) : i;
        seg_s = Segments{L ? piece_start(i + 1, n, k) - p : hi - lo, r, n, it / a.tiles, it % a.tiles, r * per + it, 0, p};
      }
    }
  }
  tc_fence_before();
  if (PAIR) cluster_sync_all();                       // both CTAs' barriers exist before either signals the other
  else __syncthreads();
  tc_fence_after();
  Segments seg = seg_s;
  const uint32_t tmem_base = tmem_base_s, tmem_o = tmem_base + 2 * kPage, tmem_q = tmem_o + HD;       // S0 | S1 | O | Q
  if (seg.left <= 0) {                                // no page for this CTA (and its pair)
    if (warp == 1) {
      if (PAIR) tmem_dealloc_pair(tmem_base, TMEM_COLS);
      else tmem_dealloc(tmem_base, TMEM_COLS);
    }
    return;
  }
  auto give_up = [&](int code) {
    tree_give_up(a.status, abort_flag, code);
    if (PAIR) st_cluster_u32(map_to_cta(smem_u32(&abort_s), rank ^ 1), 1);
  };
  // what the multiplying threads wait for is signalled in the CTA that has them; what they complete, in both
  auto signal = [&](uint64_t* bar) {
    if (PAIR) mbar_arrive_cluster(map_to_cta(smem_u32(bar), 0));
    else mbar_arrive(bar);
  };
  auto commit = [&](uint64_t* bar) {
    if (PAIR) umma_commit_pair(bar, 3);
    else umma_commit(bar);
  };
  // tile, barriers and phase of page n; pages of a segment with the one that makes it whole steps
  const int total = seg.left;
  auto k_at = [&](int n) { return Q8 ? n % ST : unit_k(n / STEP) % (2 * ST); };
  auto v_at = [&](int n) { return Q8 ? ST + n % ST : unit_v(n / STEP) % (2 * ST); };
  auto k_ph = [&](int n) { return (uint32_t)((Q8 ? n / ST : unit_k(n / STEP) / (2 * ST)) & 1); };
  auto v_ph = [&](int n) { return (uint32_t)((Q8 ? n / ST : unit_v(n / STEP) / (2 * ST)) & 1); };
  auto end_of = [&](const Segments& g) { return TWO ? g.p1 + ((g.p1 - g.p0) & 1) : g.p1; };

  if (warp == 0) {
    // ------------------------------------ TMA producer ------------------------------------------
    if (!Q8 && lane == 0) {
      // K of step n, then V of step n - 1.  The table's entries are fetched a step ahead: one thread's latencies add up.
      int p = 0, id[2] = {-1, -1};
      auto to_next = [&](bool first) {
        p += STEP;
        if (first || p >= seg.p1) {
          if (!seg.next(a)) return false;
          p = seg.p0;
        }
#pragma unroll
        for (int i = 0; i < STEP; ++i) id[i] = p + i < seg.p1 && p + i < a.width ? a.tables[(int64_t)seg.r * a.ldbt + p + i] : -1;
        return true;
      };
      // a tile of `parts` copies; slot -1: no such page, its scores are masked, its values cleared
      auto load = [&](const CUtensorMap* map, int u, int parts, const int* slot, int chunk) {
        const int at = u % (2 * ST);
        if (!tree_wait(&k_free[at], (u / (2 * ST) & 1) ^ 1, abort_flag)) { give_up(90); return false; }
        uint64_t* full = &k_full[at];
        const int bytes = KV_BYTES / parts, some = (slot[0] >= 0) + (parts > 1 && slot[STEP - 1] >= 0);
        if (some == 0) mbar_arrive(full);
        else mbar_expect_tx(full, some * bytes);
#pragma unroll
        for (int i = 0; i < STEP; ++i)
          if (i < parts && slot[i] >= 0)
#pragma unroll
            for (int c = 0; c < (map == &tmK ? NC : VC); ++c) tma_load_2d(Ks + at * KV_BYTES + i * bytes + c * VCB, map, full, (chunk + c) * 64, slot[i]);
        return true;
      };
      int v_slot[STEP], v_chunk = 0;
      bool more = to_next(true);
#pragma unroll 1
      for (int n = 0;; ++n) {
        const bool here = more;
        int slot[STEP];
#pragma unroll
        for (int i = 0; i < STEP; ++i) slot[i] = (unsigned)id[i] < (unsigned)a.pages ? id[i] * kPage : -1;
        const int chunk = seg.kvh * NC;
        if (here) {
          more = to_next(false);
          const int own = lead ? slot[0] : slot[STEP - 1];
          if (!load(&tmK, unit_k(n), 1, &own, chunk)) break;
        }
        if (n > 0 && !load(&tmV, unit_v(n - 1), STEP, v_slot, v_chunk + (int)rank * VC)) break;
        if (!here) break;
#pragma unroll
        for (int i = 0; i < STEP; ++i) v_slot[i] = slot[i];
        v_chunk = chunk;
      }
    }
  } else if (warp == 1) {
    // ------------------------------------ S = Q K^T ----------------------------------------------
    if (lead && lane == 0) {
      int n = 0;
      bool ok = true;
      for (int sg = 0; ok && seg.next(a); ++sg) {
        if (!tree_wait(&q_full, sg & 1, abort_flag)) { give_up(92); break; }
        tc_fence_after();
        for (int p = seg.p0; p < seg.p1; p += STEP, n += STEP) {
          const int s = k_at(n), sb = n & 1;
          if (!tree_wait(&k_full[s], k_ph(n), abort_flag) || !tree_wait(&s_free[sb], ((n >> 1) & 1) ^ 1, abort_flag) ||
              (TWO && !tree_wait(&s_free[1], ((n >> 1) & 1) ^ 1, abort_flag))) { give_up(93); ok = false; break; }
          tc_fence_after();
#pragma unroll
          for (int c = 0; c < NC; ++c) {
            const uint64_t kd = umma_desc_sw128(Ks + s * KV_BYTES + c * KC);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              if (PAIR) umma_f16_ta_pair(tmem_base + sb * kPage, tmem_q + c * 32 + k * 8, kd + 2 * k, IDESC_S, (c | k) != 0);
              else umma_f16_ta(tmem_base + sb * kPage, tmem_q + c * 32 + k * 8, kd + 2 * k, IDESC_S, (c | k) != 0);
            }
          }
          commit(&k_free[s]);
          commit(&s_full[sb]);
          if (TWO) commit(&s_full[1]);
        }
      }
    }
  } else if (warp == 10) {
    // ------------------------------------ O += P V -----------------------------------------------
    if (TWO && !lead) {
      // nothing is multiplied from here; the tiles that land here are reported to the CTA that does
      if (lane == 0) {
        int steps = 0;
        while (seg.next(a)) steps += (end_of(seg) - seg.p0) / STEP;
#pragma unroll 1
        for (int u = 0; u <= 2 * steps; ++u) {
          if (u == 2 * steps - 1) continue;
          if (!tree_wait(&k_full[u % (2 * ST)], (u / (2 * ST)) & 1, abort_flag)) { give_up(104); break; }
          signal(&k_full[u % (2 * ST)]);
        }
      }
    } else if (lead && lane == 0) {
      int n = 0;
      bool ok = true;
      for (int sg = 0; ok && seg.next(a); ++sg) {
        if (!tree_wait(&o_free, (sg & 1) ^ 1, abort_flag)) { give_up(94); break; }
        for (int p = seg.p0; p < end_of(seg); ++p, ++n) {
          const int s = v_at(n), sb = n & 1;
          if (!tree_wait(&p_full[sb], (n >> 1) & 1, abort_flag) || !tree_wait(&k_full[s], v_ph(n), abort_flag)) { give_up(95); ok = false; break; }
          tc_fence_after();
          const uint64_t pd = umma_desc_sw128(Ps + sb * P_BYTES);
          const uint64_t vd = umma_desc_mn_sw128(Ks + s * KV_BYTES + (TWO ? sb * (KV_BYTES / 2) : 0), VCB);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            if (PAIR) umma_f16_pair(tmem_o, pd + 2 * k, vd + (uint64_t)(k * 16 * 128 >> 4), IDESC_O, p != seg.p0 || k != 0);
            else umma_f16(tmem_o, pd + 2 * k, vd + (uint64_t)(k * 16 * 128 >> 4), IDESC_O, p != seg.p0 || k != 0);
          }
          if (!TWO || sb) commit(&k_free[s]);
          commit(&p_free[sb]);
        }
        if (ok) commit(&o_full);
      }
    }
  } else if (Q8 && warp >= 11) {
    // ------------------------------------ int8 pages ---------------------------------------------
    // Half of the loaders take the keys, half the values, each at its own pace.  16 codes of a row are a piece; a quarter warp takes four
    // pieces of each of two rows, so that its bf16 stores hit all banks once.  (Loops are kept short: with every copy unrolled the code
    // of all roles leaves the instruction cache, and a page takes twice as long.)
    constexpr int NT = kLoaders / 2, PER = kPage * HD / 16 / NT / HALF, CODES = kPage * HD / HALF;
    const int v = (threadIdx.x - 352) / NT, t = (threadIdx.x - 352) % NT;
    const int g4 = PAIR && v ? VC : NC, step = NT / 4 / g4;                             // groups of 64 channels here; rows from piece to piece
    const int row0 = t / 8 / g4 * 2 + t % 8 / 4, c0 = t / 8 % g4 * 4 + t % 4;          // piece i: row0 + i * step, c0
    const int skip = PAIR && !v ? (int)rank * KROWS : 0, cskip = PAIR && v ? (int)rank * (HD / 2) : 0;       // this CTA's first row and channel of a page
    const int chunk = v ? VCB : KC;
    const int8_t* pool = (const int8_t*)(v ? a.vpool : a.kpool);
    const float* pscale = v ? a.vscale : a.kscale;
    const float smul = v ? 1.f : a.scale_log2;
    const int64_t pitch = (int64_t)a.nkv * HD;
    unsigned char* const mine = Cs + v * 2 * CODES + t * 16;                            // two pages of this thread's own pieces
    unsigned char* const to0 = Ks + v * ST * KV_BYTES + (c0 / 4) * chunk + row0 * 128;
    const int piece = (c0 % 4) * 2, at0 = (piece ^ (row0 & 7)) << 4, at1 = ((piece + 1) ^ (row0 & 7)) << 4;      // step is a multiple of 8
    float s0 = 0.f, s1 = 0.f;                         // scale of row t of the page to convert and of the one after it
    // page to request next: its segment, its entry of the table (fetched a page ahead of its use) and the keys of its sequence
    Segments ahead = seg;
    int ap = 0, id = 0, keys = 0;
    auto to_next = [&](bool first) {
      if (first || ++ap == ahead.p1) {
        if (!ahead.next(a)) return;
        ap = ahead.p0;
        keys = cached_keys(a, ahead.r);
      }
      id = ap < a.width ? a.tables[(int64_t)ahead.r * a.ldbt + ap] : -1;
    };
    to_next(true);
#pragma unroll 1
    for (int n = -2; n < total; ++n) {
      if (n >= 0) {
        const int st = n % ST;
        asm volatile("cp.async.wait_group 1;" ::: "memory");
        if (!tree_wait(&k_free[v * ST + st], (n / ST & 1) ^ 1, abort_flag)) { if (lane == 0) give_up(96); break; }
        if (t < kPage) {
          scales[Q8 ? n % SR : 0][v][t] = s0 * smul;
          mbar_arrive(&sc_full[Q8 ? n % SR : 0]);
        }
        const unsigned char* codes = mine + (n & 1) * CODES;
        unsigned char* to = to0 + st * KV_BYTES;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
          const uint4 x = *reinterpret_cast<const uint4*>(codes + i * NT * 16);
          const uint2 x0 = codes_to_bf16(x.x), x1 = codes_to_bf16(x.y), x2 = codes_to_bf16(x.z), x3 = codes_to_bf16(x.w);
          *reinterpret_cast<uint4*>(to + i * step * 128 + at0) = make_uint4(x0.x, x0.y, x1.x, x1.y);
          *reinterpret_cast<uint4*>(to + i * step * 128 + at1) = make_uint4(x2.x, x2.y, x3.x, x3.y);
        }
        fence_async_smem();
        __syncwarp();
        if (lane == 0) signal(&k_full[v * ST + st]);
      }
      // codes of page n + 2, into the place that was just read, by the same threads
      s0 = s1;
      if (n + 2 < total) {
        const int64_t slot0 = (int64_t)id * kPage;
        const int valid = (unsigned)id < (unsigned)a.pages ? min(kPage, keys - ap * kPage) : 0;
        const uint32_t to = smem_u32(mine + (n & 1) * CODES);
        const int8_t* from = pool + (valid ? (slot0 + skip + row0) * pitch + ahead.kvh * HD + cskip + c0 * 16 : 0);
#pragma unroll
        for (int i = 0; i < PER; ++i) {
          const bool in = skip + row0 + i * step < valid;    // else zeros, and the address is not read
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to + i * NT * 16), "l"(in ? from + i * step * pitch : pool), "r"(in ? 16 : 0));
        }
        s1 = t < valid ? pscale[(slot0 + t) * a.nkv + ahead.kvh] : 1.f;
        to_next(false);
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  } else if (warp < 10) {
    // ------------------------------------ softmax, sums -------------------------------------------
    const int q = warp & 3, grp = (warp - 2) >> 2, r = q * 32 + lane;
    const uint32_t lane_base = (uint32_t)(q * 32) << 16;
    const int rows = a.C * a.rep;
    // This warp's own 4 KB of the P tiles, 32 rows of 128 bytes in 16-byte pieces c at c ^ (row % 8), between segments: rows go to and from
    // tensor memory a thread each, and to and from global memory eight threads each.
    unsigned char* const own = Ps + grp * P_BYTES + q * 4096;
    const int sub = lane >> 3, pc = lane & 7;
    auto load_q = [&](const Segments& g) {            // 32 rows of the segment's Q into tensor memory, every other 64 columns a group
      const int first = g.tile * SPAN + (int)rank * kRows + q * 32;
      if (first < rows) {
        const bf16* qs = a.q + ((int64_t)g.r * a.C * a.nh + g.kvh * a.rep) * HD;
#pragma unroll 1
        for (int i = grp; i < NC; i += 2) {
          uint4 x[8];
#pragma unroll
          for (int v = 0; v < 8; ++v) {
            const int rr = min(first + v * 4 + sub, rows - 1);
            x[v] = *reinterpret_cast<const uint4*>(qs + ((int64_t)(rr / a.rep) * a.nh + rr % a.rep) * HD + i * 64 + pc * 8);
          }
#pragma unroll
          for (int v = 0; v < 8; ++v) *reinterpret_cast<uint4*>(own + (v * 4 + sub) * 128 + ((pc ^ ((v * 4 + sub) & 7)) << 4)) = x[v];
          __syncwarp();
          uint32_t w[32];
#pragma unroll
          for (int v = 0; v < 8; ++v) *reinterpret_cast<uint4*>(w + 4 * v) = *reinterpret_cast<const uint4*>(own + lane * 128 + ((v ^ (lane & 7)) << 4));
          tmem_st32(tmem_q + lane_base + i * 32, w);
          __syncwarp();
        }
        tmem_st_wait();
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) signal(&q_full);
    };
    int n = 0;
    bool ok = true;
    Segments ahead = seg;
    bool more = ahead.next(a);
    if (more) load_q(ahead);
    for (int sg = 0; ok && more; ++sg) {
      seg = ahead;
      const int row_a = seg.tile * SPAN + (int)rank * kRows;     // this CTA's first row
      const bool idle = row_a + q * 32 >= rows;                // no row in this quadrant: its lanes only keep the barriers going
      const int keys = cached_keys(a, seg.r), row = row_a + r;
      float m = -INFINITY, l = 0.f;
      for (int p = seg.p0; p < end_of(seg); ++p, ++n) {
        const int sb = n & 1, s = n % SR;
        if (sb != grp) continue;
        const int valid = (TWO && p >= seg.p1) || page_slot(a, seg.r, p) < 0 ? 0 : min(kPage, keys - p * kPage);
        if (!tree_wait(&s_full[sb], (n >> 1) & 1, abort_flag)) { if (lane == 0) give_up(97); ok = false; break; }
        if (Q8 && !tree_wait(&sc_full[Q8 ? s : 0], (n / SR) & 1, abort_flag)) { if (lane == 0) give_up(97); ok = false; break; }
        tc_fence_after();
        // Two pages a product: the scores go to registers whole, and the accumulators are free for the next product before any exponential
        // (2 x 64 nodes behind 65536 tokens 131 us, freed behind them 174).  Else 32 columns at a time, and twice, which leaves half the
        // registers and half the code (8 x 16 nodes behind up to 16391 tokens 64.1 us, whole 65.6).
        uint32_t sv[TWO ? kPage : 32];
        auto scores = [&](int c0) {
          tmem_ld32(tmem_base + lane_base + sb * kPage + c0, sv);
          if (TWO) tmem_ld32(tmem_base + lane_base + sb * kPage + 32, sv + (TWO ? 32 : 0));
          tmem_ld_wait();
        };
        auto mask = [&](int c0) {                     // (int8: scales behind the end are 1)
          if (valid < kPage) {
#pragma unroll
            for (int c = 0; c < (TWO ? kPage : 32); ++c)
              if (c0 + c >= valid) sv[c] = __float_as_uint(-INFINITY);
          }
        };
        const uint64_t* const ks2 = reinterpret_cast<const uint64_t*>(scales[Q8 ? s : 0][0]);
        const uint64_t* const vs2 = reinterpret_cast<const uint64_t*>(scales[Q8 ? s : 0][1]);
        float mx = -INFINITY;
        if (!idle) {
          float mx1 = -INFINITY;
#pragma unroll 1
          for (int c0 = 0; c0 < kPage; c0 += TWO ? kPage : 32) {
            scores(c0);
            if (TWO) {
              tc_fence_before();
              __syncwarp();
              if (lane == 0) signal(&s_free[sb]);
            }
            mask(c0);
#pragma unroll
            for (int c = 0; c < (TWO ? kPage : 32); c += 2) {
              float s0 = __uint_as_float(sv[c]), s1 = __uint_as_float(sv[c + 1]);
              if (Q8) unpack2(mul2(pack2(s0, s1), ks2[(c0 + c) / 2]), s0, s1);
              mx = fmaxf(mx, s0);
              mx1 = fmaxf(mx1, s1);
            }
          }
          mx = fmaxf(mx, mx1);
          if (!Q8) mx *= a.scale_log2;
        } else if (TWO && lane == 0) signal(&s_free[sb]);
        if (p == seg.p0) m = mx;
        else {                                        // the other group has left the reference of the page before
          if (!tree_wait(&m_done[q][sb ^ 1], ((n - 1) >> 1) & 1, abort_flag)) { if (lane == 0) give_up(98); ok = false; break; }
          if (!idle) {
            const float was = mref[r];
            if (was != m) {
              l = l > 0.f ? l * tree_ex2(m - was) : l;
              m = was;
            }
            if (__any_sync(0xffffffffu, mx > m + 8.f)) {
              // every product that wrote O has to be complete; the one of this page cannot start before P
              if (!tree_wait(&p_free[sb ^ 1], ((n - 1) >> 1) & 1, abort_flag)) { if (lane == 0) give_up(99); ok = false; break; }
              tc_fence_after();
              const float m_new = fmaxf(m, mx), f = m_new == -INFINITY ? 1.f : tree_ex2(m - m_new);
              m = m_new;
              l *= f;
#pragma unroll 1
              for (int c0 = 0; c0 < HD; c0 += 32) {
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
          }
        }
        if (!idle) mref[r] = m;
        __syncwarp();
        if (lane == 0) mbar_arrive(&m_done[q][sb]);
        const float ms = m == -INFINITY ? 0.f : m;
        if (n >= 2 && !tree_wait(&p_free[sb], ((n - 2) >> 1) & 1, abort_flag)) { if (lane == 0) give_up(100); ok = false; break; }
        if (!idle) {
          unsigned char* prow = Ps + sb * P_BYTES + r * 128;
          uint64_t l2 = 0;
          const uint64_t scale2 = pack2(a.scale_log2, a.scale_log2), minus2 = pack2(-ms, -ms);
#pragma unroll 1
          for (int c0 = 0; c0 < kPage; c0 += TWO ? kPage : 32) {
            if (!TWO) {
              scores(c0);
              mask(c0);
            }
#pragma unroll
            for (int c = 0; c < (TWO ? 8 : 4); ++c) {
              uint32_t pk[4];
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const int k = c * 8 + i * 2;
                float p0, p1;
                unpack2(fma2(pack2(__uint_as_float(sv[k]), __uint_as_float(sv[k + 1])), Q8 ? ks2[(c0 + k) / 2] : scale2, minus2), p0, p1);
                p0 = tree_ex2(p0);
                p1 = tree_ex2(p1);
                l2 = add2(l2, pack2(p0, p1));
                if (Q8) unpack2(mul2(pack2(p0, p1), vs2[(c0 + k) / 2]), p0, p1);
                pk[i] = pack_bf162(p0, p1);           // bf16, half a step 2^-8: the product takes operands of one type, and V is bf16; the sum is of the exact ones
              }
              *reinterpret_cast<uint4*>(prow + (((c0 / 8 + c) ^ (r & 7)) << 4)) = make_uint4(pk[0], pk[1], pk[2], pk[3]);
            }
          }
          float l0, l1;
          unpack2(l2, l0, l1);
          l += l0 + l1;
        }
        if (!TWO) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) signal(&s_free[sb]);
        }
        if (!Q8 && valid < kPage) {                   // 0 times what lies behind the cache is not always 0: clear it
          if (!tree_wait(&k_full[v_at(n)], v_ph(n), abort_flag)) { if (lane == 0) give_up(101); ok = false; break; }
          const int per = (kPage - valid) * 8;        // 16-byte pieces of a chunk
          for (int i = q * 32 + lane; i < VC * per; i += 128)
            *reinterpret_cast<uint4*>(Ks + v_at(n) * KV_BYTES + (TWO ? sb * (KV_BYTES / 2) : 0) + (i / per) * VCB + valid * 128 + (i % per) * 16) = make_uint4(0, 0, 0, 0);
        }
        fence_async_smem();
        __syncwarp();
        if (lane == 0) signal(&p_full[sb]);
      }
      if (!ok) break;
      if (!tree_wait(&o_full, sg & 1, abort_flag) || !tree_wait(&m_done[q][(n - 1) & 1], ((n - 1) >> 1) & 1, abort_flag)) { if (lane == 0) give_up(102); break; }
      tc_fence_after();
      // all products of the segment are done: Q, O and the P tiles are free
      more = ahead.next(a);
      if (more) load_q(ahead);
      const float was = idle ? 0.f : mref[r];
      l = l > 0.f ? l * tree_ex2(m - was) : l;
      mbar_arrive(&pair_bar[q]);
      if (!tree_wait(&pair_bar[q], 0, abort_flag)) { if (lane == 0) give_up(103); break; }
      // the odd group's sums by way of the even group's tile, which nobody else writes
      if (grp == 1) reinterpret_cast<float*>(own - P_BYTES)[lane] = l;
      mbar_arrive(&pair_bar[q]);
      if (!tree_wait(&pair_bar[q], 1, abort_flag)) { if (lane == 0) give_up(103); break; }
      if (!idle) {
        const int64_t at = ((int64_t)worker + seg.item) * a.used + (int)rank * kRows + q * 32;         // the warp's first row
        if (grp == 0 && row < rows) *reinterpret_cast<float2*>(a.part_ml + (at + lane) * 2) = make_float2(was, l + reinterpret_cast<const float*>(own)[lane]);
        __syncwarp();
        const int here = min(32, rows - row_a - q * 32);
#pragma unroll 1
        for (int c0 = grp * (HD / 2); c0 < (grp + 1) * (HD / 2); c0 += 32) {
          uint32_t o[32];
          tmem_ld32(tmem_o + lane_base + c0, o);
          tmem_ld_wait();
#pragma unroll
          for (int v = 0; v < 8; ++v) *reinterpret_cast<uint4*>(own + lane * 128 + ((v ^ (lane & 7)) << 4)) = *reinterpret_cast<const uint4*>(o + 4 * v);
          __syncwarp();
#pragma unroll
          for (int v = 0; v < 8; ++v) {
            const int rr = v * 4 + sub;
            if (rr < here) *reinterpret_cast<uint4*>(a.part_o + (at + rr) * HD + c0 + pc * 4) = *reinterpret_cast<const uint4*>(own + rr * 128 + ((pc ^ (rr & 7)) << 4));
          }
          __syncwarp();
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) signal(&o_free);
    }
  }
  // ------------------------------------ teardown --------------------------------------------------
  tc_fence_before();
  __syncthreads();
  if (abort_s) {                                      // copies still in flight land before the shared memory is released
    const long long t0 = clock64();
    while (clock64() - t0 < 4000000ll) __nanosleep(1000);
  }
  if (PAIR) cluster_sync_all();                       // the products read and write both CTAs' memory, and both signal each other
  if (warp == 1) {
    tc_fence_after();
    if (PAIR) tmem_dealloc_pair(tmem_base, TMEM_COLS);
    else tmem_dealloc(tmem_base, TMEM_COLS);
  }
}

// EPL channels of one lane of a row, packed as they lie in memory (words of two bf16 or of four codes), and as floats (codes unscaled)
template <int EPL, bool Q8> struct RowPiece {
  static constexpr int W = Q8 ? (EPL + 3) / 4 : EPL / 2;
  uint32_t w[W];
  __device__ __forceinline__ void load(const void* pool, int64_t at) {
    const char* p = (const char*)pool + at * (Q8 ? 1 : 2);
    if (W == 4) *reinterpret_cast<uint4*>(w) = *reinterpret_cast<const uint4*>(p);
    else if (W == 2) *reinterpret_cast<uint2*>(w) = *reinterpret_cast<const uint2*>(p);
    else if (Q8 && EPL == 2) w[0] = *reinterpret_cast<const uint16_t*>(p);
    else w[0] = *reinterpret_cast<const uint32_t*>(p);
  }
  __device__ __forceinline__ float at(int e) const {
    if (Q8) return (float)(int8_t)(w[e / 4] >> (8 * (e & 3)) & 0xff);
    return __uint_as_float(e & 1 ? w[e / 2] & 0xffff0000u : w[e / 2] << 16);
  }
};

// A warp a (node, head): the node's path, the partial sums of the cache, the gate and the store.  Lanes own hd / 32 channels of a row;
// lane i also keeps the pool rows of nodes i and i + 32, and the maximum and sum of a partial.  Latency is all there is to it: tables and
// maxima are fetched by all lanes at once, keys and values of eight nodes together, partials eight at a time.
template <int HD, bool Q8>
__global__ void __launch_bounds__(256) tree_finish_kernel(const TreeAttnArgs a) {
  constexpr int EPL = HD / 32, kAtOnce = 8;
  griddep_launch();
  griddep_wait();
  const int64_t task = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (task >= (int64_t)a.R * a.C * a.nh) return;
  const int h = (int)(task % a.nh), j = (int)(task / a.nh % a.C), r = (int)(task / ((int64_t)a.nh * a.C));
  // what depends on nothing is requested first, then what depends on it: tables and the partials' maxima, then rows
  const int64_t row = (int64_t)r * a.C + j;
  const int pos0 = a.positions[r], L = *a.part_pages, mine0 = lane < a.R ? a.positions[lane] : -1;
  uint64_t on = (uint64_t)a.anc[row];
  RowPiece<EPL, false> qp, gp;
  qp.load(a.q, (row * a.nh + h) * HD + lane * EPL);
  if (a.gate) gp.load(a.gate, row * a.ldg + (int64_t)h * 2 * HD + HD + lane * EPL);
  if (on == 0 || pos0 < 0) return;
  on = (on & (~0ull >> (63 - j))) | 1ull << j;              // a path ends at its node
  const int kvh = h / a.rep;
  int64_t slot0[2];
#pragma unroll
  for (int u = 0; u < 2; ++u) slot0[u] = on >> (lane + 32 * u) & 1 ? page_slot(a, r, ((unsigned)pos0 + lane + 32 * u) / kPage) : -1;
  // the cache's partials: maxima and sums, one a lane
  auto pieces = [&](int pos) { const int n = pages_of(pos, a.width); return L ? (n + L - 1) / L : n; };
  int all = pieces(mine0), before = lane < r ? all : 0;
#pragma unroll 1
  for (int i = lane + 32; i < a.R; i += 32) {
    const int x = pieces(a.positions[i]);
    all += x;
    if (i < r) before += x;
  }
  all = __reduce_add_sync(0xffffffffu, all);
  before = __reduce_add_sync(0xffffffffu, before);
  const int n = pages_of(pos0, a.width), per = a.nkv * a.tiles, lrow = j * a.rep + h % a.rep, it = kvh * a.tiles + lrow / a.span, item = r * per + it;
  int b0 = 0, parts = 0;
  if (n > 0 && L) {
    parts = (n + L - 1) / L;
    b0 = before * per + it * parts;
  } else if (n > 0) {
    const int T = all * per, g0 = before * per + it * n, G = min(a.workers, T);
    b0 = piece_of(g0, T, G);
    parts = piece_of(g0 + n - 1, T, G) - b0 + 1;
  }
  const int64_t at0 = (int64_t)(b0 + item) * a.used + lrow % a.span;
  auto sums = [&](int b) { return b < parts ? *reinterpret_cast<const float2*>(a.part_ml + (at0 + (int64_t)b * a.used) * 2) : make_float2(-INFINITY, 0.f); };
  const float2 ml0 = sums(lane);
  // pool rows of the path; a page that is none takes its nodes off it
  int64_t kr[2];
  float ks[2] = {1.f, 1.f}, vs[2] = {1.f, 1.f};
  uint64_t path = 0;
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    kr[u] = slot0[u] < 0 ? 0 : (slot0[u] + ((unsigned)pos0 + lane + 32 * u) % kPage) * a.nkv + kvh;
    if (Q8 && slot0[u] >= 0) { ks[u] = a.kscale[kr[u]]; vs[u] = a.vscale[kr[u]]; }
    path |= (uint64_t)__ballot_sync(0xffffffffu, slot0[u] >= 0) << (32 * u);
  }
  float q[EPL], o[EPL];
#pragma unroll
  for (int e = 0; e < EPL; ++e) { q[e] = qp.at(e) * a.scale_log2; o[e] = 0.f; }
  float m = ml0.x, l = 0.f;
#pragma unroll 1
  for (int b = lane + 32; b < parts; b += 32) m = fmaxf(m, sums(b).x);
  m = warp_max(m);
  // the path, kAtOnce nodes at a time: keys and values are requested together
#pragma unroll 1
  for (uint64_t rest = path; rest;) {
    RowPiece<EPL, Q8> kp[kAtOnce], vp[kAtOnce];
    float s[kAtOnce], kf[kAtOnce], vf[kAtOnce];
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) {
      const int i = rest ? __ffsll((long long)rest) - 1 : -1;
      rest &= rest - 1;
      const int64_t at = i < 32 ? __shfl_sync(0xffffffffu, kr[0], i & 31) : __shfl_sync(0xffffffffu, kr[1], i & 31);
      kf[k] = vf[k] = 1.f;
      if (Q8) {
        kf[k] = i < 32 ? __shfl_sync(0xffffffffu, ks[0], i & 31) : __shfl_sync(0xffffffffu, ks[1], i & 31);
        vf[k] = i < 32 ? __shfl_sync(0xffffffffu, vs[0], i & 31) : __shfl_sync(0xffffffffu, vs[1], i & 31);
      }
      s[k] = i >= 0 ? 0.f : -INFINITY;
      if (i >= 0) {
        kp[k].load(a.kpool, at * HD + lane * EPL);
        vp[k].load(a.vpool, at * HD + lane * EPL);
      } else {
#pragma unroll
        for (int x = 0; x < RowPiece<EPL, Q8>::W; ++x) vp[k].w[x] = 0u;
      }
    }
    float mn = m;
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) {
      if (s[k] == 0.f) {                                    // a node (the same for the warp)
        float d = 0.f;
#pragma unroll
        for (int e = 0; e < EPL; ++e) d = fmaf(q[e], kp[k].at(e), d);
        s[k] = warp_sum(d) * kf[k];
      }
      mn = fmaxf(mn, s[k]);
    }
    const float ms = mn == -INFINITY ? 0.f : mn, c = exp2f(m - ms);
    m = mn;
    l *= c;
#pragma unroll
    for (int e = 0; e < EPL; ++e) o[e] *= c;
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) {
      const float w = exp2f(s[k] - ms);
      if (lane == 0) l += w;                                // the partials' sums are one a lane
#pragma unroll
      for (int e = 0; e < EPL; ++e) o[e] = fmaf(w * vf[k], vp[k].at(e), o[e]);
    }
  }
  const float ms = m == -INFINITY ? 0.f : m;
#pragma unroll 1
  for (int c = 0; c < parts; c += 32) {
    const float2 ml = c ? sums(c + lane) : ml0;
    const float f = exp2f(ml.x - ms);                       // 0 where these pages hold no key
    l += f * ml.y;
    const int here = min(32, parts - c);
#pragma unroll 1
    for (int b = 0; b < here; b += kAtOnce) {
      float x[kAtOnce][EPL], g[kAtOnce];
#pragma unroll
      for (int k = 0; k < kAtOnce; ++k) {
        g[k] = b + k < here ? __shfl_sync(0xffffffffu, f, b + k) : 0.f;      // (the same branch for the warp)
        if (g[k] != 0.f) {
          const float* po = a.part_o + (at0 + (int64_t)(c + b + k) * a.used) * HD + lane * EPL;
          if (EPL == 8) {
            *reinterpret_cast<float4*>(x[k]) = *reinterpret_cast<const float4*>(po);
            *reinterpret_cast<float4*>(x[k] + EPL / 2) = *reinterpret_cast<const float4*>(po + 4);
          } else {
#pragma unroll
            for (int e = 0; e < EPL; ++e) x[k][e] = po[e];
          }
        }
      }
#pragma unroll
      for (int k = 0; k < kAtOnce; ++k)
        if (g[k] != 0.f) {
#pragma unroll
          for (int e = 0; e < EPL; ++e) o[e] = fmaf(g[k], x[k][e], o[e]);
        }
    }
  }
  l = warp_sum(l);
  // no weight at all: 0.  (A sum that is no number reaches the row whatever the partial sums that were skipped: scores of a whole piece that
  // are NaN leave its maximum at -inf.)
  const float inv = l == 0.f ? 0.f : 1.f / l;
  bf16* op = a.out + row * a.ldo + (int64_t)h * HD + lane * EPL;
#pragma unroll
  for (int e = 0; e < EPL; ++e) o[e] *= inv * (a.gate ? sigmoid_f(gp.at(e)) : 1.f);
  if (EPL == 8) *reinterpret_cast<uint4*>(op) = float_to_bf16x8(o);
  else {
#pragma unroll
    for (int e = 0; e < EPL; e += 2) *reinterpret_cast<uint32_t*>(op + e) = pack_bf162(o[e], o[e + 1]);
  }
}

template <int HD, bool Q8, bool PAIR>
int launch_cache(const TreeAttnArgs& a, int64_t slots, cudaStream_t st) {
  CUtensorMap tmK = {}, tmV = {};
  if (!Q8) {
    int rc = cb_make_tmap_2d(&tmK, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, a.kpool, (uint64_t)slots, (uint64_t)a.nkv * HD, (uint64_t)a.nkv * HD, kPage, 64);
    if (!rc) rc = cb_make_tmap_2d(&tmV, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, a.vpool, (uint64_t)slots, (uint64_t)a.nkv * HD, (uint64_t)a.nkv * HD, kPage, 64);
    if (rc) return rc;
  }
  const size_t smem = TreeRing<HD, Q8, PAIR>::bytes;
  auto kern = tree_cache_kernel<HD, Q8, PAIR>;
  static SmemLimit limit;
  std::lock_guard<std::mutex> lock(limit.held);
  cudaError_t e = limit.set(kern, smem);
  if (e != cudaSuccess) return (int)e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(PAIR ? 2 * a.workers : a.workers));
  cfg.blockDim = dim3(Q8 ? 352 + kLoaders : 352);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (g_cb_use_pdl) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (PAIR) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = 2;
    attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
    ++n;
  }
  cfg.attrs = attr;
  cfg.numAttrs = (unsigned)n;
  if (g_cb_trace_names) cb_trace_name((const void*)kern);
  return (int)cudaLaunchKernelEx(&cfg, kern, tmK, tmV, a);
}

template <int HD, bool Q8>
int launch_tree(const TreeAttnArgs& a, int64_t slots, cudaStream_t st) {
  int rc;
  if constexpr (HD >= 128) rc = a.span > kRows ? launch_cache<HD, Q8, true>(a, slots, st) : launch_cache<HD, Q8, false>(a, slots, st);
  else rc = launch_cache<HD, Q8, false>(a, slots, st);
  if (rc) return rc;
  const int64_t tasks = (int64_t)a.R * a.C * a.nh;
  return (int)cb_launch_second(tree_finish_kernel<HD, Q8>, dim3((unsigned)((tasks + 7) / 8)), dim3(256), 0, st, a);
}

}  // namespace

// part: (ctas * min(rows, 128) + R * nkv * (rows <= 128 ? rows : rows rounded up to 256)) * (hd + 2) + 1 floats, rows = C * nh / nkv; `ctas` is even
CB_EXPORT int cb_attn_tree(const void* q, const void* gate, int64_t ldg, const void* kpool, const void* vpool, int64_t slots,
                           const void* kscale, const void* vscale, const void* tables, int64_t ldbt, int64_t width, const void* positions,
                           const void* anc, void* out, int64_t ldo, void* part, int64_t ctas, int64_t R, int64_t C, int64_t nh, int64_t nkv,
                           int64_t hd, void* status, void* stream) {
  if (!q || !kpool || !vpool || !tables || !positions || !anc || !out || !part || !status) return CB_ERR_ARG;
  if ((kscale == nullptr) != (vscale == nullptr)) return CB_ERR_ARG;
  if (R < 1 || C < 1 || C > kMaxNodes || nkv < 1 || nh < 1 || nh % nkv || ctas < 2 || ctas % 2 || ctas > 65534 || width < 1 || width > (1 << 24) ||
      R * C * nh > (1ll << 30) || R * width * nkv * ((C * (nh / nkv) + kRows - 1) / kRows) > 0x7fff0000 || slots > 0x7fffffff || ((uintptr_t)part & 15))
    return CB_ERR_SHAPE;
  // More than 128 rows a kv head: pairs of CTAs, each with half of every page.  (64 channels a head cannot be halved.)
  const int64_t rows = C * (nh / nkv), span = rows > kRows && hd >= 128 ? 2 * kRows : kRows, workers = span > kRows ? ctas / 2 : ctas;
  const int64_t tiles = (rows + span - 1) / span, used = rows < span ? rows : span;
  const int64_t places = (workers + R * nkv * tiles) * used;
  TreeAttnArgs a{(const bf16*)q, (const bf16*)gate, ldg, kpool, vpool, (const float*)kscale, (const float*)vscale, (const int*)tables, ldbt,
                 (int)width, (int)(slots / kPage), (const int*)positions, (const int64_t*)anc, (bf16*)out, ldo, (float*)part,
                 (float*)part + places * hd, (int*)part + places * (hd + 2), (int)R, (int)C, (int)nh, (int)nkv, (int)(nh / nkv), (int)span,
                 (int)tiles, (int)used, (int)workers,
                 1.4426950408889634f / sqrtf((float)hd), (int*)status};
  cudaStream_t st = (cudaStream_t)stream;
  if (hd == 256) return kscale ? launch_tree<256, true>(a, slots, st) : launch_tree<256, false>(a, slots, st);
  if (hd == 128) return kscale ? launch_tree<128, true>(a, slots, st) : launch_tree<128, false>(a, slots, st);
  if (hd == 64) return kscale ? launch_tree<64, true>(a, slots, st) : launch_tree<64, false>(a, slots, st);
  return CB_ERR_SHAPE;
}
