// Attention of one query token per request over the 8-bit page cache.
//
// The codes go into the tensor cores as they lie in the cache; nothing is converted. With keys
// k = ks·K, values v = vs·V (K, V the e4m3 codes of a page, ks, vs its scales) and the heads of a
// group as columns:
//   * logits:  Sᵀ = K·Qᵀ, tcgen05 kind::f8f6f4, M = 128 keys. The 16-bit q enters as three e4m3
//     parts, q = a·(q₁ + q₂/16 + q₃/256), a the power of two that puts the row's largest entry into
//     [128, 256): each part takes what the ones before left, 4 bits at a time, so 16-bit entries
//     are met exactly but for 2^-26 of the row's largest. The parts are columns of one MMA and are
//     added in fp32.
//   * weights: w = exp2(s − M) in fp32 with s = c·ks·Σ…, their sum l in fp32. V needs the weight
//     times its page's scale, so the reference M is the running maximum of s + log2 vs: then
//     p = 256·w·vs ≤ 256 whatever the scales are. M is only raised, and the sums rescaled, when it
//     would grow by more than 2^0.8, so p ≤ 446 fits e4m3 (448).
//   * values:  Oᵀ += Vᵀ·Pᵀ, M = 128 dimensions, p as four e4m3 parts, p₁ + p₂/16 + p₃/256 + p₄/4096:
//     16 bits of each weight, in steps of 2^-21: what a weight loses is at most 2^-30 of the largest
//     w·vs. (A page louder than the others counts with its scale, whatever its tokens' weights are.)
//     Three parts of p ≤ 16 in the same columns lost what lay below 2^-22 of the largest, a third of
//     the result where one key of value zero stood 23 bits above 16384 others.
//   * o = Oᵀ/(256·l).
//
// Bound by HBM: 2 bytes per key, kv head and dimension. Per tile of 128 keys and 256 dimensions
// (64 KB, 1.5 µs of one SM's share of HBM) the MMAs are 16 instructions of N = 32 and the softmax
// 8 exponentials a thread, so one warpgroup hides behind the loads; narrower heads load faster and
// get two or three CTAs per SM. Measured: 64 requests of 8192 tokens, 32 heads on 8 of 128, 169 us in
// pages of 128 (6380 GB/s, 97 % of the measured copy rate) and 181 us in pages of 16; of lengths 1 to
// 16384, 186 us (5850 GB/s). Groups of 8 heads 204 us, of 16 395 us: there the softmax bounds it. Short
// requests are bound by latency: one of 1005 tokens takes 9.8 us, 32 of 700 to 1100 14.8 us.
//
// Work split: the tiles of all (request, kv head) units are numbered in one row and every CTA takes
// an equal, contiguous share, whatever the lengths are; when that is only a few tiles, as many CTAs as
// there are take pieces of whole units instead. A unit that lies in several CTAs leaves
// partials (unnormalised sums, M, l) that a second kernel joins in the order of the CTAs, so results
// do not depend on timing.
//
// Warp roles: warp 0 producer (a lane per page: TMA boxes of one page into a ring of K and V tiles),
// warp 1 MMA issuer, warps 2-5 softmax and output (a thread per key, then per dimension).
#pragma once

#include "paged_common.cuh"
#include "paged_tc.cuh"

namespace pi0 {
namespace paged {

struct DecodeArgs {
  const void* q;       // [batch, heads, head_dim]
  void* out;
  int64_t q_tok, q_head, o_tok, o_head;
  Cache cache;
  const int* table;    // [batch, max_pages]
  int64_t table_stride;
  const int* kv_lens;
  int* err;
  float* ws;           // partials of the tensor-core form
  float c;             // logit scale · log2 e
  int batch, heads, max_pages;
};

template <typename T>
struct PagedKV {
  const Cache* c;
  const int* table;
  int head;
  __device__ __forceinline__ int64_t ph(int j) const {
    return (int64_t)table[j / c->page_size] * c->kv_heads + head;
  }
  __device__ __forceinline__ void k8(int j, int d, float (&x)[8]) const {
    const int64_t p = ph(j);
    load8(c->k + (p * c->page_size + j % c->page_size) * c->head_dim + d, c->ks[p], x);
  }
  __device__ __forceinline__ void v8(int j, int d, float (&x)[8]) const {
    const int64_t p = ph(j);
    load8(c->v + (p * c->page_size + j % c->page_size) * c->head_dim + d, c->vs[p], x);
  }
};

// a request's length, held to what its table row can hold
__device__ __forceinline__ int held_len(const DecodeArgs& a, int b, bool report) {
  const int64_t most = (int64_t)a.max_pages * a.cache.page_size;
  const int n = a.kv_lens[b];
  if (n >= 0 && n <= most) return n;
  if (report) set_err(a.err, PI0_PAGED_ERR_TABLE);
  return n < 0 ? 0 : (int)min(most, (int64_t)0x7fffffff);
}

// Cached tokens of request b that can be read: its length, held to its table row and to the pages
// before the first number that names no page of the pool. Uniform over the warp.
__device__ __forceinline__ int readable_len(const DecodeArgs& a, int b) {
  const int lane = threadIdx.x & 31, ps = a.cache.page_size;
  const int n = held_len(a, b, lane == 0);
  const int* row = a.table + b * a.table_stride;
  const int pages = (int)(((int64_t)n + ps - 1) / ps);
  for (int p = 0; p < pages; p += 32) {
    const bool bad = p + lane < pages && (unsigned)row[p + lane] >= (unsigned)a.cache.num_pages;
    const unsigned any = __ballot_sync(~0u, bad);
    if (any) {
      if (lane == 0) set_err(a.err, PI0_PAGED_ERR_PAGE);
      return (p + __ffs(any) - 1) * ps;
    }
  }
  return n;
}

// One warp per (request, head), for the head and page sizes without a tensor-core form: a key at a time,
// 0.8 us each. 32 requests of 900 tokens take 710 us in pages of 24 or 48 (16 us in pages of 64), one
// of 16384 tokens with heads of 96 12.9 ms.
template <typename T>
__global__ void __launch_bounds__(32) paged_rows_kernel(DecodeArgs a) {
  const int b = blockIdx.y, h = blockIdx.x;
  const int n = readable_len(a, b);
  const PagedKV<T> kv{&a.cache, a.table + b * a.table_stride, h / (a.heads / a.cache.kv_heads)};
  attend_row(reinterpret_cast<const T*>(a.q) + b * a.q_tok + h * a.q_head, a.cache.head_dim, n, a.c,
             kv, reinterpret_cast<T*>(a.out) + b * a.o_tok + h * a.o_head);
}

// ---- tensor-core form -----------------------------------------------------------------------------

constexpr int kDecTile = 128;          // keys per tile
constexpr int kDecThreads = 192;
constexpr int kWholeTiles = 8;         // pieces of up to so many tiles keep to one unit
constexpr int kWholeTries = 4;         // lengths tried: the least that could do, and some more
constexpr float kDecTop = 256.f;       // the weight at M, as it enters the product
constexpr float kDecGrow = 0.8f;       // M is raised when it would grow by more than 2^0.8

template <int HD, int NH>
struct DecCfg {
  static constexpr int ROW = HD < 128 ? HD : 128;   // bytes of a tile row, the swizzle span
  static constexpr int HB = (HD + 127) / 128;       // 128-wide blocks of the head dimension
  static constexpr int SLOT = kDecTile * HD;        // a K or a V tile
  static constexpr int BLOCK = kDecTile * ROW;      // one 128-wide block of it
  // columns: parts × heads (the fourth of q is empty), then empty ones; COLS of them are read back
  static constexpr int N = NH < 8 ? 32 : 4 * NH;
  static constexpr int COLS = 4 * NH;
  static constexpr int Q_BYTES = N * HD;
  static constexpr int P_BYTES = kDecTile * N;
  static constexpr int FIXED = Q_BYTES + 2 * P_BYTES + 1024;
  // CTAs per SM: a narrow head's tile loads faster than one softmax warpgroup takes it (16 heads:
  // no registers for a second)
  static constexpr int OCC = HD == 256 || NH > 8 ? 1 : HD == 64 && NH == 4 ? 3 : 2;
  static constexpr int ROOM = (OCC == 1 ? 225 : OCC == 2 ? 110 : 72) * 1024 - FIXED;
  static constexpr int SLOTS = (ROOM / SLOT) & ~1;
  static constexpr int SMEM = SLOTS * SLOT + FIXED;
  static constexpr int S_COL = 0, O_COL = 2 * N;
  static constexpr int USED = O_COL + HB * N;
  static constexpr int TMEM = USED <= 128 ? 128 : 256;
  // a partial: NH rows of HD sums, then M and l of each head
  static constexpr int PARTIAL = NH * HD + 2 * NH;
};

// what a CTA leaves for the joining kernel about the unit that begins in it and goes on in others
struct DecMeta {
  int batch, head, heads, count;
};

// A CTA's tiles as pieces, each a run of tiles of one unit. Every role walks the same pieces.
struct DecWalk {
  const DecodeArgs& a;
  int subs;            // units per request: kv heads × chunks of their heads
  int b, sub, t0;      // next tile
  int rem;             // tiles left
  int n, nt, take;     // the piece: tokens and tiles of its unit, tiles taken
  __device__ __forceinline__ bool next() {
    if (rem <= 0) return false;
    for (;;) {
      if (b >= a.batch) return false;
      n = held_len(a, b, false);
      nt = (int)(((int64_t)n + kDecTile - 1) / kDecTile);
      if (nt > 0) break;
      ++b;
    }
    take = min(rem, nt - t0);
    return true;
  }
  __device__ __forceinline__ void done() {
    rem -= take;
    t0 += take;
    if (t0 == nt) {
      t0 = 0;
      if (++sub == subs) {
        sub = 0;
        ++b;
      }
    }
  }
};

// two floats to e4m3 codes, saturating (NaN stays NaN), low byte first
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
  return (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E4M3);
}

// The e4m3 number nearest to x, |x| ≤ 448, ties to even: steps of 2^-3 of x's binade, of 2^-9 below
// 2^-6. Adding 1.5·2^20 times that binade leaves exactly these steps as the last bit of an fp32.
__device__ __forceinline__ float on_e4m3(float x) {
  const uint32_t binade = max(__float_as_uint(x) & 0x7f800000u, 0x3c800000u);
  const float big = __uint_as_float(binade + 0x0a400000u);
  return __fsub_rn(__fadd_rn(x, big), big);
}

// x = p₁ + p₂/16 + p₃/256 …, each an e4m3 code: the codes of two values for each part
template <int PARTS>
__device__ __forceinline__ void split(float x, float y, uint32_t (&part)[PARTS]) {
#pragma unroll
  for (int i = 0; i < PARTS; ++i) {
    part[i] = e4m3x2(x, y);
    if (i + 1 == PARTS) break;
    x = (x - on_e4m3(x)) * 16.f;
    y = (y - on_e4m3(y)) * 16.f;
  }
}

template <typename T, int HD, int NH>
__global__ void __launch_bounds__(kDecThreads, DecCfg<HD, NH>::OCC)
    paged_decode_kernel(const __grid_constant__ CUtensorMap tmK,
                        const __grid_constant__ CUtensorMap tmV, DecodeArgs a) {
  using C = DecCfg<HD, NH>;
  constexpr int N = C::N, ROW = C::ROW;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  uint8_t* sQ = base + C::SLOTS * C::SLOT;
  uint8_t* sP = sQ + C::Q_BYTES;
  __shared__ __align__(8) uint64_t full[C::SLOTS], empty[C::SLOTS], q_full, s_full[2], s_free[2],
      p_full[2], pv_done[2], drain;
  __shared__ uint32_t s_tmem;
  __shared__ float s_red[2][4][NH], s_qa[NH], s_l[4][NH];
  __shared__ int s_scan[1 + kWholeTries][kDecThreads / 32], s_begin, s_total, s_whole, s_rem, s_at[3], s_stop;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const Waits waits{a.err, &s_stop};
  const int group = a.heads / a.cache.kv_heads, chunks = (group + NH - 1) / NH;
  const int subs = a.cache.kv_heads * chunks;
  const int ps = a.cache.page_size, ctas = gridDim.x, cta = blockIdx.x;
  pdl_trigger();  // every CTA of this grid is resident at once: the joining blocks may move in

  if (tid == 0) {
    for (int i = 0; i < C::SLOTS; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    mbar_init(&q_full, 4);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&s_free[i], 4);
      mbar_init(&p_full[i], 4);
      mbar_init(&pv_done[i], 1);
    }
    mbar_init(&drain, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
    s_stop = 0;
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(&s_tmem)),
                 "r"((uint32_t)C::TMEM));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }

  // ---- this CTA's share: tiles before each thread's requests, then where the share begins ----
  {
    const int per = (a.batch + kDecThreads - 1) / kDecThreads;
    const int b0 = min(a.batch, tid * per), b1 = min(a.batch, b0 + per);
    auto tiles_of = [&](int b, bool report) {
      return (int)(((int64_t)held_len(a, b, report) + kDecTile - 1) / kDecTile);
    };
    int mine[1 + kWholeTries] = {};  // tiles; and CTAs of whole pieces of each length tried
    for (int b = b0; b < b1; ++b) mine[0] += tiles_of(b, cta == 0) * subs;
    // sums of the first n numbers over the threads before this one, and over all
    int before[1 + kWholeTries], all[1 + kWholeTries];
    auto scan = [&](int from, int to) {
#pragma unroll
      for (int v = 0; v <= kWholeTries; ++v) {
        if (v < from || v >= to) continue;
        int inc = mine[v];
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
          const int up = __shfl_up_sync(~0u, inc, d);
          if (lane >= d) inc += up;
        }
        if (lane == 31) s_scan[v][warp] = inc;
        before[v] = inc - mine[v];
      }
      __syncthreads();
#pragma unroll
      for (int v = 0; v <= kWholeTries; ++v) {
        if (v < from || v >= to) continue;
        all[v] = 0;
#pragma unroll
        for (int w = 0; w < kDecThreads / 32; ++w) {
          if (w < warp) before[v] += s_scan[v][w];
          all[v] += s_scan[v][w];
        }
      }
    };
    scan(0, 1);
    const int total = all[0], most = (total + ctas - 1) / ctas;
    int whole = 0, x0 = Shares<int>(total, ctas).begin(cta, total), b_before = before[0], b_mine = mine[0];
    if (total > 0 && most <= kWholeTiles) {
      // Few tiles: pieces of `whole` tiles that never cross from one unit into another, if there
      // are CTAs enough, as beginning and ending a unit costs more than a tile or two.
      for (int b = b0; b < b1; ++b) {
        const int nt = tiles_of(b, false);
#pragma unroll
        for (int v = 0; v < kWholeTries; ++v) mine[1 + v] += subs * ((nt + most + v - 1) / (most + v));
      }
      scan(1, 1 + kWholeTries);
#pragma unroll
      for (int v = kWholeTries - 1; v >= 0; --v)
        if (all[1 + v] <= ctas && v <= 1 + most / 2) {
          whole = most + v;
          x0 = cta < all[1 + v] ? cta : -1;
          b_before = before[1 + v];
          b_mine = mine[1 + v];
        }
    }
    if (tid == 0) {
      s_begin = x0;
      s_total = total;
      s_whole = whole;
      s_rem = 0;
    }
    __syncthreads();
    if (x0 >= b_before && x0 < b_before + b_mine) {
      int x = x0 - b_before;
      for (int b = b0; b < b1; ++b) {
        const int nt = tiles_of(b, false), each = whole ? (nt + whole - 1) / whole : nt;
        if (x < each * subs) {
          s_at[0] = b;
          s_at[1] = x / each;
          s_at[2] = x % each * (whole ? whole : 1);
          s_rem = whole ? min(whole, nt - s_at[2])
                        : Shares<int>(total, ctas).begin(cta + 1, total) - x0;
          break;
        }
        x -= each * subs;
      }
    }
    // requests without tokens: zeros
    for (int b = cta; b < a.batch; b += ctas)
      if (held_len(a, b, false) == 0)
        for (int i = tid; i < a.heads * (HD / 8); i += kDecThreads)
          *reinterpret_cast<uint4*>(reinterpret_cast<T*>(a.out) + b * a.o_tok +
                                    (i / (HD / 8)) * a.o_head + (i % (HD / 8)) * 8) =
              make_uint4(0, 0, 0, 0);
  }
  // the empty fourth part of Q, whose columns nobody reads
  for (int i = tid; i < C::Q_BYTES / 16; i += kDecThreads)
    reinterpret_cast<uint4*>(sQ)[i] = make_uint4(0, 0, 0, 0);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_tmem;
  const Shares<int> shares(s_total, ctas);
  const int whole_tiles = s_whole;
  DecWalk w{a, subs, s_at[0], s_at[1], s_at[2], s_rem, 0, 0, 0};

  if (warp == 0) {
    // ---- producer: one lane per box ----
    int slot = 0, loads = 0;
    uint32_t ph = 0;
    bool ok = true;
    constexpr int kMaxBoxes = kDecTile / 8;
    const int box = min(ps, kDecTile), boxes = kDecTile / box;  // boxes ≤ 16 per 128-wide block
    while (ok && w.next()) {
      const int kv = w.sub / chunks;
      const int* row = a.table + w.b * a.table_stride;
      for (int i = 0; i < w.take && ok; ++i) {
        const int key0 = (w.t0 + i) * kDecTile, key = key0 + lane * box;
        int page = -1;
        if (lane < boxes && key < w.n) {
          page = row[key / ps];
          if ((unsigned)page >= (unsigned)a.cache.num_pages) {
            set_err(a.err, PI0_PAGED_ERR_PAGE);
            page = -1;
          }
        }
        const int valid = __popc(__ballot_sync(~0u, page >= 0));
        const int z = page * a.cache.kv_heads + kv, y = key % ps;
#pragma unroll
        for (int half = 0; half < 2; ++half) {  // K, then V
          int good = 1;
          if (lane == 0) {
            if (loads >= C::SLOTS)
              good = mbar_wait(&empty[slot], ph ^ 1, waits, tc::ERR_TIMEOUT_PRODUCER);
            if (good) mbar_expect_tx(&full[slot], (uint32_t)(valid * box * HD));
          }
          ok = __shfl_sync(~0u, good, 0);
          if (!ok) break;
          if (page >= 0) {
            uint8_t* dst = base + slot * C::SLOT + lane * box * ROW;
#pragma unroll
            for (int hb = 0; hb < C::HB; ++hb)
              tma_load_3d(dst + hb * C::BLOCK, half ? &tmV : &tmK, &full[slot], hb * 128, y, z);
          }
          ++loads;
          if (++slot == C::SLOTS) {
            slot = 0;
            ph ^= 1;
          }
        }
      }
      w.done();
    }
    static_assert(kMaxBoxes <= 32, "a lane per box");
    // no copy into this CTA's shared memory may be in flight when it exits
    if (lane == 0)
      for (int i = max(0, loads - C::SLOTS); i < loads; ++i)
        mbar_wait(&full[i % C::SLOTS], (i / C::SLOTS) & 1, waits, tc::ERR_TIMEOUT_PRODUCER, false);
    __syncwarp();
  } else if (warp == 1) {
    // ---- MMA issuer ----
    constexpr uint32_t id_s = idesc_e4m3(128, N, false, false);
    constexpr uint32_t id_o = idesc_e4m3(128, N, true, true);
    const uint32_t ring = __shfl_sync(~0u, smem_u32(base), 0), tm = __shfl_sync(~0u, tmem, 0);
    const uint32_t qs = ring + C::SLOTS * C::SLOT, pb = qs + C::Q_BYTES;
    bool ok = true;
    int g = 0, piece = 0;  // tiles and pieces so far
    // tile g of the CTA has its K in load 2g and its V in load 2g + 1
    auto full_of = [&](int load) {
      return mbar_wait(&full[load % C::SLOTS], (load / C::SLOTS) & 1, waits, tc::ERR_TIMEOUT_MMA);
    };
    auto qk = [&](int i) -> bool {
      const int slot = (2 * i) % C::SLOTS;
      if (!full_of(2 * i)) return false;
      if (i >= 2 && !mbar_wait(&s_free[i & 1], ((i >> 1) - 1) & 1, waits, tc::ERR_TIMEOUT_MMA))
        return false;
      tc_fence_after();
      const uint64_t dk = sdesc<ROW>(ring + slot * C::SLOT, 8 * ROW, 0);
      const uint64_t dq = sdesc<ROW>(qs, 8 * ROW, 0);
      if (elect_one()) {
#pragma unroll
        for (int k = 0; k < HD / 32; ++k) {
          constexpr int PER = ROW / 32;  // steps of 32 bytes in a row
          umma_f8(tm + C::S_COL + (i & 1) * N, dk + (k / PER * C::BLOCK + k % PER * 32) / 16,
                  dq + (k / PER * (N * ROW) + k % PER * 32) / 16, id_s, k != 0);
        }
        umma_commit(&s_full[i & 1]);
        umma_commit(&empty[slot]);
      }
      __syncwarp();
      return true;
    };
    auto pv = [&](int i, bool first) -> bool {
      const int slot = (2 * i + 1) % C::SLOTS;
      if (!full_of(2 * i + 1) ||
          !mbar_wait(&p_full[i & 1], (i >> 1) & 1, waits, tc::ERR_TIMEOUT_MMA))
        return false;
      tc_fence_after();
      // 64-wide heads: both halves of M read the same 64 dimensions (lbo 0)
      const uint64_t dv = sdesc<ROW>(ring + slot * C::SLOT, 8 * ROW, 0);
      const uint64_t dp = sdesc<N>(pb + (i & 1) * C::P_BYTES, 8 * N, 0);
      const uint32_t more = !first;
      if (elect_one()) {
#pragma unroll
        for (int hb = 0; hb < C::HB; ++hb)
#pragma unroll
          for (int k = 0; k < kDecTile / 32; ++k)  // 32 keys a step
            umma_f8(tm + C::O_COL + hb * N, dv + (hb * C::BLOCK + k * 32 * ROW) / 16,
                    dp + k * 32 * N / 16, id_o, k == 0 ? more : 1u);
        umma_commit(&pv_done[i & 1]);
        umma_commit(&empty[slot]);
      }
      __syncwarp();
      return true;
    };
    while (ok && w.next()) {
      ok = mbar_wait(&q_full, piece & 1, waits, tc::ERR_TIMEOUT_MMA) && qk(g);
      for (int i = 0; i < w.take && ok; ++i, ++g) {
        if (i + 1 < w.take) ok = qk(g + 1);
        ok = ok && pv(g, i == 0);
      }
      ++piece;
      w.done();
    }
    // every issued MMA completes before TMEM is released
    if (elect_one()) umma_commit(&drain);
    __syncwarp();
    mbar_wait(&drain, 0, waits, tc::ERR_TIMEOUT_MMA, false);
  } else {
    // ---- softmax and output: warps 2-5 ----
    const int q4 = warp & 3, r = q4 * 32 + lane;
    const uint32_t tlane = tmem + ((uint32_t)(q4 * 32) << 16);
    constexpr int STEP = C::COLS < 32 ? 16 : 32;  // columns read at a time
    bool ok = true;
    int g = 0;
    int x = s_begin;
    DecMeta meta{0, 0, 0, 0};
    while (w.next()) {
      const int kv = w.sub / chunks, h0 = kv * group + (w.sub % chunks) * NH;
      const int nh = min(NH, group - (w.sub % chunks) * NH);
      // q in three parts, a warp per head; every QK of the piece before has been read by now
      constexpr int E = HD / 32;                    // entries of a row per lane
      __align__(16) T qraw[NH / 4][E];
#pragma unroll
      for (int u = 0; u < NH / 4; ++u) {            // all rows of the warp are requested at once
        const T* q = reinterpret_cast<const T*>(a.q) + w.b * a.q_tok +
                     (h0 + min(q4 + 4 * u, nh - 1)) * a.q_head + lane * E;
        if constexpr (E == 8) *reinterpret_cast<uint4*>(qraw[u]) = *reinterpret_cast<const uint4*>(q);
        else if constexpr (E == 4) *reinterpret_cast<uint2*>(qraw[u]) = *reinterpret_cast<const uint2*>(q);
        else *reinterpret_cast<uint32_t*>(qraw[u]) = *reinterpret_cast<const uint32_t*>(q);
      }
#pragma unroll
      for (int u = 0; u < NH / 4; ++u) {
        const int h = q4 + 4 * u;
        float v[E];
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = h < nh ? Tr<T>::f(qraw[u][e]) : 0.f;
        float am = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) am = fmaxf(am, isfinite(v[e]) ? fabsf(v[e]) : 0.f);
        am = warp_max_f32(am);
        // 2^k with am·2^-k in [128, 256); a row of zeros takes the smallest
        const int k = max((int)(__float_as_uint(am) >> 23) - 127, -100) - 7;
        const float inv = __uint_as_float((uint32_t)(127 - k) << 23);
        if (lane == 0) s_qa[h] = __uint_as_float((uint32_t)(127 + k) << 23) * a.c;
        uint16_t codes[3][E / 2];
#pragma unroll
        for (int e = 0; e < E; e += 2) {
          uint32_t part[3];
          // an infinite entry has no code and makes the whole row NaN, as every logit would be
          const float y0 = isinf(v[e]) ? NAN : v[e] * inv, y1 = isinf(v[e + 1]) ? NAN : v[e + 1] * inv;
          split(y0, y1, part);
#pragma unroll
          for (int p = 0; p < 3; ++p) codes[p][e / 2] = (uint16_t)part[p];
        }
#pragma unroll
        for (int p = 0; p < 3; ++p) {
          const uint32_t d = lane * E, n = p * NH + h;
          uint8_t* dst = sQ + (d / 128) * (N * ROW) + swz<ROW>(n * ROW + d % 128);
#pragma unroll
          for (int e = 0; e < E / 2; ++e) reinterpret_cast<uint16_t*>(dst)[e] = codes[p][e];
        }
      }
      fence_async_smem();
      named_sync<1, 128>();  // s_qa
      if (lane == 0) mbar_arrive(&q_full);

      float m[NH], l[NH], qa[NH];
#pragma unroll
      for (int h = 0; h < NH; ++h) {
        m[h] = -INFINITY;
        l[h] = 0.f;
        qa[h] = s_qa[h];
      }
      const int* row = a.table + w.b * a.table_stride;
      // page of this thread's key in tile t (−1: none), and its scales
      auto page_of = [&](int t) -> int {
        const int key = t * kDecTile + r;
        if (t >= w.t0 + w.take || key >= w.n) return -1;
        const int p = row[key / ps];
        return (unsigned)p < (unsigned)a.cache.num_pages ? p : -1;
      };
      auto scales_of = [&](int page) -> float2 {
        if (page < 0) return make_float2(0.f, 0.f);
        const int64_t i = (int64_t)page * a.cache.kv_heads + kv;
        return make_float2(__ldg(a.cache.ks + i), __ldg(a.cache.vs + i));
      };
      int page = page_of(w.t0), page1 = page_of(w.t0 + 1);
      float2 sc = scales_of(page);
      for (int i = 0; i < w.take; ++i, ++g) {
        // the next tile's scales and the page after it are requested a tile ahead
        const float2 sc1 = scales_of(page1);
        const int page2 = page_of(w.t0 + i + 2);
        const int buf = g & 1;
        if (ok) ok = mbar_wait(&s_full[buf], (g >> 1) & 1, waits, tc::ERR_TIMEOUT_EPI);
        ok = __all_sync(~0u, ok);
        float s[NH];
        if (ok) {
          tc_fence_after();
#pragma unroll
          for (int n0 = 0; n0 < C::COLS; n0 += STEP) {
            uint32_t raw[STEP];
            tmem_ld_cols(tlane + C::S_COL + buf * N + n0, raw);
#pragma unroll
            for (int j = 0; j < STEP; ++j) {
              const int p = (n0 + j) / NH, h = (n0 + j) % NH;
              const float f = __uint_as_float(raw[j]);
              if (p == 0) s[h] = f;
              else if (p == 1) s[h] = fmaf(f, 1.f / 16.f, s[h]);
              else if (p == 2) s[h] = fmaf(f, 1.f / 256.f, s[h]);
            }
          }
          tc_fence_before();
        }
        __syncwarp();
        if (ok && lane == 0) mbar_arrive(&s_free[buf]);
        const float lv = fmaxf(__log2f(sc.y), -126.f);
#pragma unroll
        for (int h = 0; h < NH; ++h) {
          s[h] = page < 0 || !ok ? -INFINITY : s[h] * (sc.x * qa[h]);
          const float mx = warp_max_f32(s[h] + lv);
          if (lane == 0) s_red[buf][q4][h] = mx;
        }
        named_sync<1, 128>();
        float top[NH];
        bool grow = false;
#pragma unroll
        for (int h = 0; h < NH; ++h) {
          top[h] = fmaxf(fmaxf(s_red[buf][0][h], s_red[buf][1][h]),
                         fmaxf(s_red[buf][2][h], s_red[buf][3][h]));
          grow |= top[h] > m[h] + kDecGrow;
        }
        // P's buffer is free once the P·V of two tiles ago has finished; O may be rescaled once
        // the last one has
        if (ok && g >= 2)
          ok = mbar_wait(&pv_done[buf], ((g >> 1) - 1) & 1, waits, tc::ERR_TIMEOUT_EPI);
        if (i == 0) {
#pragma unroll
          for (int h = 0; h < NH; ++h) m[h] = top[h];
        } else if (grow) {  // the same for all 128 threads
          if (ok) ok = mbar_wait(&pv_done[buf ^ 1], ((g - 1) >> 1) & 1, waits, tc::ERR_TIMEOUT_EPI);
          ok = __all_sync(~0u, ok);
          float al[NH];
#pragma unroll
          for (int h = 0; h < NH; ++h) {
            al[h] = 1.f;
            if (top[h] > m[h] + kDecGrow) {
              al[h] = m[h] == -INFINITY ? 0.f : exp2_fast(m[h] - top[h]);
              m[h] = top[h];
              l[h] *= al[h];
            }
          }
          if (ok) {
            tc_fence_after();
#pragma unroll
            for (int c0 = 0; c0 < C::HB * C::COLS; c0 += STEP) {
              const uint32_t at = tlane + C::O_COL + c0 / C::COLS * N + c0 % C::COLS;
              uint32_t o[STEP];
              tmem_ld_cols(at, o);
#pragma unroll
              for (int j = 0; j < STEP; ++j)
                o[j] = __float_as_uint(__uint_as_float(o[j]) * al[(c0 + j) % NH]);
              tmem_st_cols(at, o);
            }
            tmem_wait_st();
            tc_fence_before();
          }
        }
        ok = __all_sync(~0u, ok);
        // weights, in four parts each, as this key's row of P: N consecutive bytes
        uint32_t word[4][NH / 4];
#pragma unroll
        for (int h = 0; h < NH; h += 2) {
          const float r0 = m[h] == -INFINITY ? 0.f : m[h];
          const float r1 = m[h + 1] == -INFINITY ? 0.f : m[h + 1];
          const float e0 = exp2_fast(s[h] - r0), e1 = exp2_fast(s[h + 1] - r1);
          l[h] += e0;
          l[h + 1] += e1;
          uint32_t part[4];
          const float f = kDecTop * sc.y;
          split(e0 * f, e1 * f, part);
#pragma unroll
          for (int p = 0; p < 4; ++p) {
            if (h % 4 == 0) word[p][h / 4] = part[p];
            else word[p][h / 4] |= part[p] << 16;
          }
        }
        if (ok) {
          uint8_t* p = sP + buf * C::P_BYTES;
#pragma unroll
          for (int n0 = 0; n0 < C::COLS; n0 += 16) {
            uint4 q;
            uint32_t* qw = reinterpret_cast<uint32_t*>(&q);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const int n = n0 + 4 * j;
              qw[j] = word[n / NH][(n % NH) / 4];
            }
            *reinterpret_cast<uint4*>(p + swz<N>(r * N + n0)) = q;
          }
          // a key that is none: its weight is zero, and so must its V row be, which is whatever
          // lay in the page or in the ring
          if (__any_sync(~0u, page < 0)) {
            const int load = 2 * g + 1, slot = load % C::SLOTS;
            ok = mbar_wait(&full[slot], (load / C::SLOTS) & 1, waits, tc::ERR_TIMEOUT_EPI);
            ok = __all_sync(~0u, ok);
            if (ok && page < 0)
#pragma unroll
              for (int d = 0; d < HD; d += 16)  // a whole row: the swizzle only permutes it
                *reinterpret_cast<uint4*>(base + slot * C::SLOT + (d / 128) * C::BLOCK + r * ROW +
                                          d % 128) = make_uint4(0, 0, 0, 0);
          }
        }
        fence_async_smem();
        __syncwarp();
        if (ok && lane == 0) mbar_arrive(&p_full[buf]);
        page = page1;
        page1 = page2;
        sc = sc1;
      }
      // ---- the piece's sums: l while the last P·V runs ----
#pragma unroll
      for (int h = 0; h < NH; ++h) {
        const float sum = warp_sum(l[h]);
        if (lane == 0) s_l[q4][h] = sum;
      }
      named_sync<1, 128>();
      float inv[NH];
#pragma unroll
      for (int h = 0; h < NH; ++h) {
        l[h] = (s_l[0][h] + s_l[1][h]) + (s_l[2][h] + s_l[3][h]);
        inv[h] = 1.f / (kDecTop * l[h]);
      }
      if (ok) ok = mbar_wait(&pv_done[(g - 1) & 1], ((g - 1) >> 1) & 1, waits, tc::ERR_TIMEOUT_EPI);
      ok = __all_sync(~0u, ok);
      named_sync<1, 128>();  // s_l may be written again
      const bool whole = w.take == w.nt;
      float* part = a.ws + (size_t)ctas * 4 + ((size_t)cta * 2 + (w.t0 > 0 ? 0 : 1)) * C::PARTIAL;
      tc_fence_after();
#pragma unroll
      for (int hb = 0; hb < C::HB; ++hb) {
        float o[NH];
#pragma unroll
        for (int n0 = 0; n0 < C::COLS; n0 += STEP) {
          uint32_t raw[STEP];
          tmem_ld_cols(tlane + C::O_COL + hb * N + n0, raw);
#pragma unroll
          for (int j = 0; j < STEP; ++j) {
            const int p = (n0 + j) / NH, h = (n0 + j) % NH;
            const float f = ok ? __uint_as_float(raw[j]) : NAN;
            if (p == 0) o[h] = f;
            else if (p == 1) o[h] = fmaf(f, 1.f / 16.f, o[h]);
            else if (p == 2) o[h] = fmaf(f, 1.f / 256.f, o[h]);
            else o[h] = fmaf(f, 1.f / 4096.f, o[h]);
          }
        }
        const int d = hb * 128 + r;
        if (d < HD) {
#pragma unroll
          for (int h = 0; h < NH; ++h) {
            if (h >= nh) break;
            if (whole)
              reinterpret_cast<T*>(a.out)[w.b * a.o_tok + (h0 + h) * a.o_head + d] =
                  Tr<T>::t(o[h] * inv[h]);
            else
              part[h * HD + d] = o[h];
          }
        }
      }
      tc_fence_before();
      if (!whole) {
        if (r == 0)
#pragma unroll
          for (int h = 0; h < NH; ++h) {
            part[NH * HD + h] = m[h];
            part[NH * HD + NH + h] = l[h];
          }
        if (w.t0 == 0) {
          meta = DecMeta{w.b, h0, nh, whole_tiles ? (w.nt + whole_tiles - 1) / whole_tiles
                                                  : shares.owner(x + w.nt - 1) - cta + 1};
        }
      }
      x += w.take;
      w.done();
    }
    if (r == 0) reinterpret_cast<DecMeta*>(a.ws)[cta] = meta;
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem),
                 "r"((uint32_t)C::TMEM));
  }
}

// Joins the partials of the unit that begins in CTA blockIdx.x and ends in another: one block per
// (CTA, head), out = Σ 2^(Mᵢ−M)·oᵢ / (256·Σ 2^(Mᵢ−M)·lᵢ). A thread takes one dimension of every JS-th
// eight partials, whose loads are in flight together; the JS sums are joined in order.
constexpr int kJoinThreads = 512;

template <typename T, int HD, int NH>
__global__ void __launch_bounds__(kJoinThreads) paged_join_kernel(DecodeArgs a, int ctas) {
  using C = DecCfg<HD, NH>;
  constexpr int JS = kJoinThreads / HD;
  __shared__ float s_o[JS][HD], s_m[JS], s_l[JS];
  pdl_wait();
  const int cta = blockIdx.x, h = blockIdx.y, d = threadIdx.x % HD, js = threadIdx.x / HD;
  const DecMeta meta = reinterpret_cast<const DecMeta*>(a.ws)[cta];
  if (h >= meta.heads || meta.count == 0) return;
  const float* first = a.ws + (size_t)ctas * 4 + ((size_t)cta * 2 + 1) * C::PARTIAL;
  // partial i: slot 1 of the first CTA, slot 0 of those behind it
  auto part = [&](int i) { return first + (i == 0 ? 0 : ((size_t)i * 2 - 1) * C::PARTIAL); };
  float M = -INFINITY, o = 0.f, l = 0.f;
  for (int i0 = js * 8; i0 < meta.count; i0 += JS * 8) {
    float pm[8], pl[8], po[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const bool have = i0 + i < meta.count;
      const float* p = part(have ? i0 + i : 0);
      pm[i] = have ? p[NH * HD + h] : -INFINITY;
      pl[i] = have ? p[NH * HD + NH + h] : 0.f;
      po[i] = have ? p[h * HD + d] : 0.f;
    }
    float top = M;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = fmaxf(top, pm[i]);
    const float ref = top == -INFINITY ? 0.f : top, old = exp2f(M - ref);
    o *= old;
    l *= old;
    M = top;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float f = exp2f(pm[i] - ref);
      o = fmaf(f, po[i], o);
      l = fmaf(f, pl[i], l);
    }
  }
  if (meta.count > 8) {  // uniform: a block has one unit
    s_o[js][d] = o;
    if (d == 0) {
      s_m[js] = M;
      s_l[js] = l;
    }
    __syncthreads();
    float top = s_m[0];
#pragma unroll
    for (int j = 1; j < JS; ++j) top = fmaxf(top, s_m[j]);
    const float ref = top == -INFINITY ? 0.f : top;
    o = l = 0.f;
#pragma unroll
    for (int j = 0; j < JS; ++j) {
      const float f = exp2f(s_m[j] - ref);
      o = fmaf(f, s_o[j][d], o);
      l = fmaf(f, s_l[j], l);
    }
  }
  if (js == 0)
    reinterpret_cast<T*>(a.out)[meta.batch * a.o_tok + (meta.head + h) * a.o_head + d] =
        Tr<T>::t(o / (kDecTop * l));
}

}  // namespace paged
}  // namespace pi0
