// Attention over packed prompts: grouped heads, causal with a bidirectional prefix per request.
//
// Query i of a request with Lq new tokens and Lk keys sees the keys j < n(i),
// n(i) = min(Lk, max(i + Lk − Lq + 1, prefix)): always a leading part of the request's keys. A row is
//   o = Σ_j 2^(c·q·k_j − m) v_j / Σ_j 2^(c·q·k_j − m),   c = scale·log2 e,
// in one pass over the keys with a running reference m that is raised, and the sums rescaled, only
// when a row's maximum outgrows it by 2^8 (kLift).
//
// Tensor-core form (head sizes 64, 128, 256). A tile of query rows is the group's heads of as many
// tokens as fit into 128 rows, so heads that share keys share their loads, and a tile of one kv head
// with eight query heads spans 16 tokens: little of its last tile of keys is masked. A CTA works on
// one such tile (256 dimensions: 512 tensor-memory columns hold two tiles of logits and its sums) or
// on two. Per step, 128 queries × 128 keys:
//   * S = Q·Kᵀ, tcgen05 kind::f16, from shared memory into tensor memory;
//   * a thread per row takes its 128 logits into registers, masks, exponentiates, and writes the
//     weights back over the logits in the type of V; P·V starts before the last of them;
//   * O += P·V with P from tensor memory.
// The products of a step take 512, 1024 and 2048 clocks with 64, 128 and 256 dimensions, the
// exponentials 1024 (16 a clock), and each waits for the other: two tiles per CTA work in turns, one in
// its exponentials while the other is in its products. What a step takes with 128 dimensions is 3300 to
// 3600 clocks for two tiles (2048 of products): from logits to logits a tile spends 600 on loading them
// and their maximum, 1450 in its exponentials, 1100 in P·V and the next logits, whose reads of shared
// memory compete with the loads of K and V, and the rest on handing over; power lowers the clock.
// Measured: 8192 tokens, 32 heads on 8 of 128, all keys 849 us (1295 TFLOP/s, 78 % of the measured
// 1661), causal 480 us (1145); 8 heads on 1 of 256, all keys 404 us (1360); 32 heads on 8 of 64, all
// keys 740 us (740), where the exponentials alone are 500 us at the clock that it runs at.
//
// Work split: the steps of all (tile, kv head) are numbered in one row, and every CTA takes an equal,
// contiguous share, whatever the lengths are. What lies in several CTAs leaves partial sums that a
// second kernel joins in the order of the CTAs: eight chunks of up to 300 tokens on 1000 to 4000
// earlier keys take 59 us instead of 85 with a CTA per tile.
#pragma once

#include <type_traits>

#include "paged_common.cuh"
#include "paged_tc.cuh"

namespace pi0 {
namespace paged {

struct PromptArgs {
  const void* q;
  const void* k;
  const void* v;
  void* out;
  int64_t q_tok, q_head, k_tok, k_head, v_tok, v_head, o_tok, o_head;  // strides, elements
  const int* cu_q;
  const int* cu_k;
  const int* prefix;   // or null: causal
  int* err;
  float* ws;           // partials of the tensor-core form
  float c;             // logit scale · log2 e
  int batch, total_q, total_k, heads, kv_heads, head_dim;
};

// first token and length of request r, inside [0, total)
__device__ __forceinline__ void seq_span(const int* cu, int r, int total, int& t0, int& n) {
  t0 = min(max(cu[r], 0), total);
  n = min(max(cu[r + 1], t0), total) - t0;
}

// keys that query i of a request sees
__device__ __forceinline__ int visible(int i, int lq, int lk, int prefix) {
  return max(0, min(lk, max(i + lk - lq + 1, prefix)));
}

template <typename T>
struct PromptKV {
  const T* k;
  const T* v;
  int64_t k_tok, v_tok;
  __device__ __forceinline__ void k8(int j, int d, float (&x)[8]) const {
    load8(k + (int64_t)j * k_tok + d, x);
  }
  __device__ __forceinline__ void v8(int j, int d, float (&x)[8]) const {
    load8(v + (int64_t)j * v_tok + d, x);
  }
};

constexpr int kRowWarps = 4;

// One warp per (token, head), for the head sizes without a tensor-core form and scales that are not
// positive: 3 TFLOP/s with heads of 96 (8 prompts of 900 tokens and 8 heads 2.8 ms, against 0.04 ms with
// heads of 128), 8 with heads of 256.
template <typename T>
__global__ void __launch_bounds__(32 * kRowWarps) prompt_rows_kernel(PromptArgs a) {
  const int64_t row = (int64_t)blockIdx.x * kRowWarps + (threadIdx.x >> 5);
  const int t = (int)(row / a.heads), h = (int)(row % a.heads);
  if (t >= a.total_q) return;
  T* out = reinterpret_cast<T*>(a.out) + t * a.o_tok + h * a.o_head;
  // the last request that starts at or before t
  int lo = 0, hi = a.batch;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a.cu_q[mid] <= t) lo = mid; else hi = mid;
  }
  int q0, lq, k0, lk;
  seq_span(a.cu_q, lo, a.total_q, q0, lq);
  seq_span(a.cu_k, lo, a.total_k, k0, lk);
  const int i = t - q0;
  // a token outside of every request (padding of the packed batch) gives zeros
  const int n = i >= 0 && i < lq ? visible(i, lq, lk, a.prefix ? a.prefix[lo] : 0) : 0;
  const int g = h / (a.heads / a.kv_heads);
  const PromptKV<T> kv{reinterpret_cast<const T*>(a.k) + k0 * a.k_tok + g * a.k_head,
                       reinterpret_cast<const T*>(a.v) + k0 * a.v_tok + g * a.v_head, a.k_tok,
                       a.v_tok};
  attend_row(reinterpret_cast<const T*>(a.q) + t * a.q_tok + h * a.q_head, a.head_dim, n, a.c, kv,
             out);
}

// ---- tensor-core form -----------------------------------------------------------------------------

constexpr int kKeys = 128;             // keys per tile
constexpr float kPromptGrow = 8.f;     // the reference is raised when the maximum has outgrown it by 2^8

// How far the reference lies below the maximum that it is taken from. Weights are held in the type of V:
// in fp16, those below 2^-14 lose bits and those below 2^-25 are zero, while the fp32 sum counts them.
// Lifted by 2^7 they reach 2^15 at most, with what the maximum may outgrow, and keep their bits down
// to 2^-21 of the largest. bf16 has fp32's range.
template <typename T>
constexpr float kLift = Tr<T>::kBf16 ? 0.f : 7.f;

template <int HD>
struct PromptCfg {
  static constexpr int NQ = HD == 256 ? 1 : 2;      // tiles of 128 query rows per CTA
  static constexpr int SPT = HD == 256 ? 2 : 1;     // ring slots per K or V tile
  static constexpr int SLOT = kKeys * HD * 2 / SPT;
  static constexpr int SLOTS = HD == 64 ? 8 : 5;
  static constexpr int Q_TILE = 128 * HD * 2;
  static constexpr int SMEM = NQ * Q_TILE + SLOTS * SLOT + 1024;
  static constexpr int THREADS = 128 + NQ * 128;   // producer, MMA issuers (and an idle warp); softmax
  static constexpr int VKEYS = kKeys / SPT;         // keys of a V slot
  // P·V starts on the first weights while the last are worked on: what is left then holds up the
  // next logits. A half is the most where V comes in halves (96 against 64 of 128: 1 %).
  static constexpr int FIRST = SPT == 1 ? 96 : 64;
  // tensor memory: two tiles of logits, each overlaid by its weights, then the sums
  static constexpr int O_COL = 256;
  // a partial: for each tile of rows the sums as [HD / 4][128 rows][4], then M and l of the rows
  static constexpr int PART_TILE = 128 * HD + 256;
  static constexpr int PARTIAL = NQ * PART_TILE;
};

// what a CTA leaves for the joining kernel about the tile that begins in it and goes on in others
struct PromptMeta {
  int request, tile, kv, count;
};

// A request, and the steps of its tiles: a step is a tile of query rows against a tile of keys.
struct PromptSeq {
  int q0, lq, k0, lk, prefix;
  __device__ __forceinline__ void load(const PromptArgs& a, int b) {
    seq_span(a.cu_q, b, a.total_q, q0, lq);
    seq_span(a.cu_k, b, a.total_k, k0, lk);
    prefix = a.prefix ? a.prefix[b] : 0;
  }
  __device__ __forceinline__ int sees(int i) const { return visible(i, lq, lk, prefix); }
  // steps of the tile of queries [t0, t0 + span): its last query sees the most keys. A tile that
  // sees none still takes one, which writes its zeros.
  __device__ __forceinline__ int steps(int t0, int span) const {
    return max(1, (sees(min(lq, t0 + span) - 1) + kKeys - 1) / kKeys);
  }
};

// Writing a tile's rows takes about as long as a step (6000 clocks to 2500 with 256 dimensions, 4000
// to 3900 below), so in the shares a (tile, kv head) counts for more than its steps.
__host__ __device__ constexpr int tile_cost(int head_dim) { return head_dim == 256 ? 2 : 1; }

// A CTA's steps as pieces, each a run of steps of one (tile, kv head). Every role walks the same.
struct PromptWalk {
  const PromptArgs& a;
  int span;
  int b, tile, kv, j0;  // next step: request, tile, kv head, tile of keys
  int64_t at, end;      // its number, and the share's end
  PromptSeq seq;
  int nt, n, take;      // tiles of the request; steps of the piece's tile, steps taken
  bool known;
  __device__ __forceinline__ bool next() {
    while (at < end) {
      if (!known) {
        for (;; ++b) {
          if (b >= a.batch) return false;
          seq.load(a, b);
          nt = (seq.lq + span - 1) / span;
          if (nt > 0) break;
        }
        known = true;
      }
      n = seq.steps(tile * span, span);
      take = (int)min(end - at, (int64_t)(n - j0));
      if (take > 0) return true;
      done();  // the share begins behind the tile's last step
    }
    return false;
  }
  __device__ __forceinline__ void done() {
    at += take;
    j0 += take;
    if (j0 < n) return;  // the share ends inside the tile
    at += n + tile_cost(a.head_dim) - j0;
    j0 = 0;
    if (++kv < a.kv_heads) return;
    kv = 0;
    if (++tile < nt) return;
    tile = 0;
    ++b;
    known = false;
  }
};


// A piece, as the producer hands it to the other warps.
struct __align__(16) PromptPiece {
  int take, key0, fewest, first;   // steps (0: no more); first key; keys all its rows see; first query
  int q0, lq, lk, prefix;          // its request
  int kv, slot, count, request;    // whole: slot < 0, else of the CTA's partials; see PromptMeta
  int k0, tile;
};

// largest of 128 logits, in four chains
__device__ __forceinline__ float max128(const float (&s)[128]) {
  float a = s[0], b = s[1], c = s[2], d = s[3];
#pragma unroll
  for (int j = 4; j < 124; j += 8) {
    a = max3(a, s[j], s[j + 1]);
    b = max3(b, s[j + 2], s[j + 3]);
    c = max3(c, s[j + 4], s[j + 5]);
    d = max3(d, s[j + 6], s[j + 7]);
  }
  return fmaxf(max3(a, s[124], s[125]), max3(max3(b, s[126], s[127]), c, d));
}

// whether all threads of NQ softmax warpgroups say so: they leave their loops together
template <int NQ>
__device__ __forceinline__ bool softmax_all(bool v, int id = 1) {
  uint32_t r;
  asm volatile(
      "{\n .reg .pred p, q;\n setp.ne.u32 p, %1, 0;\n barrier.cta.red.and.pred q, %2, %3, p;\n"
      " selp.u32 %0, 1, 0, q;\n}\n"
      : "=r"(r)
      : "r"((uint32_t)v), "r"(id), "n"(NQ * 128)
      : "memory");
  return r != 0;
}

template <typename T, int HD>
__global__ void __launch_bounds__(PromptCfg<HD>::THREADS, 1)
    prompt_tc_kernel(const __grid_constant__ CUtensorMap tmQ,
                     const __grid_constant__ CUtensorMap tmK,
                     const __grid_constant__ CUtensorMap tmV, PromptArgs a, int tok) {
  using C = PromptCfg<HD>;
  constexpr int NQ = C::NQ, SPT = C::SPT, SLOTS = C::SLOTS, WARPS = C::THREADS / 32;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  uint8_t* sQ = base + SLOTS * C::SLOT;
  __shared__ __align__(8) uint64_t full[SLOTS], empty[SLOTS], q_full, q_empty, s_full[2],
      p_full[2][2], pv_done[2], turn[2], drain;
  __shared__ uint32_t s_tmem;
  __shared__ int s_tiles[C::THREADS], s_scan[WARPS], s_at[4], s_stop;
  __shared__ uint32_t s_odd[kKeys / 32];  // keys of a tile whose values are no numbers
  __shared__ int64_t s_steps[WARPS], s_begin, s_total;
  __shared__ PromptPiece s_piece[2];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const Waits waits{a.err, &s_stop};
  const int group = a.heads / a.kv_heads, span = NQ * tok;
  const int ctas = gridDim.x, cta = blockIdx.x;
  pdl_trigger();  // every CTA of this grid is resident at once: the joining blocks may queue up
  for (int b = tid; b < a.batch; b += C::THREADS) {  // read below, one after the other
    pf_l1(a.cu_k + b);
    if (a.prefix) pf_l1(a.prefix + b);
  }

  if (tid == 0) {
    for (int i = 0; i < SLOTS; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], NQ);
    }
    mbar_init(&q_full, 1);
    mbar_init(&q_empty, 2 * NQ);  // its QKs are done, and the softmax warps have begun it
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i][0], 4);
      mbar_init(&p_full[i][1], 4);
      mbar_init(&pv_done[i], 1);
      mbar_init(&turn[i], 4);
    }
    mbar_init(&drain, NQ);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    tma_prefetch_desc(&tmQ);
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
    s_stop = 0;
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(&s_tmem)),
                 "r"(512u));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }

  // ---- this CTA's share of the steps ----
  {
    // tiles before each thread's requests
    const int per = (a.batch + C::THREADS - 1) / C::THREADS;
    const int b0 = min(a.batch, tid * per), b1 = min(a.batch, b0 + per);
    auto tiles_of = [&](int b) {
      int t0, n;
      seq_span(a.cu_q, b, a.total_q, t0, n);
      return (n + span - 1) / span;
    };
    int mine = 0;
    for (int b = b0; b < b1; ++b) mine += tiles_of(b);
    int inc = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int up = __shfl_up_sync(~0u, inc, d);
      if (lane >= d) inc += up;
    }
    if (lane == 31) s_scan[warp] = inc;
    __syncthreads();
    int before = inc - mine, tiles = 0;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      if (w < warp) before += s_scan[w];
      tiles += s_scan[w];
    }
    s_tiles[tid] = before;
    __syncthreads();
    // steps before each thread's tiles
    const int each = (tiles + C::THREADS - 1) / C::THREADS;
    const int g0 = min(tiles, tid * each), g1 = min(tiles, g0 + each);
    PromptSeq seq;
    int b = 0, t = 0, nt = 0;        // request and tile of g0
    if (g0 < g1) {
      int lo = 0, hi = C::THREADS;   // the last thread whose requests start at or before tile g0
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (s_tiles[mid] <= g0) lo = mid; else hi = mid;
      }
      t = g0 - s_tiles[lo];
      for (b = lo * per; t >= (nt = tiles_of(b)) && b + 1 < a.batch; ++b) t -= nt;
      seq.load(a, b);
    }
    const int bg = b, tg = t;
    int64_t sum = 0;
    auto steps_of_next = [&]() {     // what tile (b, t) counts for, and on to the one behind it
      while (t >= nt && b + 1 < a.batch) {
        t = 0;
        nt = tiles_of(++b);
        if (nt > 0) seq.load(a, b);
      }
      return seq.steps(t++ * span, span) + tile_cost(HD);
    };
    for (int g = g0; g < g1; ++g) sum += steps_of_next();
    sum *= a.kv_heads;
    int64_t incs = sum;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int64_t up = __shfl_up_sync(~0u, incs, d);
      if (lane >= d) incs += up;
    }
    if (lane == 31) s_steps[warp] = incs;
    __syncthreads();
    int64_t first = incs - sum, total = 0;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      if (w < warp) first += s_steps[w];
      total += s_steps[w];
    }
    const int64_t x0 = Shares<int64_t>(total, ctas).begin(cta, total);
    if (tid == 0) {
      s_begin = x0;
      s_total = total;
    }
    if (x0 >= first && x0 < first + sum) {
      int64_t x = x0 - first;
      b = bg;
      t = tg;
      if (g0 < g1) {
        nt = tiles_of(b);
        seq.load(a, b);
      }
      for (;;) {
        const int n = steps_of_next();
        if (x < (int64_t)n * a.kv_heads) {
          s_at[0] = b;
          s_at[1] = t - 1;
          s_at[2] = (int)x / n;
          s_at[3] = (int)x % n;
          break;
        }
        x -= (int64_t)n * a.kv_heads;
      }
    }
    // tokens of no request: zeros
    const int head = min(max(a.cu_q[0], 0), a.total_q);
    const int tail = min(max(a.cu_q[a.batch], head), a.total_q);
    const int64_t none = (int64_t)(head + a.total_q - tail) * a.heads * (HD / 8);
    for (int64_t i = (int64_t)cta * C::THREADS + tid; i < none; i += (int64_t)ctas * C::THREADS) {
      const int64_t row = i / (HD / 8);
      int tk = (int)(row / a.heads);
      tk = tk < head ? tk : tail + tk - head;
      *reinterpret_cast<uint4*>(reinterpret_cast<T*>(a.out) + tk * a.o_tok +
                                (row % a.heads) * a.o_head + (i % (HD / 8)) * 8) =
          make_uint4(0, 0, 0, 0);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_tmem;
  const int64_t total = s_total;
  const Shares<int64_t> shares(total, ctas);
  // Position of the K or V of a piece's step j (of n) in the order of the loads, in units of SPT
  // slots: the order in which the MMAs take them.
  auto k_unit = [](int j) { return NQ == 2 ? 2 * j : (j == 0 ? 0 : 2 * j - 1); };
  auto v_unit = [](int j, int n) { return NQ == 2 ? 2 * j + 1 : min(2 * j + 2, n + j); };

  // A row whose sum meets an infinity or a NaN may owe it to a value that it does not see (weight
  // zero times infinity): then the CTA does its share once more, with such values taken out of the
  // V tiles that some rows of a piece see in part, and added to the sums of the rows that see them.
  // A row of 128 logits takes more registers than 1/12 of an SM's: where there are twelve warps, the
  // first warpgroup gives some of its own. (80 + 2·208)·128 of the 168·384 that the block was
  // launched with.
  if (warp < 4) {
    if constexpr (NQ == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 80;");
    int done = 0, pieces = 0;  // steps and pieces so far
    bool ok = true;
    for (int pass = 0; pass < 2; ++pass) {
      if (warp == 0) {
        if (lane == 0) {
          // ---- producer ----
          PromptWalk w{a, span, s_at[0], s_at[1], s_at[2], s_at[3], s_begin,
                       shares.begin(cta + 1, total), PromptSeq{}, 0, 0, 0, false};
          int load = done * 2 * SPT;
          auto slot_of = [&]() -> uint8_t* {
            const int s = load % SLOTS;
            if (load >= SLOTS)
              ok = ok &&
                   bar_wait(&empty[s], (load / SLOTS - 1) & 1, waits, tc::ERR_TIMEOUT_PRODUCER);
            if (!ok) return nullptr;
            mbar_expect_tx(&full[s], C::SLOT);
            ++load;
            return base + s * C::SLOT;
          };
          auto load_k = [&](int j) {
#pragma unroll 1
            for (int h = 0; h < SPT; ++h) {
              uint8_t* dst = slot_of();
              if (!dst) return;
              uint64_t* bar = &full[(load - 1) % SLOTS];
#pragma unroll
              for (int kb = 0; kb < HD / 64 / SPT; ++kb)
                tma_load_3d(dst + kb * 16384, &tmK, bar, (h * (HD / 64 / SPT) + kb) * 64, w.kv,
                            w.seq.k0 + (w.j0 + j) * kKeys);
            }
          };
          auto load_v = [&](int j) {
#pragma unroll 1
            for (int h = 0; h < SPT; ++h) {
              uint8_t* dst = slot_of();
              if (!dst) return;
              uint64_t* bar = &full[(load - 1) % SLOTS];
#pragma unroll
              for (int kb = 0; kb < HD / 64; ++kb)
                tma_load_3d(dst + kb * (C::VKEYS * 128), &tmV, bar, kb * 64, w.kv,
                            w.seq.k0 + (w.j0 + j) * kKeys + h * C::VKEYS);
            }
          };
          for (;;) {
            const bool more = ok && w.next();
            if (more) load_k(0);
            // the piece before has been begun, and its QKs have read Q
            if (ok && pieces > 0)
              ok = bar_wait(&q_empty, (pieces - 1) & 1, waits, tc::ERR_TIMEOUT_PRODUCER);
            if (!ok) break;
            PromptPiece& pc = s_piece[pieces & 1];
            if (!more) {
              pc.take = 0;
              mbar_arrive(&q_full);
              ++pieces;
              break;
            }
            const bool whole = w.take == w.n;
            pc = PromptPiece{w.take, w.j0 * kKeys, w.seq.sees(w.tile * span), w.tile * span,
                             w.seq.q0, w.seq.lq, w.seq.lk, w.seq.prefix,
                             w.kv, whole ? -1 : w.j0 > 0 ? 0 : 1,
                             !whole && w.j0 == 0 ? shares.owner(w.at + w.n - 1) - cta + 1 : 0, w.b,
                             w.seq.k0, w.tile};
            // bytes of whole boxes: what lies out of bounds arrives as zeros
            mbar_expect_tx(&q_full, (uint32_t)(NQ * HD / 64 * tok * group * 128));
#pragma unroll
            for (int q = 0; q < NQ; ++q)
#pragma unroll
              for (int kb = 0; kb < HD / 64; ++kb)
                tma_load_3d(sQ + q * C::Q_TILE + kb * 16384, &tmQ, &q_full, kb * 64, w.kv * group,
                            w.seq.q0 + w.tile * span + q * tok);
            ++pieces;
#pragma unroll 1
            for (int j = 0; j < w.take && ok; ++j) {
              if (NQ == 2 ? j > 0 : j + 1 < w.take) load_k(NQ == 2 ? j : j + 1);
              if (ok) load_v(j);
            }
            done += w.take;
            w.done();
          }
          // no copy into this CTA's shared memory may be in flight when it exits
          if (ok)
            bar_wait(&q_full, (pieces - 1) & 1, waits, tc::ERR_TIMEOUT_PRODUCER, false);
          for (int l = max(0, load - SLOTS); l < load; ++l)
            bar_wait(&full[l % SLOTS], (l / SLOTS) & 1, waits, tc::ERR_TIMEOUT_PRODUCER, false);
        }
        __syncwarp();
      } else if (warp <= NQ) {
        // ---- MMA issuers: with two tiles of rows a warp for each, so that neither waits for the
        // other's weights. A tile's logits and weights share their columns, and MMAs of one thread
        // run in order: P·V j, then the logits that overwrite P.
        constexpr uint32_t id_s = tc::idesc_f16<T>(128, kKeys);
        constexpr uint32_t id_o = tc::idesc_f16<T>(128, HD) | (1u << 16);  // V is MN-major
        constexpr int kAhead = NQ == 2 ? 1 : 2;  // steps whose logits come before the first weights
        const int q = warp - 1;
        int take = 0;
        const uint32_t ring = __shfl_sync(~0u, smem_u32(base), 0), tm = __shfl_sync(~0u, tmem, 0);
        const uint32_t qs = ring + SLOTS * C::SLOT + q * C::Q_TILE, to = tm + C::O_COL + q * HD;
        auto full_of = [&](int load) {
          return bar_wait(&full[load % SLOTS], (load / SLOTS) & 1, waits, tc::ERR_TIMEOUT_MMA);
        };
        auto job_of = [&](int j) { return NQ == 2 ? 2 * (done + j) + q : done + j; };
        auto qk = [&](int j) {
          const int buf = job_of(j) & 1, load = (2 * done + k_unit(j)) * SPT;
#pragma unroll
          for (int h = 0; h < SPT; ++h) {
            if (!ok || ((NQ == 1 || j == 0) && !(ok = full_of(load + h)))) return;
            tc_fence_after();
            const int slot = (load + h) % SLOTS;
            const uint64_t da = tc::desc_sw128(qs + h * (HD / 64 / SPT) * 16384);
            const uint64_t db = tc::desc_sw128(ring + slot * C::SLOT);
            if (elect_one()) {
#pragma unroll
              for (int kb = 0; kb < HD / 64 / SPT; ++kb)
#pragma unroll
                for (int k = 0; k < 4; ++k)
                  tc::umma_f16(tm + buf * kKeys, da + 1024 * kb + 2 * k, db + 1024 * kb + 2 * k, id_s,
                               (h | kb | k) != 0);
              if (h == SPT - 1) umma_commit(&s_full[buf]);
              umma_commit(&empty[slot]);
              if (h == SPT - 1 && j + 1 == take) umma_commit(&q_empty);
            }
            __syncwarp();
          }
        };
        auto pv = [&](int j) {
          const int job = job_of(j), buf = job & 1, load = (2 * done + v_unit(j, take)) * SPT;
          // The keys of the logits behind this product, and V, are there before the weights are, which
          // come in two parts: waiting for them here takes nothing from between the products.
          if (NQ == 2 && j + 1 < take && !(ok = full_of(2 * done + k_unit(j + 1)))) return;
#pragma unroll
          for (int h = 0; h < SPT; ++h)
            if (!ok || !(ok = full_of(load + h))) return;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            if (!(ok = bar_wait(&p_full[buf][h], (job >> 1) & 1, waits, tc::ERR_TIMEOUT_MMA)))
              return;
            tc_fence_after();
            const int slot = (load + h * (SPT - 1)) % SLOTS;
            const uint64_t dv = sdesc<128>(ring + slot * C::SLOT, 1024, C::VKEYS * 128) +
                                (SPT == 1 ? C::FIRST * 8 * h : 0);
            const uint32_t tp = tm + buf * kKeys + C::FIRST / 2 * h;
            const uint32_t more = (j | h) != 0;
            if (elect_one()) {
#pragma unroll
              for (int k = 0; k < (h == 0 ? C::FIRST : kKeys - C::FIRST) / 16; ++k)
                // 16 keys, 2048 bytes of V rows, each
                umma_f16_ta(to, tp + 8 * k, dv + 128 * k, id_o, k == 0 ? more : 1u);
              if (h == 1) umma_commit(&pv_done[buf]);
              if (h >= 2 - SPT) umma_commit(&empty[slot]);
            }
            __syncwarp();
          }
        };
        for (;;) {
          ok = ok && bar_wait(&q_full, pieces & 1, waits, tc::ERR_TIMEOUT_MMA);
          if (!ok) break;
          take = s_piece[pieces & 1].take;
          ++pieces;
          if (take == 0) {
            if (lane == 0) mbar_arrive(&q_empty);
            break;
          }
#pragma unroll
          for (int j = 0; j < kAhead; ++j)
            if (j < take) qk(j);
          for (int j = 0; j < take && ok; ++j) {
            pv(j);
            if (j + kAhead < take) qk(j + kAhead);
          }
          done += take;
        }
        // every issued MMA completes before TMEM is released
        if (elect_one()) umma_commit(&drain);
        __syncwarp();
        bar_wait(&drain, pass, waits, tc::ERR_TIMEOUT_MMA, false);
      }
      if (!block_any<C::THREADS>(false)) break;
    }
  } else {
    if constexpr (NQ == 2) asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    // ---- softmax and output: one thread per query row ----
    const int wg = (warp - 4) >> 2, q4 = warp & 3, r = q4 * 32 + lane;
    const uint32_t tl = tmem + ((uint32_t)(q4 * 32) << 16);
    const uint32_t tO = tl + C::O_COL + wg * HD;
    int done = 0, pieces = 0;
    bool ok = true;
    if (NQ == 2 && wg == 1 && lane == 0) mbar_arrive(&turn[0]);  // warpgroup 0's is the first
    for (int pass = 0; pass < 2; ++pass) {
      PromptMeta meta{0, 0, 0, 0};
      bool again = false;
      for (;;) {
        ok = ok && bar_wait(&q_full, pieces & 1, waits, tc::ERR_TIMEOUT_EPI);
        // in the second pass the warpgroups meet below: there one's failure is the other's
        ok = pass == 1 ? softmax_all<NQ>(ok) : softmax_all<1>(ok, 2 + wg);
        if (!ok) break;
        const PromptPiece& pc = s_piece[pieces & 1];
        ++pieces;
        const int take = pc.take;
        if ((tid & 127) == 0) mbar_arrive(&q_empty);
        if (take == 0) break;
        const int tq = pc.first + wg * tok;            // the first query of these rows
        const int i = tq + r / group;                  // the row's
        const bool row = r < tok * group && i < pc.lq;
        const int mine = row ? visible(i, pc.lq, pc.lk, pc.prefix) : 0;
        // keys below these need no mask in this warpgroup's rows
        const int clear = tq < pc.lq ? visible(tq, pc.lq, pc.lk, pc.prefix) : 0;
        float m = -INFINITY, l = 0.f;
        // one step; the second pass has a copy of its own, to keep the first's code short
        auto step = [&](int t, auto second) {
          constexpr bool careful = decltype(second)::value;
          const int job = NQ == 2 ? 2 * (done + t) + wg : done + t, buf = job & 1;
          const int key0 = pc.key0 + t * kKeys;
          if (ok) ok = bar_wait(&s_full[buf], (job >> 1) & 1, waits, tc::ERR_TIMEOUT_EPI);
          ok = __all_sync(~0u, ok);
          if (ok) {
            tc_fence_after();
            float s[128];
            const float c = a.c;
#pragma unroll
            for (int q = 0; q < 4; ++q)
              tmem_ld32_async(tl + buf * kKeys + 32 * q, reinterpret_cast<uint32_t*>(s) + 32 * q);
            tmem_wait_ld();
            if (key0 + kKeys > clear) {
              const int lim = mine - key0;
#pragma unroll
              for (int u = 0; u < 128; ++u) s[u] = u < lim ? s[u] : -INFINITY;
            }
            const float top = max128(s) * c - kLift<T>;
            if (t == 0) {
              m = top;
            } else if (__any_sync(~0u, top > m + kPromptGrow)) {
              // the sums so far are complete once the P·V before has finished
              const int prev = NQ == 2 ? job - 2 : job - 1;
              ok = bar_wait(&pv_done[prev & 1], (prev >> 1) & 1, waits, tc::ERR_TIMEOUT_EPI);
              ok = __all_sync(~0u, ok);
              if (ok) {
                float al = 1.f;
                if (top > m + kPromptGrow) {
                  al = m == -INFINITY ? 0.f : exp2_fast(m - top);
                  m = top;
                  l *= al;
                }
                tc_fence_after();
#pragma unroll 1
                for (int d = 0; d < HD; d += 32) {
                  uint32_t o[32];
                  tmem_ld32(tO + d, o);
#pragma unroll
                  for (int u = 0; u < 32; ++u)
                    o[u] = __float_as_uint(__uint_as_float(o[u]) * al);
                  tmem_st32(tO + d, o);
                }
              }
            }
            // The exponentials of the two warpgroups take turns: at the same time they would hold
            // each other up, and then both leave the tensor cores without work.
            if constexpr (NQ == 2)
              ok = bar_wait(&turn[wg], (done + t) & 1, waits, tc::ERR_TIMEOUT_EPI);
            const float ref = m == -INFINITY ? 0.f : m;
            const uint64_t c2 = pack2(c, c), r2 = pack2(-ref, -ref);
            uint64_t sum0 = 0, sum1 = 0;  // two zeros each
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              uint32_t pw[16];
#pragma unroll
              for (int u = 0; u < 16; ++u) {
                const float2 f = unpack2(fma2(pack2(s[32 * q + 2 * u], s[32 * q + 2 * u + 1]), c2, r2));
                const float e0 = exp2_fast(f.x), e1 = exp2_fast(f.y);
                if (u & 1) sum1 = add2(sum1, pack2(e0, e1));
                else sum0 = add2(sum0, pack2(e0, e1));
                // weights in the type of V, as a 16-bit product asks; their sum is of the fp32 ones
                pw[u] = Tr<T>::pack(e0, e1);
              }
              tmem_st16(tl + buf * kKeys + 16 * q, pw);
              if (q == C::FIRST / 32 - 1) {  // the first weights may go
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (!careful && lane == 0) mbar_arrive(&p_full[buf][0]);
              }
            }
            const float2 sums = unpack2(add2(sum0, sum1));
            l += sums.x + sums.y;
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (!careful && lane == 0) mbar_arrive(&p_full[buf][1]);  // the other tile can wait, P·V not
            if (NQ == 2 && lane == 0) mbar_arrive(&turn[wg ^ 1]);
          }
          const bool in_part = careful && key0 + kKeys > pc.fewest;  // the same for all rows
          if (in_part) {
            // V rows of this tile, by all softmax warps: values that are no numbers become zero
            named_sync<1, NQ * 128>();  // s_odd of the step before has been read
            if (tid - 128 < kKeys / 32) s_odd[tid - 128] = 0;
            named_sync<1, NQ * 128>();
            const int load = (2 * done + v_unit(t, take)) * SPT;
#pragma unroll 1
            for (int h = 0; h < SPT; ++h) {
              const int sl = (load + h) % SLOTS;
              if (ok) ok = bar_wait(&full[sl], ((load + h) / SLOTS) & 1, waits, tc::ERR_TIMEOUT_EPI);
              ok = __all_sync(~0u, ok);
              if (!ok) break;
#pragma unroll 1
              for (int v = tid - 128; v < C::SLOT / 16; v += NQ * 128) {
                const int key = h * C::VKEYS + (v / 8) % C::VKEYS;  // within the tile
                uint4* at = reinterpret_cast<uint4*>(base + sl * C::SLOT) + v;
                uint4 x4 = *at;
                T* e = reinterpret_cast<T*>(&x4);
                bool hit = false;
#pragma unroll
                for (int u = 0; u < 8; ++u)
                  if (!isfinite(Tr<T>::f(e[u]))) {
                    e[u] = Tr<T>::t(0.f);
                    hit = true;
                  }
                if (hit) {
                  *at = x4;
                  if (key0 + key < pc.lk) atomicOr(&s_odd[key / 32], 1u << (key % 32));
                }
              }
            }
            fence_async_smem();
            named_sync<1, NQ * 128>();
          }
          __syncwarp();
          if (careful && ok && lane == 0) {  // only now is V what it should be
            mbar_arrive(&p_full[buf][0]);
            mbar_arrive(&p_full[buf][1]);
          }
          if (in_part && (s_odd[0] | s_odd[1] | s_odd[2] | s_odd[3])) {
            // what was taken out reaches the rows that see it as it is: any weight of an infinity is one
            if (ok) ok = bar_wait(&pv_done[buf], (job >> 1) & 1, waits, tc::ERR_TIMEOUT_EPI);
            ok = __all_sync(~0u, ok);
            if (ok) {
              tc_fence_after();
              const T* v0 = reinterpret_cast<const T*>(a.v) + (int64_t)(pc.k0 + key0) * a.v_tok +
                            pc.kv * a.v_head;
#pragma unroll 1
              for (int d = 0; d < HD; d += 32) {
                uint32_t o[32];
                tmem_ld32(tO + d, o);
#pragma unroll 1
                for (int j = 0; j < kKeys; ++j) {
                  if (!(s_odd[j / 32] >> (j % 32) & 1)) continue;
                  const bool sees = key0 + j < mine;
#pragma unroll
                  for (int c = 0; c < 4; ++c) {
                    float x[8];
                    load8(v0 + j * a.v_tok + d + c * 8, x);
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                      if (sees && !isfinite(x[e]))
                        o[c * 8 + e] = __float_as_uint(__uint_as_float(o[c * 8 + e]) + x[e]);
                  }
                }
                __syncwarp();
                tmem_st32(tO + d, o);
              }
              tmem_wait_st();
              tc_fence_before();
            }
          }
        };
        if (pass == 0) {
          for (int t = 0; t < take; ++t) step(t, std::false_type{});
        } else {
          for (int t = 0; t < take; ++t) step(t, std::true_type{});
        }
        const int last = NQ == 2 ? 2 * (done + take - 1) + wg : done + take - 1;
        done += take;
        const bool whole = pc.slot < 0;
        const int64_t row_at = (int64_t)(pc.q0 + i) * a.o_tok +
                               (int64_t)(pc.kv * group + r % group) * a.o_head;
        if (ok) ok = bar_wait(&pv_done[last & 1], (last >> 1) & 1, waits, tc::ERR_TIMEOUT_EPI);
        ok = __all_sync(~0u, ok);
        tc_fence_after();
        // o = O / l, or O as it is for the joining kernel. A row that sees no key is zero, and one
        // whose products were not waited for to the end NaN.
        const float inv = !ok ? NAN : whole ? 1.f / l : 1.f;
        const uint64_t inv2 = pack2(inv, inv);
        uint64_t nan2[2] = {0, 0};  // sums of 0·o: NaN once an element is no number
        const uint32_t keep = mine > 0 ? ~0u : 0u;
        if (whole) {
          // A lane has a row, and storing straight from it every instruction would touch 32 lines of
          // global memory. Four lanes exchange chunks of 16 bytes first: lane 4a + c then has chunk c
          // of the rows 4a, 4a + 1, 4a + 2, 4a + 3. The loop stays rolled: code that runs once a
          // piece comes from far away.
          T* to[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int64_t at = __shfl_sync(~0u, row ? row_at : (int64_t)-1, (lane & ~3) + k);
            to[k] = at < 0 ? nullptr : reinterpret_cast<T*>(a.out) + at + (lane & 3) * 8;
          }
          uint32_t next[32];
          tmem_ld32_async(tO, next);
#pragma unroll 1
          for (int d = 0; d < HD; d += 32) {
            uint32_t pw[4][4];  // the row's four chunks
            tmem_wait_ld();
#pragma unroll
            for (int u = 0; u < 16; ++u) {
              const uint64_t y = mul2(pack2(__uint_as_float(next[2 * u]),
                                            __uint_as_float(next[2 * u + 1])), inv2);
              nan2[u & 1] = fma2(y, 0, nan2[u & 1]);
              const float2 f = unpack2(y);
              pw[u / 4][u % 4] = Tr<T>::pack(f.x, f.y) & keep;
            }
            if (d + 32 < HD) tmem_ld32_async(tO + d + 32, next);
            // transpose of 4 × 4 chunks in two exchanges: with the lane one away, then two away
#pragma unroll
            for (int st = 1; st <= 2; st *= 2) {
              const bool up = lane & st;
#pragma unroll
              for (int c = 0; c < 4; ++c) {
                if (c & st) continue;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  const uint32_t give = up ? pw[c][e] : pw[c + st][e];
                  const uint32_t got = __shfl_xor_sync(~0u, give, st);
                  if (up) pw[c][e] = got;
                  else pw[c + st][e] = got;
                }
              }
            }
#pragma unroll
            for (int k = 0; k < 4; ++k)
              if (to[k])
                *reinterpret_cast<uint4*>(to[k] + d) =
                    make_uint4(pw[k][0], pw[k][1], pw[k][2], pw[k][3]);
          }
        } else {
          float* part = a.ws + (size_t)ctas * 4 + ((size_t)cta * 2 + pc.slot) * C::PARTIAL +
                        wg * C::PART_TILE;
#pragma unroll 1
          for (int d = 0; d < HD; d += 32) {
            uint32_t o[32];
            tmem_ld32(tO + d, o);
#pragma unroll
            for (int u = 0; u < 32; u += 4) {
              const uint64_t y0 = mul2(pack2(__uint_as_float(o[u]), __uint_as_float(o[u + 1])), inv2);
              const uint64_t y1 =
                  mul2(pack2(__uint_as_float(o[u + 2]), __uint_as_float(o[u + 3])), inv2);
              nan2[0] = fma2(y0, 0, nan2[0]);
              nan2[1] = fma2(y1, 0, nan2[1]);
              const float2 f0 = unpack2(y0), f1 = unpack2(y1);
              *reinterpret_cast<float4*>(part + ((size_t)(d + u) / 4 * 128 + r) * 4) =
                  make_float4(f0.x, f0.y, f1.x, f1.y);
            }
          }
        }
        const float2 nan = unpack2(add2(nan2[0], nan2[1]));
        const bool odd = row && mine > 0 && ok && !(nan.x + nan.y == 0.f);
        again |= odd;
        tc_fence_before();
        if (!whole) {
          float* ml = a.ws + (size_t)ctas * 4 + ((size_t)cta * 2 + pc.slot) * C::PARTIAL +
                      wg * C::PART_TILE + 128 * HD;
          ml[r] = m;
          ml[128 + r] = l;
          if (pc.count > 0) meta = PromptMeta{pc.request, pc.tile, pc.kv, pc.count};
        }
      }
      if (tid == 128) reinterpret_cast<PromptMeta*>(a.ws)[cta] = meta;
      if (!block_any<C::THREADS>(again)) break;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u));
  }
}

// Joins the partials of the tile that begins in CTA blockIdx.x and ends in another, in the order of
// the CTAs: one block per (CTA, tile of rows, 32 dimensions), one thread per row.
template <typename T, int HD>
__global__ void __launch_bounds__(128) prompt_join_kernel(PromptArgs a, int tok, int ctas) {
  using C = PromptCfg<HD>;
  pdl_wait();
  const int cta = blockIdx.x, wg = blockIdx.y / (HD / 32), d0 = blockIdx.y % (HD / 32) * 32;
  const PromptMeta meta = reinterpret_cast<const PromptMeta*>(a.ws)[cta];
  if (meta.count == 0) return;
  const int r = threadIdx.x, group = a.heads / a.kv_heads;
  PromptSeq seq;
  seq.load(a, meta.request);
  const int tq = meta.tile * C::NQ * tok + wg * tok, i = tq + r / group;
  const bool row = r < tok * group && i < seq.lq;
  const float* first = a.ws + (size_t)ctas * 4 + ((size_t)cta * 2 + 1) * C::PARTIAL +
                       wg * C::PART_TILE;
  float M = -INFINITY, l = 0.f, o[32];
#pragma unroll
  for (int u = 0; u < 32; ++u) o[u] = 0.f;
  for (int p = 0; p < meta.count; ++p) {
    // partial p: slot 1 of the first CTA, slot 0 of those behind it
    const float* part = first + (p == 0 ? 0 : ((size_t)p * 2 - 1) * C::PARTIAL);
    const float pm = part[128 * HD + r], pl = part[128 * HD + 128 + r];
    float4 v[8];
#pragma unroll
    for (int u = 0; u < 8; ++u)
      v[u] = *reinterpret_cast<const float4*>(part + ((size_t)(d0 / 4 + u) * 128 + r) * 4);
    const float top = fmaxf(M, pm), ref = top == -INFINITY ? 0.f : top;
    const float old = exp2f(M - ref), f = exp2f(pm - ref);
    M = top;
    l = l * old + f * pl;
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      o[4 * u] = o[4 * u] * old + f * v[u].x;
      o[4 * u + 1] = o[4 * u + 1] * old + f * v[u].y;
      o[4 * u + 2] = o[4 * u + 2] * old + f * v[u].z;
      o[4 * u + 3] = o[4 * u + 3] * old + f * v[u].w;
    }
  }
  const int64_t h = meta.kv * group + r % group;
  if (row) {
    const float inv = 1.f / l;
    const uint32_t keep = seq.sees(i) > 0 ? ~0u : 0u;  // a row that sees no key is zero
    T* out = reinterpret_cast<T*>(a.out) + (int64_t)(seq.q0 + i) * a.o_tok + h * a.o_head + d0;
#pragma unroll
    for (int u = 0; u < 32; u += 8) {
      uint4 pk;
      uint32_t* pw = reinterpret_cast<uint32_t*>(&pk);
#pragma unroll
      for (int e = 0; e < 4; ++e) pw[e] = Tr<T>::pack(o[u + 2 * e] * inv, o[u + 2 * e + 1] * inv) & keep;
      *reinterpret_cast<uint4*>(out + u) = pk;
    }
  }
}

}  // namespace paged
}  // namespace pi0
