// Attention over packed prompts: grouped heads, causal with a bidirectional prefix per request.
//
// Query i of a request with Lq new tokens and Lk keys sees the keys j < n(i),
// n(i) = min(Lk, max(i + Lk − Lq + 1, prefix)): always a leading part of the request's keys.
#pragma once

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

// One warp per (token, head), for the head sizes without a tensor-core form.
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
constexpr float kPromptGrow = 8.f;     // the reference maximum is raised when it would grow by 2^8

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
  // tensor memory: two tiles of logits, each overlaid by its weights, then the sums
  static constexpr int O_COL = 256;
};

struct PromptTile {
  int q0, lq, k0, lk, prefix, t0;
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
  return fmaxf(max3(a, s[124], s[125]), fmaxf(max3(b, s[126], s[127]), fmaxf(c, d)));
}

template <typename T, int HD>
__global__ void __launch_bounds__(PromptCfg<HD>::THREADS, 1)
    prompt_tc_kernel(const __grid_constant__ CUtensorMap tmQ,
                     const __grid_constant__ CUtensorMap tmK,
                     const __grid_constant__ CUtensorMap tmV, PromptArgs a, int tok) {
  using C = PromptCfg<HD>;
  constexpr int NQ = C::NQ, SPT = C::SPT, SLOTS = C::SLOTS;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  uint8_t* sQ = base + SLOTS * C::SLOT;
  __shared__ __align__(8) uint64_t full[SLOTS], empty[SLOTS], q_full, s_full[2],
      p_full[2][2], pv_done[2], drain;
  __shared__ uint32_t s_tmem;
  __shared__ int s_scan[C::THREADS / 32], s_req, s_tile, s_bad;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int kv = blockIdx.x % a.kv_heads, index = blockIdx.x / a.kv_heads;
  const int group = a.heads / a.kv_heads;

  if (tid == 0) {
    for (int i = 0; i < SLOTS; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], NQ);
    }
    mbar_init(&q_full, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i][0], 4);
      mbar_init(&p_full[i][1], 4);
      mbar_init(&pv_done[i], 1);
    }
    mbar_init(&drain, NQ);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    tma_prefetch_desc(&tmQ);
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
    s_req = -1;
    s_bad = 0x7fffffff;
  }
  // ---- which tile: the tiles of the requests are numbered in order; `index` lies in one of them
  const int span = NQ * tok;
  {
    const int per = (a.batch + C::THREADS - 1) / C::THREADS;
    const int b0 = min(a.batch, tid * per), b1 = min(a.batch, b0 + per);
    int mine = 0, t0, n;
    for (int b = b0; b < b1; ++b) {
      seq_span(a.cu_q, b, a.total_q, t0, n);
      mine += (n + span - 1) / span;
    }
    int inc = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int up = __shfl_up_sync(~0u, inc, d);
      if (lane >= d) inc += up;
    }
    if (lane == 31) s_scan[warp] = inc;
    __syncthreads();
    int before = inc - mine;
#pragma unroll
    for (int w = 0; w < C::THREADS / 32; ++w)
      if (w < warp) before += s_scan[w];
    if (index >= before && index < before + mine) {
      int x = index - before;
      for (int b = b0;; ++b) {
        seq_span(a.cu_q, b, a.total_q, t0, n);
        const int nt = (n + span - 1) / span;
        if (x < nt) {
          s_req = b;
          s_tile = nt - 1 - x;  // the last tile of a request sees the most keys: first
          break;
        }
        x -= nt;
      }
    }
    // tokens of no request: zeros
    if (index == 0 && kv == 0) {
      const int first = min(max(a.cu_q[0], 0), a.total_q);
      const int behind = min(max(a.cu_q[a.batch], first), a.total_q);
      const int64_t none = (int64_t)(first + a.total_q - behind) * a.heads * (HD / 8);
      for (int64_t i = tid; i < none; i += C::THREADS) {
        const int64_t row = i / (HD / 8);
        int t = (int)(row / a.heads);
        t = t < first ? t : behind + t - first;
        *reinterpret_cast<uint4*>(reinterpret_cast<T*>(a.out) + t * a.o_tok +
                                  (row % a.heads) * a.o_head + (i % (HD / 8)) * 8) =
            make_uint4(0, 0, 0, 0);
      }
    }
  }
  __syncthreads();
  if (s_req < 0) return;  // the grid is an upper bound of the tiles
  PromptTile p;
  seq_span(a.cu_q, s_req, a.total_q, p.q0, p.lq);
  seq_span(a.cu_k, s_req, a.total_k, p.k0, p.lk);
  p.prefix = a.prefix ? a.prefix[s_req] : 0;
  p.t0 = s_tile * span;
  // keys that the tile's last query sees, the most; and its first, the fewest
  const int most = visible(min(p.lq, p.t0 + span) - 1, p.lq, p.lk, p.prefix);
  const int fewest = visible(p.t0, p.lq, p.lk, p.prefix);
  const int n = (most + kKeys - 1) / kKeys;

  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(&s_tmem)),
                 "r"(512u));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_tmem;
  // position of a tile's K or V in the order of the loads, in units of SPT slots: the order in
  // which the MMAs take them
  auto k_unit = [&](int j) { return NQ == 2 ? 2 * j : (j == 0 ? 0 : 2 * j - 1); };
  auto v_unit = [&](int j) { return NQ == 2 ? 2 * j + 1 : min(2 * j + 2, n + j); };

  // A row whose sum meets an infinity or a NaN may owe it to a value that it does not see (weight
  // zero times infinity): then the CTA does its tile once more, with such values taken out of the
  // V tiles that some of its rows see in part.
  //
  // A row of 128 logits takes more registers than 1/12 of an SM's: where there are twelve warps, the
  // first warpgroup gives some of its own. (80 + 2·208)·128 of the 168·384 that the block was
  // launched with.
  if (warp < 4) {
   if constexpr (NQ == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 80;");
   for (int pass = 0; pass < 2; ++pass) {
    const int load0 = pass * 2 * n * SPT, job0 = pass * NQ * n;
    if (warp == 0) {
      if (lane == 0 && n > 0) {
        // ---- producer ----
        bool ok = true;
        int load = load0;
        if (pass == 0) {
          // bytes of whole boxes: what lies out of bounds arrives as zeros
          mbar_expect_tx(&q_full, (uint32_t)(NQ * HD / 64 * tok * group * 128));
#pragma unroll
          for (int q = 0; q < NQ; ++q)
#pragma unroll
            for (int kb = 0; kb < HD / 64; ++kb)
              tma_load_3d(sQ + q * C::Q_TILE + kb * 16384, &tmQ, &q_full, kb * 64, kv * group,
                          p.q0 + p.t0 + q * tok);
        }
        auto slot_of = [&]() -> uint8_t* {
          const int s = load % SLOTS;
          if (load >= SLOTS)
            ok = ok && bar_wait(&empty[s], (load / SLOTS - 1) & 1, a.err, tc::ERR_TIMEOUT_PRODUCER);
          if (!ok) return nullptr;
          mbar_expect_tx(&full[s], C::SLOT);
          ++load;
          return base + s * C::SLOT;
        };
        auto load_k = [&](int j) {
#pragma unroll
          for (int h = 0; h < SPT; ++h) {
            uint8_t* dst = slot_of();
            if (!dst) return;
            uint64_t* bar = &full[(load - 1) % SLOTS];
#pragma unroll
            for (int kb = 0; kb < HD / 64 / SPT; ++kb)
              tma_load_3d(dst + kb * 16384, &tmK, bar, (h * (HD / 64 / SPT) + kb) * 64, kv,
                          p.k0 + j * kKeys);
          }
        };
        auto load_v = [&](int j) {
#pragma unroll
          for (int h = 0; h < SPT; ++h) {
            uint8_t* dst = slot_of();
            if (!dst) return;
            uint64_t* bar = &full[(load - 1) % SLOTS];
#pragma unroll
            for (int kb = 0; kb < HD / 64; ++kb)
              tma_load_3d(dst + kb * (C::VKEYS * 128), &tmV, bar, kb * 64, kv,
                          p.k0 + j * kKeys + h * C::VKEYS);
          }
        };
        if constexpr (NQ == 2) {
          for (int j = 0; j < n && ok; ++j) {
            load_k(j);
            if (ok) load_v(j);
          }
        } else {
          load_k(0);
          for (int j = 0; j < n && ok; ++j) {
            if (j + 1 < n) load_k(j + 1);
            if (ok) load_v(j);
          }
        }
        // no copy into this CTA's shared memory may be in flight when it exits
        bar_wait(&q_full, 0, a.err, tc::ERR_TIMEOUT_PRODUCER, false);
        for (int l = max(load0, load - SLOTS); l < load; ++l)
          bar_wait(&full[l % SLOTS], (l / SLOTS) & 1, a.err, tc::ERR_TIMEOUT_PRODUCER, false);
      }
      __syncwarp();
    } else if (warp <= NQ) {
      if (n > 0) {
        // ---- MMA issuers: with two tiles of rows a warp for each, so that neither waits for the
        // other's weights. A tile's logits and weights share their columns, and MMAs of one thread
        // run in order: P·V j, then the logits that overwrite P.
        constexpr uint32_t id_s = tc::idesc_f16<T>(128, kKeys);
        constexpr uint32_t id_o = tc::idesc_f16<T>(128, HD) | (1u << 16);  // V is MN-major
        const int q = warp - 1;
        const uint32_t ring = __shfl_sync(~0u, smem_u32(base), 0), tm = __shfl_sync(~0u, tmem, 0);
        const uint32_t qs = ring + SLOTS * C::SLOT + q * C::Q_TILE, to = tm + C::O_COL + q * HD;
        bool ok = bar_wait(&q_full, 0, a.err, tc::ERR_TIMEOUT_MMA);
        auto full_of = [&](int load) {
          return bar_wait(&full[load % SLOTS], (load / SLOTS) & 1, a.err, tc::ERR_TIMEOUT_MMA);
        };
        auto job_of = [&](int j) { return job0 + (NQ == 2 ? 2 * j + q : j); };
        auto qk = [&](int j) {
          const int buf = job_of(j) & 1, load = load0 + k_unit(j) * SPT;
#pragma unroll
          for (int h = 0; h < SPT; ++h) {
            if (!ok || !(ok = full_of(load + h))) return;
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
            }
            __syncwarp();
          }
        };
        auto pv = [&](int j) {
          const int job = job_of(j), buf = job & 1, load = load0 + v_unit(j) * SPT;
          // V is there before the weights are; these come in two halves of the keys
#pragma unroll
          for (int h = 0; h < SPT; ++h)
            if (!ok || !(ok = full_of(load + h))) return;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            if (!(ok = bar_wait(&p_full[buf][h], (job >> 1) & 1, a.err, tc::ERR_TIMEOUT_MMA)))
              return;
            tc_fence_after();
            const int slot = (load + h * (SPT - 1)) % SLOTS;
            const uint64_t dv = sdesc<128>(ring + slot * C::SLOT, 1024, C::VKEYS * 128) +
                                (SPT == 1 ? 512 * h : 0);
            const uint32_t tp = tm + buf * kKeys + 32 * h;
            const uint32_t more = (j | h) != 0;
            if (elect_one()) {
#pragma unroll
              for (int k = 0; k < 4; ++k)  // 16 keys (2048 bytes of V rows) a step
                umma_f16_ta(to, tp + 8 * k, dv + 128 * k, id_o, k == 0 ? more : 1u);
              if (h == 1) umma_commit(&pv_done[buf]);
              if (h >= 2 - SPT) umma_commit(&empty[slot]);
            }
            __syncwarp();
          }
        };
        constexpr int kAhead = NQ == 2 ? 1 : 2;  // tiles of logits before the first weights
#pragma unroll
        for (int j = 0; j < kAhead; ++j)
          if (j < n) qk(j);
        for (int j = 0; j < n && ok; ++j) {
          pv(j);
          if (j + kAhead < n) qk(j + kAhead);
        }
        // every issued MMA completes before TMEM is released
        if (elect_one()) umma_commit(&drain);
        __syncwarp();
        bar_wait(&drain, pass, a.err, tc::ERR_TIMEOUT_MMA, false);
      }
      __syncwarp();
    }
    if (!block_any<C::THREADS>(false)) break;
   }
  } else {
   if constexpr (NQ == 2) asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
   for (int pass = 0; pass < 2; ++pass) {
      bool again = false;
      const int load0 = pass * 2 * n * SPT, job0 = pass * NQ * n;
      // ---- softmax and output: one thread per query row ----
      const int wg = (warp - 4) >> 2, q4 = warp & 3, r = q4 * 32 + lane;
      const uint32_t tl = tmem + ((uint32_t)(q4 * 32) << 16);
      const uint32_t tO = tl + C::O_COL + wg * HD;
      const int i = p.t0 + wg * tok + r / group;     // the row's query
      const bool row = r < tok * group && i < p.lq;
      const int mine = row ? visible(i, p.lq, p.lk, p.prefix) : 0;
      // keys below this need no mask in this warpgroup's rows
      const int clear = p.t0 + wg * tok < p.lq ? visible(p.t0 + wg * tok, p.lq, p.lk, p.prefix) : 0;
      float m = -INFINITY, l = 0.f;
      bool ok = true;
      for (int j = 0; j < n; ++j) {
        const int job = job0 + (NQ == 2 ? 2 * j + wg : j), buf = job & 1;
        if (ok) ok = bar_wait(&s_full[buf], (job >> 1) & 1, a.err, tc::ERR_TIMEOUT_EPI);
        ok = __all_sync(~0u, ok);
        if (ok) {
          tc_fence_after();
          float s[128];
#pragma unroll
          for (int q = 0; q < 4; ++q)
            tmem_ld32_async(tl + buf * kKeys + 32 * q, reinterpret_cast<uint32_t*>(s) + 32 * q);
          tmem_wait_ld();
          float c = a.c;
          if (c <= 0.f) {  // the largest logit is not the largest product: scale first
#pragma unroll
            for (int u = 0; u < 128; ++u) s[u] *= c;
            c = 1.f;
          }
          if ((j + 1) * kKeys > clear) {
            const int lim = mine - j * kKeys;
#pragma unroll
            for (int u = 0; u < 128; ++u) s[u] = u < lim ? s[u] : -INFINITY;
          }
          const float top = max128(s) * c;
          if (j == 0) {
            m = top;
          } else if (__any_sync(~0u, top > m + kPromptGrow)) {
            // the sums so far are complete once the P·V before has finished
            const int prev = NQ == 2 ? job - 2 : job - 1;
            ok = bar_wait(&pv_done[prev & 1], (prev >> 1) & 1, a.err, tc::ERR_TIMEOUT_EPI);
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
          const float ref = m == -INFINITY ? 0.f : m;
          const uint64_t c2 = pack2(c, c), r2 = pack2(-ref, -ref);
          uint64_t sum0 = 0, sum1 = 0;  // two zeros each
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            uint32_t w[16];
#pragma unroll
            for (int u = 0; u < 16; ++u) {
              const int at = 32 * q + 2 * u;
              uint64_t x = fma2(pack2(s[at], s[at + 1]), c2, r2);
              const float2 f = unpack2(x);
              x = pack2(exp2_fast(f.x), exp2_fast(f.y));
              if (u & 1) sum1 = add2(sum1, x);
              else sum0 = add2(sum0, x);
              // weights in the type of V, as a 16-bit product asks; their sum is of the fp32 ones
              const float2 e = unpack2(x);
              w[u] = Tr<T>::pack(e.x, e.y);
            }
            tmem_st16(tl + buf * kKeys + 16 * q, w);
            if (q == 1) {  // the first 64 weights may go
              tmem_wait_st();
              tc_fence_before();
              __syncwarp();
              if (pass == 0 && lane == 0) mbar_arrive(&p_full[buf][0]);
            }
          }
          const float2 sums = unpack2(add2(sum0, sum1));
          l += sums.x + sums.y;
          tmem_wait_st();
          tc_fence_before();
        }
        if (pass == 1 && (j + 1) * kKeys > fewest) {
          // V rows of this tile, in halves for two warpgroups: values that are no numbers become
          // zero; s_bad keeps the first key of the request that lost one
          const int load = load0 + v_unit(j) * SPT;
#pragma unroll
          for (int h = 0; h < SPT; ++h) {
            const int s = (load + h) % SLOTS;
            if (ok) ok = bar_wait(&full[s], ((load + h) / SLOTS) & 1, a.err, tc::ERR_TIMEOUT_EPI);
            ok = __all_sync(~0u, ok);
            if (!ok) break;
            for (int v = tid - 128; v < C::SLOT / 16; v += NQ * 128) {
              const int key = j * kKeys + h * C::VKEYS + (v / 8) % C::VKEYS;
              uint4* at = reinterpret_cast<uint4*>(base + s * C::SLOT) + v;
              uint4 x = *at;
              T* e = reinterpret_cast<T*>(&x);
              bool hit = false;
#pragma unroll
              for (int u = 0; u < 8; ++u)
                if (!isfinite(Tr<T>::f(e[u]))) {
                  e[u] = Tr<T>::t(0.f);
                  hit = true;
                }
              if (hit) {
                *at = x;
                if (key < p.lk) atomicMin(&s_bad, key);
              }
            }
          }
          fence_async_smem();
          named_sync<1, NQ * 128>();
        }
        __syncwarp();
        if (ok && lane == 0) {
          if (pass == 1) mbar_arrive(&p_full[buf][0]);  // only now is V what it should be
          mbar_arrive(&p_full[buf][1]);
        }
      }
      if (n > 0) {
        const int last = job0 + (NQ == 2 ? 2 * (n - 1) + wg : n - 1);
        if (ok) ok = bar_wait(&pv_done[last & 1], (last >> 1) & 1, a.err, tc::ERR_TIMEOUT_EPI);
        ok = __all_sync(~0u, ok);
        tc_fence_after();
      }
      // ---- o = O / l ----
      T* out = reinterpret_cast<T*>(a.out) + (int64_t)(p.q0 + i) * a.o_tok +
               (int64_t)(kv * group + r % group) * a.o_head;
      const float inv = 1.f / l;
      bool odd = false, all = true;  // some, and every, element that is no number
#pragma unroll 1
      for (int d = 0; d < HD; d += 32) {
        uint32_t o[32];
        if (n > 0 && ok) tmem_ld32(tO + d, o);
        uint4 pk[4];
        uint32_t* pw = reinterpret_cast<uint32_t*>(pk);
#pragma unroll
        for (int u = 0; u < 16; ++u) {
          float x = __uint_as_float(o[2 * u]) * inv, y = __uint_as_float(o[2 * u + 1]) * inv;
          if (mine == 0) x = y = 0.f;
          else if (!ok) x = y = NAN;
          const bool fx = isfinite(x), fy = isfinite(y);
          odd |= !fx || !fy;
          all &= !fx && !fy;
          pw[u] = Tr<T>::pack(x, y);
        }
        if (row)
#pragma unroll
          for (int u = 0; u < 4; ++u) reinterpret_cast<uint4*>(out + d)[u] = pk[u];
      }
      tc_fence_before();
      again = row && odd && ok;
      if (pass == 1) {
        named_sync<1, NQ * 128>();  // s_bad is final, and so is the other warpgroup's tile
        // rows that do see a value that was taken out, unless they are NaN throughout as it is
        unsigned redo = __ballot_sync(~0u, row && ok && mine > s_bad && !all);
        while (redo) {
          const int src = __ffs(redo) - 1;
          redo &= redo - 1;
          const int rr = q4 * 32 + src, ii = p.t0 + wg * tok + rr / group;
          const int64_t h = kv * group + rr % group;
          const PromptKV<T> src_kv{
              reinterpret_cast<const T*>(a.k) + p.k0 * a.k_tok + kv * a.k_head,
              reinterpret_cast<const T*>(a.v) + p.k0 * a.v_tok + kv * a.v_head, a.k_tok, a.v_tok};
          attend_row(reinterpret_cast<const T*>(a.q) + (p.q0 + ii) * a.q_tok + h * a.q_head, HD,
                     visible(ii, p.lq, p.lk, p.prefix), a.c, src_kv,
                     reinterpret_cast<T*>(a.out) + (p.q0 + ii) * a.o_tok + h * a.o_head);
        }
      }
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

}  // namespace paged
}  // namespace pi0
