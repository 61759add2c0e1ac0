// prefix_fa.cuh -- shared-prefix attention on the tensor cores (tcgen05), bf16.
//
// The mathematics is that of prefix_attn.cuh; this is the kernel for work with enough query rows
// to fill 128-row tiles.  An item is a run of up to T * (128 / G) tokens of one key head: T query
// tiles of 128 rows, row r of a tile = (token r / G, query head r % G), which share every key
// tile.  An item reads prefix tiles [p0, p0 + np) and, behind them, the own keys of its sequence:
//   whole items   one sequence's tokens against the whole prefix and its own keys; the result is
//                 final (nothing to join);
//   prefix items  tokens of the whole batch, regardless of their sequences, against a part of the
//                 prefix; the result is one of the parts that sp_join_kernel joins.
//
// Roles of a CTA (one per SM, persistent): warps 4t .. 4t+3 are the softmax of query tile t, one
// row per thread; then one warp that issues the TMA loads and one MMA issuer warp per query tile.
// S_t = Q_t K^T (128 x 64) and O_t (128 x D) live in tensor memory, P_t goes back there as bf16;
// S of the next key tile is issued before P V of the present one.
//
// Per query tile and 64 keys there are 8192 exponentials (16 per clock and SM: 512 clocks; a quarter
// of them run as a polynomial on the FMA pipe) and 4 * 128 * 64 * D tensor FLOPs (48 clocks per 128 x
// 64 x 16 MMA of S, at D = 128 64 clocks per 128 x 128 x 16 MMA of P V).  Neither bounds it: at D = 128
// with two query tiles a step takes 2290 clocks, of which the MMAs fill 1280, and dropping the
// exponentials, the MMAs, or both in a test build leaves 98, 89 and 62 % of the time -- the hand-overs
// between softmax, issuer and tensor core (commit, mbarrier, wake-up) do, once per 64 keys.  With P beside
// S and O of 128 columns for each query tile, tensor memory holds one such step of two query tiles; steps
// of 128 keys with P over S (2 x 128 + 2 x 128 columns) would halve the hand-overs and have not been built.
// Measured: 16 sequences of 700 to 1024 tokens behind 4096 keys, 32/8 heads of 128, 980 GFLOP: 1115 us in
// calls one after another, at power-capped clocks (0.52 of the measured bf16 burst rate, 0.64 of the
// sustained one); 990 us in a short run (0.59 of burst).  In short runs, two threads to a row (32 keys
// each, twice the warps) 1075 us; two S buffers with P over S, so that S of the next tile and the store of
// P wait for nothing, 1000 us; both 1098 us.
//
// Roundings, each within those of one bf16 output: P goes to bf16 for its product (at most half a step,
// 2^-8 relative, averaged over the keys) while its sum stays in float32; the polynomial share of the
// exponentials is within 1.1e-4 (below 2^-12), the others are ex2.approx (2^-22).
#pragma once

#include "attn.cuh"
#include "prefix_attn.cuh"

namespace fcv {

constexpr int kSfKeys = 64;
constexpr int kSfRing = 4;

template <int D>
struct SpFa {
  static constexpr int T = D == 64 ? 3 : 2;         // query tiles of an item
  static constexpr int QBUF = D == 64 ? 2 : 1;      // items' Q in flight
  static constexpr int STAGES = D == 64 ? 6 : 5;    // key tiles in flight
  static constexpr int SUB = D / 64;                // 128-byte column blocks of a row
  static constexpr int Q_TILE = 128 * D * 2;
  static constexpr int KV_TILE = kSfKeys * D * 2;
  static constexpr int OFF_KV = QBUF * T * Q_TILE;  // per stage: K, then V
  static constexpr int OFF_BAR = OFF_KV + STAGES * 2 * KV_TILE;
  // mbarriers
  static constexpr int bQFull = 0, bQEmpty = bQFull + QBUF, bKvFull = bQEmpty + QBUF, bKvEmpty = bKvFull + STAGES;
  static constexpr int bSFull = bKvEmpty + STAGES, bSEmpty = bSFull + T, bPFull = bSEmpty + T, bODone = bPFull + T;
  static constexpr int bOFinal = bODone + T, bOEmpty = bOFinal + T, bInfoFull = bOEmpty + T;
  static constexpr int bInfoEmpty = bInfoFull + kSfRing, bDrain = bInfoEmpty + kSfRing, bCount = bDrain + T;
  static constexpr int RING_OFF = (bCount * 8 + 8 + 15) / 16 * 16;
  // TMEM columns: S_t (64), P_t (32), O_t (D)
  static constexpr int cS = 0, cP = 64 * T, cO = cP + 32 * T;
  static_assert(cO + D * T <= 512, "TMEM columns");
  static constexpr int PRODUCER = 4 * T;            // first warp behind the softmax warps
  static constexpr int THREADS = 32 * (4 * T + 4);
};

// What the roles need of an item; ntok == 0 marks the end of the CTA's items.
struct SfSlot {
  int tok0, ntok;   // first token and tokens
  int hk;           // key head
  int p0, np;       // prefix tiles
  int nk, rel;      // own keys of the sequence; nk - nq + (index of tok0 in its sequence)
  int own;          // first own key row
  int part;         // part that the result is, or -1: final
  int n[3];         // key tiles of each query tile (0: no tokens)
};
template <int D>
constexpr int sf_smem_bytes() {
  return 1024 + SpFa<D>::OFF_BAR + (SpFa<D>::RING_OFF + kSfRing * static_cast<int>(sizeof(SfSlot)) + 127) / 128 * 128;
}
static_assert(sf_smem_bytes<64>() <= 227 * 1024 && sf_smem_bytes<128>() <= 227 * 1024, "shared memory");

struct SfArgs {
  SpArgs a;
  int tile_tokens;      // 128 / G
  // whole items: the list of (sequence, block) entries that sp_list_kernel wrote; count[0] entries,
  // count[1] the next item to be taken
  const int2* list;
  int* count;
  int list_cap;
  // prefix items: blocks of T * tile_tokens tokens x key heads x parts
  int prefix_items, prefix_blocks;
  int none_row;         // a row number behind the own keys' tensor: reads as zeros
};

// The list of whole items, longest first: entry = (sequence, block of `block` tokens).  One block
// of threads; a warp takes a sequence, its lanes the blocks.  Entries are ordered by a counting
// sort over their key tiles; their order inside a bucket is free, since items do not depend on it.
__global__ void __launch_bounds__(1024) sp_list_kernel(const SpArgs a, int block, int2* list, int cap, int* count) {
  griddep_wait();
  griddep_launch();
  __shared__ int hist[1024], most, total;
  __shared__ int2 lens[1024];  // queries and own keys of the first sequences; later ones are read each time
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  auto read = [&](int b, bool report) -> int2 {
    const int c0 = a.cu[b], c1 = a.cu[b + 1];
    int nq = c1 - c0;
    const int nk = a.kv_lens ? a.kv_lens[b] : nq;
    if (c0 < 0 || c1 < c0 || c1 > a.N) {
      if (report) record_error(611);
      nq = 0;
    }
    return make_int2(nq, nk);
  };
  for (int b = tid; b < a.B; b += 1024) {
    const int2 s = read(b, true);
    if (b < 1024) lens[b] = s;
    if (s.x == 0) sp_sequence(a, b, true);  // without queries: no item will check its own keys
  }
  hist[tid] = 0;
  if (tid == 0) most = 1;
  __syncthreads();
  auto each = [&](auto f) {
    for (int b = warp; b < a.B; b += 32) {
      const int2 s = b < 1024 ? lens[b] : read(b, false);
      for (int i = lane; (long)i * block < s.x; i += 32) {
        const int last = min((long)(i + 1) * block, (long)s.x) - 1;
        f(b, i, (sp_limit_at(a, s.y, s.y - s.x + last) + kSfKeys - 1) / kSfKeys);
      }
    }
  };
  each([&](int, int, int cost) { atomicMax(&most, cost); });
  __syncthreads();
  const int top = most;
  auto bucket = [&](int cost) { return 1023 - static_cast<int>((long)max(0, min(cost, top)) * 1023 / top); };
  each([&](int, int, int cost) { atomicAdd(&hist[bucket(cost)], 1); });
  __syncthreads();
  // exclusive prefix sum of the 1024 buckets
  const int own = hist[tid];
  int sum = own;
#pragma unroll
  for (int w = 1; w < 32; w <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, sum, w);
    if (lane >= w) sum += v;
  }
  __shared__ int warps[32];
  if (lane == 31) warps[warp] = sum;
  __syncthreads();
  if (warp == 0) {
    int v = warps[lane];
#pragma unroll
    for (int w = 1; w < 32; w <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, v, w);
      if (lane >= w) v += u;
    }
    warps[lane] = v;
  }
  __syncthreads();
  sum += warp > 0 ? warps[warp - 1] : 0;
  hist[tid] = sum - own;
  if (tid == 1023) total = sum;
  __syncthreads();
  each([&](int b, int i, int cost) {
    const int at = atomicAdd(&hist[bucket(cost)], 1);
    if (at < cap) list[at] = make_int2(b, i);  // cu_seqlens that run back could name more blocks than there are
  });
  if (tid == 0) {
    count[0] = min(total, cap);
    count[1] = 0;
  }
}

template <int D>
__global__ void __launch_bounds__(SpFa<D>::THREADS, 1)
    sp_fa_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmPK,
                 const __grid_constant__ CUtensorMap tmPV, const __grid_constant__ CUtensorMap tmK,
                 const __grid_constant__ CUtensorMap tmV, const __grid_constant__ CUtensorMap tmV8,
                 const __grid_constant__ CUtensorMap tmV1, const SfArgs f) {
  using C = SpFa<D>;
  constexpr int T = C::T, STAGES = C::STAGES, QBUF = C::QBUF, SUB = C::SUB;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const SpArgs& A = f.a;
  const uint32_t s0 = smem_u32(smem);
  const uint32_t sQ = s0, sKV = s0 + C::OFF_KV;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::OFF_BAR);
  auto bar = [&](int i) { return smem_u32(bars + i); };
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + C::bCount);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  SfSlot* ring = reinterpret_cast<SfSlot*>(smem + C::OFF_BAR + C::RING_OFF);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  int prefix_items = f.prefix_items, prefix_parts = A.prefix_parts, prefix_ctas = gridDim.x;
  if (A.split.n > 0) {
    griddep_wait();
    griddep_launch();  // only after the wait: the kernels behind this one rely on it (fcv_common.cuh)
    // this kernel's share of the SMs follows from the own keys
    __shared__ unsigned long long units;
    if (threadIdx.x == 0) units = 0;
    __syncthreads();
    long mine = 0;
    for (int b = threadIdx.x; b < A.B; b += C::THREADS) {
      const SpSeq s = sp_sequence(A, b, false);
      mine += ss_count(A, s.nq, s.nk).all(A.Hkv);
    }
#pragma unroll
    for (int w = 16; w > 0; w >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, w);
    if (lane == 0) atomicAdd(&units, static_cast<unsigned long long>(mine));
    __syncthreads();
    const int pick = sp_pick(A.split, static_cast<long>(units));
    prefix_parts = A.split.parts[pick];
    prefix_ctas = A.split.ctas[pick];
    if (static_cast<int>(blockIdx.x) >= prefix_ctas) return;  // leaves its SM to the own keys
    prefix_items = f.prefix_blocks * A.Hkv * prefix_parts;
  }

  if (threadIdx.x == 0) {
    for (int i = 0; i < QBUF; ++i) {
      mbar_init(bar(C::bQFull + i), 1);
      mbar_init(bar(C::bQEmpty + i), T);
    }
    for (int t = 0; t < T; ++t) {
      mbar_init(bar(C::bSFull + t), 1);
      mbar_init(bar(C::bSEmpty + t), 4);
      mbar_init(bar(C::bPFull + t), 4);
      mbar_init(bar(C::bODone + t), 1);
      mbar_init(bar(C::bOFinal + t), 1);
      mbar_init(bar(C::bOEmpty + t), 4);
      mbar_init(bar(C::bDrain + t), 1);
    }
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(bar(C::bKvFull + i), 1);
      mbar_init(bar(C::bKvEmpty + i), T);
    }
    for (int i = 0; i < kSfRing; ++i) {
      mbar_init(bar(C::bInfoFull + i), 1);
      mbar_init(bar(C::bInfoEmpty + i), T + 4 * T);
    }
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tmQ);
    tma_prefetch_desc(&tmPK);
    tma_prefetch_desc(&tmPV);
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
  }
  if (warp == C::PRODUCER + 1) {
    tmem_alloc(smem_u32(tmem_slot), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  if (A.split.n == 0) {
    griddep_wait();
    griddep_launch();  // only after the wait, as above
  }

  if (warp >= C::PRODUCER) {
    if constexpr (T == 3) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kFaRegsProducer));
    if (warp == C::PRODUCER && lane == 0) {
      // ---------------- TMA producer: resolves items, publishes them, loads Q and the key tiles
      const int block = T * f.tile_tokens;
      const int items = f.list ? min(max(f.count[0], 0), f.list_cap) * A.Hkv : prefix_items;
      int g = 0, i = 0;
      bool ok = true;
      auto take = [&](int now) -> int { return f.list ? atomicAdd(f.count + 1, 1) : now; };
      auto resolve = [&](int it, SfSlot& o) -> bool {  // false: nothing to do
        int seen[3];
        if (f.list) {
          o.hk = it % A.Hkv;
          const int2 e = f.list[it / A.Hkv];
          SpSeq s;
          {  // as sp_sequence(), by one thread
            const int c0 = A.cu[e.x], c1 = A.cu[e.x + 1];
            s.q0 = c0;
            s.nq = c1 - c0;
            if (c0 < 0 || c1 < c0 || c1 > A.N) s.q0 = s.nq = 0;
            s.base = A.kv_base ? A.kv_base[e.x] : s.q0;
            s.nk = A.kv_lens ? A.kv_lens[e.x] : s.nq;
            if (s.nk < 0 || s.base < 0 || s.base + s.nk > A.kv_rows) {
              if (s.nk != 0) record_error(612);
              s.base = 0;
              s.nk = 0;
            }
          }
          const int i0 = e.y * block;
          if (i0 >= s.nq) return false;
          o.tok0 = s.q0 + i0;
          o.ntok = min(block, s.nq - i0);
          o.p0 = 0;
          o.np = (A.P + kSfKeys - 1) / kSfKeys;
          o.nk = s.nk;
          o.rel = s.nk - s.nq + i0;
          o.own = static_cast<int>(s.base);
          o.part = -1;
        } else {
          o.part = it % prefix_parts;
          it /= prefix_parts;
          o.hk = it % A.Hkv;
          const long t0 = (long)(it / A.Hkv) * block;
          const int first = max(0, min(A.N, A.cu[0])), end = max(0, min(A.N, A.cu[A.B]));
          const long lo = t0 > first ? t0 : first, hi = min(t0 + block, (long)end);
          if (lo >= hi) return false;
          o.tok0 = static_cast<int>(lo);
          o.ntok = static_cast<int>(hi - lo);
          int t1;
          sp_piece((A.P + kSfKeys - 1) / kSfKeys, prefix_parts, sp_least<bf16>(), o.part, o.p0, t1);
          o.np = t1 - o.p0;
          o.nk = o.rel = o.own = 0;
        }
#pragma unroll
        for (int t = 0; t < 3; ++t) {
          const int r0 = t * f.tile_tokens;
          seen[t] = 0;
          if (t < T && r0 < o.ntok) {
            const int last = min(r0 + f.tile_tokens, o.ntok) - 1;
            // at least one tile: a row that sees nothing still has to be written
            seen[t] = max(1, o.np + (o.part < 0 ? (sp_limit_at(A, o.nk, o.rel + last) + kSfKeys - 1) / kSfKeys : 0));
          }
          o.n[t] = seen[t];
        }
        return true;
      };
      auto publish = [&](const SfSlot& o) -> bool {
        const int sl = i % kSfRing;
        if (!mbar_wait(bar(C::bInfoEmpty + sl), ((i / kSfRing) & 1) ^ 1, 640, abort_flag)) return false;
        ring[sl] = o;
        mbar_arrive(bar(C::bInfoFull + sl));
        return true;
      };
      SfSlot o{};
      for (int it = take(blockIdx.x); it < items && ok; it = take(it + prefix_ctas)) {
        if (!resolve(it, o)) continue;
        const int qb = i % QBUF;
        if (!publish(o)) { ok = false; break; }
        if (!mbar_wait(bar(C::bQEmpty + qb), ((i / QBUF) & 1) ^ 1, 641, abort_flag)) { ok = false; break; }
        mbar_arrive_expect_tx(bar(C::bQFull + qb), T * f.tile_tokens * A.G * D * 2);
#pragma unroll
        for (int t = 0; t < T; ++t)  // tiles without tokens load other rows (or zeros): unused
#pragma unroll
          for (int u = 0; u < SUB; ++u)
            tma_load_3d(sQ + (qb * T + t) * C::Q_TILE + u * 16384, &tmQ, bar(C::bQFull + qb), u * 64, o.hk * A.G,
                        o.tok0 + t * f.tile_tokens);
        int nkv = 0;
#pragma unroll
        for (int t = 0; t < T; ++t) nkv = max(nkv, o.n[t]);
        for (int j = 0; j < nkv; ++j, ++g) {
          const int st = g % STAGES;
          if (!mbar_wait(bar(C::bKvEmpty + st), ((g / STAGES) & 1) ^ 1, 642, abort_flag)) { ok = false; break; }
          const uint32_t full = bar(C::bKvFull + st);
          const uint32_t dk = sKV + st * 2 * C::KV_TILE, dv = dk + C::KV_TILE;
          mbar_arrive_expect_tx(full, 2 * C::KV_TILE);
          if (j < o.np) {  // rows past the prefix read as zeros
            const int y = (o.p0 + j) * kSfKeys;
#pragma unroll
            for (int u = 0; u < SUB; ++u) {
              tma_load_2d(dk + u * 8192, &tmPK, full, o.hk * D + u * 64, y);
              tma_load_2d(dv + u * 8192, &tmPV, full, o.hk * D + u * 64, y);
            }
          } else {
            const int at = (j - o.np) * kSfKeys, y = o.own + at;
            const int valid = max(0, min(kSfKeys, o.nk - at));
#pragma unroll
            for (int u = 0; u < SUB; ++u) {
              const int x = o.hk * D + u * 64;
              tma_load_2d(dk + u * 8192, &tmK, full, x, y);
              if (valid == kSfKeys) {
                tma_load_2d(dv + u * 8192, &tmV, full, x, y);
              } else {
                // the sequence ends inside the tile: rows behind it may hold anything, and a weight of
                // zero does not stop a NaN, so the tile is put together from boxes of 8 rows and of
                // one row, those without keys from behind the tensor (zeros)
                const int none = f.none_row;
                for (int r = 0; r < kSfKeys; r += 8) {
                  if (r + 8 <= valid || r >= valid) {
                    tma_load_2d(dv + u * 8192 + r * 128, &tmV8, full, x, r < valid ? y + r : none);
                  } else {
                    for (int e = r; e < r + 8; ++e)
                      tma_load_2d(dv + u * 8192 + e * 128, &tmV1, full, x, e < valid ? y + e : none);
                  }
                }
              }
            }
          }
        }
        ++i;
      }
      if (ok) {
        SfSlot end{};
        publish(end);
      }
      // our own copies have landed before the CTA may exit (all phases already issued)
      for (int k = (g > STAGES ? g - STAGES : 0); k < g; ++k)
        mbar_wait(bar(C::bKvFull + k % STAGES), (k / STAGES) & 1, 643, nullptr);
      for (int k = (i > QBUF ? i - QBUF : 0); k < i; ++k)
        mbar_wait(bar(C::bQFull + k % QBUF), (k / QBUF) & 1, 644, nullptr);
    } else if (warp > C::PRODUCER && warp <= C::PRODUCER + T && lane == 0) {
      // ---------------- MMA issuer of slot t (see attn_fa_kernel: the same protocol)
      const int t = warp - C::PRODUCER - 1;
      constexpr uint32_t idesc_s = idesc_bf16_f32(128, kSfKeys, false, false);
      constexpr uint32_t idesc_o = idesc_bf16_f32(128, D, false, true);  // V is MN-major
      int sc = 0, pvc = 0, items_t = 0;
      int pv_g = 0, pv_item = 0;
      bool pv_on = false, pv_first = false, pv_last = false, ok = true, pend = false;
      auto issue_pv = [&]() -> bool {
        if (pv_on) {
          if (!mbar_wait(bar(C::bPFull + t), pvc & 1, 645, abort_flag)) return false;
          if (pv_first && !mbar_wait(bar(C::bOEmpty + t), (pv_item & 1) ^ 1, 646, abort_flag)) return false;
          tc_fence_after();
          const uint32_t v = sKV + (pv_g % STAGES) * 2 * C::KV_TILE + C::KV_TILE;
          // 64-column blocks of V are 8 KB apart; 16 keys further are 16 rows of 128 bytes
          const uint64_t dv = SUB == 1 ? sdesc_sw128(v) : sdesc_sw128_lbo(v, 8192);
#pragma unroll
          for (int k = 0; k < kSfKeys / 16; ++k)
            umma_bf16_ts(tmem + C::cO + D * t, tmem + C::cP + 32 * t + 8 * k, dv + 128 * k, idesc_o,
                         (!pv_first || k != 0) ? 1u : 0u);
          umma_commit(bar(C::bODone + t));
          if (pv_last) umma_commit(bar(C::bOFinal + t));
          ++pvc;
          umma_commit(bar(C::bKvEmpty + pv_g % STAGES));
        } else {
          mbar_arrive(bar(C::bKvEmpty + pv_g % STAGES));
        }
        return true;
      };
      int g = 0;
      for (int i = 0; ok; ++i) {
        const int sl = i % kSfRing;
        if (!mbar_wait(bar(C::bInfoFull + sl), (i / kSfRing) & 1, 639, abort_flag)) { ok = false; break; }
        const SfSlot a = ring[sl];
        mbar_arrive(bar(C::bInfoEmpty + sl));
        if (a.ntok == 0) break;
        const int rt = (t + i) % T;  // the item's query tile of this slot (rotates per item)
        int nkv = 0, nt = 0;
#pragma unroll
        for (int u = 0; u < T; ++u) {
          nkv = max(nkv, a.n[u]);
          if (u == rt) nt = a.n[u];
        }
        const int qb = i % QBUF;
        if (!mbar_wait(bar(C::bQFull + qb), (i / QBUF) & 1, 647, abort_flag)) { ok = false; break; }
        if (nt == 0) mbar_arrive(bar(C::bQEmpty + qb));
        for (int j = 0; j < nkv && ok; ++j, ++g) {
          const int st = g % STAGES;
          if (!mbar_wait(bar(C::bKvFull + st), (g / STAGES) & 1, 648, abort_flag)) { ok = false; break; }
          if (j < nt) {
            if (sc > 0 && !mbar_wait(bar(C::bSEmpty + t), (sc - 1) & 1, 649, abort_flag)) { ok = false; break; }
            tc_fence_after();
#pragma unroll
            for (int k = 0; k < D / 16; ++k) {
              const uint64_t dq = sdesc_sw128(sQ + (qb * T + rt) * C::Q_TILE + (k / 4) * 16384);
              const uint64_t dk = sdesc_sw128(sKV + st * 2 * C::KV_TILE + (k / 4) * 8192);
              umma_bf16(tmem + C::cS + kSfKeys * t, dq + 2 * (k % 4), dk + 2 * (k % 4), idesc_s, k != 0);
            }
            umma_commit(bar(C::bSFull + t));
            ++sc;
            if (j == nt - 1) umma_commit(bar(C::bQEmpty + qb));
          }
          if (pend && !issue_pv()) { ok = false; break; }
          pv_g = g;
          pv_on = j < nt;
          pv_first = j == 0;
          pv_last = j == nt - 1;
          pv_item = items_t;
          pend = true;
        }
        items_t += nt > 0 ? 1 : 0;
      }
      if (ok && pend) issue_pv();
      umma_commit(bar(C::bDrain + t));
      mbar_wait(bar(C::bDrain + t), 0, 650, nullptr);
    }
  } else {
    if constexpr (T == 3) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kFaRegsSoftmax));
    // ---------------- softmax of slot t: one row per thread
    const int t = warp >> 2;
    const int qd = warp & 3;
    const int r = qd * 32 + lane;  // row within the tile = TMEM lane
    const int r_tok = r / A.G, r_head = r - r_tok * A.G;
    const uint32_t lane_base = tmem + (static_cast<uint32_t>(qd * 32) << 16);
    const uint32_t colS = lane_base + C::cS + kSfKeys * t, colP = lane_base + C::cP + 32 * t,
                   colO = lane_base + C::cO + D * t;
    const float sl2 = A.scale_log2;
    int cnt = 0, it_t = 0;
    bool ok = true;
    bool pend = false, p_row = false;  // deferred epilogue of the slot's previous item
    int p_idx = 0, p_part = 0, p_head = 0;
    long p_tok = 0;
    float p_l = 0.f, p_m = 0.f;
    auto epilogue = [&]() -> bool {
      if (!mbar_wait(bar(C::bOFinal + t), p_idx & 1, 651, abort_flag)) return false;
      tc_fence_after();
      const bool some = p_l > 0.f || p_l != p_l;
      const float inv = some ? 1.f / p_l : 0.f;
      const long at = p_part < 0 ? 0 : ((long)p_part * A.N + p_tok) * A.H + p_head;
      bf16* orow = static_cast<bf16*>(A.out) + p_tok * A.out_stride + (long)p_head * D;
      float* frow = A.part_o + at * D;
      if (p_row && p_part >= 0) A.part_ml[at] = make_float2(p_m, p_l);
#pragma unroll
      for (int c = 0; c < D / 16; ++c) {
        uint32_t o[16];
        tmem_ld16(colO + 16 * c, o);
        tmem_wait_ld();
        if (c == D / 16 - 1) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(bar(C::bOEmpty + t));
        }
        if (p_row) {
          if (p_part < 0) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              uint32_t w[4];
#pragma unroll
              for (int e = 0; e < 4; ++e)
                w[e] = some ? pack_bf16x2(__uint_as_float(o[8 * h + 2 * e]) * inv,
                                          __uint_as_float(o[8 * h + 2 * e + 1]) * inv)
                            : 0u;  // saw no key
              *reinterpret_cast<uint4*>(orow + 16 * c + 8 * h) = make_uint4(w[0], w[1], w[2], w[3]);
            }
          } else {
#pragma unroll
            for (int h = 0; h < 4; ++h)
              *reinterpret_cast<uint4*>(frow + 16 * c + 4 * h) =
                  make_uint4(o[4 * h], o[4 * h + 1], o[4 * h + 2], o[4 * h + 3]);
          }
        }
      }
      pend = false;
      return true;
    };
    for (int i = 0; ok; ++i) {
      const int sl = i % kSfRing;
      if (!mbar_wait(bar(C::bInfoFull + sl), (i / kSfRing) & 1, 638, abort_flag)) { ok = false; break; }
      const SfSlot a = ring[sl];
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(C::bInfoEmpty + sl));
      if (a.ntok == 0) break;
      const int rt = (t + i) % T;
      int ntile = 0;
#pragma unroll
      for (int u = 0; u < T; ++u)
        if (u == rt) ntile = a.n[u];
      if (ntile == 0) continue;
      const int tok = rt * f.tile_tokens + r_tok;  // token of the item
      const bool row_ok = r_tok < f.tile_tokens && tok < a.ntok;
      const bool warp_rows = __any_sync(0xffffffffu, row_ok);
      // visible keys, counted from the item's first: the prefix tiles, then the own keys
      const int pre = min(a.np * kSfKeys, A.P - a.p0 * kSfKeys);
      const int lim = a.part < 0 ? sp_limit_at(A, a.nk, a.rel + min(tok, a.ntok - 1)) : 0;
      const int lmax = __reduce_max_sync(0xffffffffu, lim), lmin = __reduce_min_sync(0xffffffffu, lim);
      float m_ref = -INFINITY;
      float lsum[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      for (int j = 0; j < ntile; ++j, ++cnt) {
        if (!mbar_wait(bar(C::bSFull + t), cnt & 1, 652, abort_flag)) { ok = false; break; }
        tc_fence_after();
        // keys of this tile that the row sees, and the most and the fewest over the warp's rows
        const bool own = j >= a.np;
        const int k0 = (own ? j - a.np : j) * kSfKeys;
        const int nvis = (own ? lim : pre) - k0, vmax = (own ? lmax : pre) - k0, vmin = (own ? lmin : pre) - k0;
        const int nch = warp_rows ? min(2, max(0, (vmax + 31) / 32)) : 0;  // 32-key halves that some row sees
        uint32_t s[64];
        tmem_ld32(colS, *reinterpret_cast<uint32_t(*)[32]>(s));
        if (nch > 1) tmem_ld32(colS + 32, *reinterpret_cast<uint32_t(*)[32]>(s + 32));
        tmem_wait_ld();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(C::bSEmpty + t));
        if (vmin < kSfKeys) {
#pragma unroll
          for (int c = 0; c < 64; ++c)
            if (c >= nvis) s[c] = __float_as_uint(-INFINITY);
        }
        float mt = -INFINITY;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          if (c < nch) {
            float m8[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
              const uint32_t* v = s + 32 * c + 8 * u;
              m8[u] = fmax3_nan(fmax3_nan(__uint_as_float(v[0]), __uint_as_float(v[1]), __uint_as_float(v[2])),
                                fmax3_nan(__uint_as_float(v[3]), __uint_as_float(v[4]), __uint_as_float(v[5])),
                                fmax_nan(__uint_as_float(v[6]), __uint_as_float(v[7])));
            }
            mt = fmax3_nan(mt, fmax_nan(m8[0], m8[1]), fmax_nan(m8[2], m8[3]));
          }
        }
        const float m_tile = mt * sl2;
        const bool need = m_tile > m_ref + kRescaleThreshold;
        const float m_new = need ? m_tile : m_ref;
        bool o_ready = cnt == 0;
        if (j > 0 && __any_sync(0xffffffffu, need)) {
          if (!mbar_wait(bar(C::bODone + t), (cnt - 1) & 1, 653, abort_flag)) { ok = false; break; }
          tc_fence_after();
          o_ready = true;
          const float alpha = need ? ex2_approx(m_ref - m_new) : 1.0f;
#pragma unroll 1
          for (int piece = 0; piece < D / 16; ++piece) {
            uint32_t o[16];
            tmem_ld16(colO + 16 * piece, o);
            tmem_wait_ld();
#pragma unroll
            for (int d = 0; d < 16; ++d) o[d] = __float_as_uint(__uint_as_float(o[d]) * alpha);
            tmem_st16(colO + 16 * piece, o);
          }
          tmem_wait_st();
#pragma unroll
          for (int u = 0; u < 8; ++u) lsum[u] *= alpha;
        }
        m_ref = m_new;
        // a score that is NaN or +inf makes its row NaN, as it does in the formula (the polynomial
        // exponentials would drop it)
        const float mo = !(mt < INFINITY) ? __int_as_float(0x7fffffff) : (m_ref == -INFINITY ? 0.f : m_ref);
        uint32_t pw[32];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          if (c < nch) {
#pragma unroll
            for (int p = 0; p < 16; ++p) {
              float x0, x1, e0, e1;
              fma2(x0, x1, __uint_as_float(s[32 * c + 2 * p]), __uint_as_float(s[32 * c + 2 * p + 1]), sl2, sl2, -mo,
                   -mo);
              if (p % 8 < kFaPolyPairs) {
                exp2_poly2(x0, x1, e0, e1);
              } else {
                e0 = ex2_approx(x0);
                e1 = ex2_approx(x1);
              }
              add2(lsum[2 * (p & 3)], lsum[2 * (p & 3) + 1], lsum[2 * (p & 3)], lsum[2 * (p & 3) + 1], e0, e1);
              pw[16 * c + p] = pack_bf16x2(e0, e1);
            }
          } else {
#pragma unroll
            for (int p = 0; p < 16; ++p) pw[16 * c + p] = 0u;
          }
        }
        if (!o_ready) {
          if (!mbar_wait(bar(C::bODone + t), (cnt - 1) & 1, 654, abort_flag)) { ok = false; break; }
          tc_fence_after();
        }
        tmem_st32(colP, pw);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(C::bPFull + t));
        if (pend && !epilogue()) { ok = false; break; }
      }
      if (!ok) break;
      pend = true;
      p_idx = it_t++;
      p_row = row_ok;
      p_part = a.part;
      p_tok = a.tok0 + tok;
      p_head = a.hk * A.G + r_head;
      p_m = m_ref;
      p_l = ((lsum[0] + lsum[1]) + (lsum[2] + lsum[3])) + ((lsum[4] + lsum[5]) + (lsum[6] + lsum[7]));
    }
    if (ok && pend) epilogue();
  }
  tc_fence_before();
  __syncthreads();
  if (warp == C::PRODUCER + 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

}  // namespace fcv
