// prefix_stream.cuh -- the own keys of a decode step: few query rows against many ragged stretches.
//
// The mathematics is that of prefix_attn.cuh.  With up to 16 query rows (tokens x query heads of a
// key head) per sequence every key is used for a handful of products, so the keys' bytes bound it,
// and what matters is that the loads never pause.  The tiles of all (sequence, row block, key
// head) items are laid end to end and cut into equal stretches, one for each CTA, wherever the
// cuts fall: a CTA streams its stretch through one shared-memory ring without a break between
// items.  An item that lies inside one stretch leaves one part; an item that is cut leaves a part in
// every stretch it meets, which sp_join_kernel finds by the same arithmetic.
//
// One block for each item and part, instead, loses a few microseconds at each start and end: for 64
// sequences of 1 to 1024 keys (8 key heads of 128, 134 MB) behind 4096 the call then took 61 us of device
// time in one part each, 70 in two, 90 in four; it takes 43 us with the stretches, which run 34 to 35 us
// on 108 SMs beside the prefix parts on 40, 3.9 TB/s.  256 sequences (1.07 GB) on 100 SMs: 225 us,
// 4.7 TB/s.  18 CTAs alone took in 59 GB/s each.  Measured and not
// kept: a fifth stage paid for by a join in two rounds (49 against 44 us), a group of warps for every
// other item, and key heads outermost in the order (no change).
#pragma once

#include "prefix_attn.cuh"

namespace fcv {

template <int D>
struct SpStream {
  static constexpr int SUB = D / 64;
  static constexpr int TILE = kSpKeys * D * 2;
  static constexpr int Q_TILE = 16 * D * 2;
  static constexpr int STAGE = 2 * TILE + Q_TILE;  // K, V and, with an item's first tiles, its queries
  static constexpr int STAGES = D == 64 ? 10 : 4;
  static constexpr int WARPS = 8;                  // two groups of four: tiles j, j + 2, ... of an item each
  static constexpr int OFF_O = STAGES * STAGE;     // [warp][16][D] partial outputs
  static constexpr int OFF_ML = OFF_O + WARPS * 16 * D * 4;
  static constexpr int OFF_BAR = OFF_ML + WARPS * 16 * 8;
  static constexpr int RING = 4;                   // items published ahead
  static constexpr int THREADS = 32 * (WARPS + 1);
};
struct SsItem {
  int tok0, rows;  // first token, stacked rows (tokens x G)
  int hk, nk, rel; // key head, own keys, own position of the first token
  int t0, nt;      // key tiles; nt == 0 marks the end
  int slot;        // boundary slot, or -1: the item lies in this stretch as a whole
};
template <int D>
constexpr int ss_smem_bytes() {
  using C = SpStream<D>;
  return 1024 + C::OFF_BAR + (2 * C::STAGES + 2 * C::RING) * 8 + 64 + C::RING * static_cast<int>(sizeof(SsItem));
}
static_assert(ss_smem_bytes<64>() <= 227 * 1024 && ss_smem_bytes<128>() <= 227 * 1024, "shared memory");

// Barrier of the eight consumer warps.
__device__ __forceinline__ void ss_bar() { asm volatile("bar.sync 1, 256;" ::: "memory"); }

template <int D>
__global__ void __launch_bounds__(SpStream<D>::THREADS, 1)
    sp_stream_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                     const __grid_constant__ CUtensorMap tmV, const SpArgs a) {
  using C = SpStream<D>;
  constexpr int STAGES = C::STAGES, SUB = C::SUB;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t s0 = smem_u32(smem);
  float* so = reinterpret_cast<float*>(smem + C::OFF_O);
  float2* sml = reinterpret_cast<float2*>(smem + C::OFF_ML);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::OFF_BAR);
  auto full = [&](int i) { return smem_u32(bars + i); };
  auto empty = [&](int i) { return smem_u32(bars + STAGES + i); };
  auto info_full = [&](int i) { return smem_u32(bars + 2 * STAGES + i); };
  auto info_empty = [&](int i) { return smem_u32(bars + 2 * STAGES + C::RING + i); };
  long* sstart = reinterpret_cast<long*>(bars + 2 * STAGES + 2 * C::RING);  // first sequence, its first tile, total
  // the abort flag, and whether a consumer warp gave up on an item's announcement or on its tiles
  volatile int* abort_flag = reinterpret_cast<volatile int*>(sstart + 3);
  volatile int* no_item = abort_flag + 1;
  volatile int* no_tile = abort_flag + 2;
  SsItem* ring = reinterpret_cast<SsItem*>(sstart + 5);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  if (tid == 0) {
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(full(i), 1);
      mbar_init(empty(i), 4);
    }
    for (int i = 0; i < C::RING; ++i) {
      mbar_init(info_full(i), 1);
      mbar_init(info_empty(i), C::WARPS);
    }
    *abort_flag = *no_item = *no_tile = 0;
    sstart[0] = a.B;
    sstart[1] = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tmQ);
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
  }
  if (!a.beside) griddep_wait();
  griddep_launch();
  // units before every sequence: each thread adds up a run of sequences, then a scan over the threads
  __shared__ long wsum[C::WARPS + 1];
  const int run = (a.B + C::THREADS - 1) / C::THREADS;
  const int b0 = min(a.B, tid * run), b1 = min(a.B, b0 + run);
  long mine = 0;
  SpSeq s_first{};  // with one sequence a thread, its lengths are read once
  for (int b = b0; b < b1; ++b) {
    const SpSeq s = sp_sequence(a, b, blockIdx.x == 0);
    if (b == b0) s_first = s;
    mine += ss_count(a, s.nq, s.nk).all(a.Hkv);
  }
  long sum = mine;
#pragma unroll
  for (int w = 1; w < 32; w <<= 1) {
    const long v = __shfl_up_sync(0xffffffffu, sum, w);
    if (lane >= w) sum += v;
  }
  if (lane == 31) wsum[warp] = sum;
  __syncthreads();
  long before = sum - mine, total = 0;
#pragma unroll
  for (int w = 0; w <= C::WARPS; ++w) {
    if (w < warp) before += wsum[w];
    total += wsum[w];
  }
  const int cuts = a.split.n > 0 ? sp_pick_cuts(a.split, sp_pick(a.split, total)) : a.cuts;
  const int n = ss_stretches(total, cuts), me = static_cast<int>(blockIdx.x);
  const long lo = me < n ? ss_cut(total, n, me) : 0, hi = me < n ? ss_cut(total, n, me + 1) : 0;
  {
    long at = before;
    for (int b = b0; b < b1; ++b) {
      if (blockIdx.x == 0) a.tile_start[b] = at;
      const SpSeq s = b == b0 ? s_first : sp_sequence(a, b, false);
      const long units = ss_count(a, s.nq, s.nk).all(a.Hkv);
      if (lo >= at && lo < at + units) {
        sstart[0] = b;
        sstart[1] = at;
      }
      at += units;
    }
    if (blockIdx.x == 0 && tid == 0) a.tile_start[a.B] = total;
  }
  __syncthreads();

  if (warp == C::WARPS) {
    if (lane == 0) {
      // ---------------- TMA producer: walks the stretch item by item
      long pos = lo;
      int b = static_cast<int>(sstart[0]);
      long off = lo - sstart[1];
      int g = 0, i = 0;
      bool ok = true;
      const int per = 16 / a.G;
      while (pos < hi && b < a.B && ok) {
        const SpSeq s = sp_sequence(a, b, false);
        const SsCount c = ss_count(a, s.nq, s.nk);
        const long all = c.all(a.Hkv);
        while (off < all && pos < hi) {
          const int units = c.units(), item = static_cast<int>(off / units);
          const int u0 = static_cast<int>(off - (long)item * units);  // units of the item before the stretch
          const int u1 = static_cast<int>(min((long)units, u0 + hi - pos));
          off += u1 - u0;
          pos += u1 - u0;
          SsItem o;
          o.t0 = max(0, u0 - kSsItem);
          o.nt = u1 - kSsItem - o.t0;
          if (o.nt <= 0) continue;  // only units of the item's own cost
          const int rb = item / a.Hkv;
          o.hk = item - rb * a.Hkv;
          o.tok0 = s.q0 + rb * per;
          o.rows = min(per, s.nq - rb * per) * a.G;
          o.nk = s.nk;
          o.rel = s.nk - s.nq + rb * per;
          o.slot = o.nt == c.tiles ? -1 : 2 * static_cast<int>(blockIdx.x) + (o.t0 > 0 ? 0 : 1);
          const int sl = i % C::RING;
          if (!mbar_wait(info_empty(sl), ((i / C::RING) & 1) ^ 1, 660, abort_flag)) { ok = false; break; }
          ring[sl] = o;
          mbar_arrive(info_full(sl));
          ++i;
          for (int j = 0; j < o.nt; ++j, ++g) {
            const int st = g % STAGES;
            if (!mbar_wait(empty(st), ((g / STAGES) & 1) ^ 1, 661, abort_flag)) { ok = false; break; }
            const uint32_t dk = s0 + st * C::STAGE, dv = dk + C::TILE, dq = dv + C::TILE;
            // each of the two groups finds the queries beside its first tile
            mbar_arrive_expect_tx(full(st), 2 * C::TILE + (j < 2 ? per * a.G * D * 2 : 0));
            const int y = static_cast<int>(s.base) + (o.t0 + j) * kSpKeys;
#pragma unroll
            for (int u = 0; u < SUB; ++u) {
              tma_load_2d(dk + u * 8192, &tmK, full(st), o.hk * D + u * 64, y);
              tma_load_2d(dv + u * 8192, &tmV, full(st), o.hk * D + u * 64, y);
              if (j < 2) tma_load_3d(dq + u * 2048, &tmQ, full(st), u * 64, o.hk * a.G, o.tok0);
            }
          }
          if (!ok) break;
        }
        ++b;
        off = 0;
      }
      if (ok) {
        const int sl = i % C::RING;
        if (mbar_wait(info_empty(sl), ((i / C::RING) & 1) ^ 1, 662, abort_flag)) {
          ring[sl].nt = 0;
          mbar_arrive(info_full(sl));
        }
      }
      for (int k = (g > STAGES ? g - STAGES : 0); k < g; ++k)
        mbar_wait(full(k % STAGES), (k / STAGES) & 1, 663, nullptr);
    }
  } else {
    // ---------------- consumers: warp = group (tiles j % 2) x quarter of the tile's keys
    const int grp = warp >> 2, wk = warp & 3;
    auto put = [&](uint32_t base, int sub_bytes, int r, int c) {
      return base + (c >> 3) * sub_bytes + r * 128 + (((c & 7) ^ (r & 7)) << 4);
    };
    int g0 = 0;  // tiles before the item
    for (int i = 0;; ++i) {
      const int sl = i % C::RING;
      if (!mbar_wait(info_full(sl), (i / C::RING) & 1, 664, abort_flag)) *no_item = 1;
      // all consumer warps have read the join of the item before, and they go on or leave together:
      // no_item is written before this barrier only, no_tile before the next one only
      ss_bar();
      if (*no_item) break;
      const SsItem it = ring[sl];
      __syncwarp();
      if (lane == 0) mbar_arrive(info_empty(sl));
      if (it.nt == 0) break;
      const int rl = lane >> 2;  // this thread's rows: rl and rl + 8
      const int lim0 = rl < it.rows ? sp_limit_at(a, it.nk, it.rel + rl / a.G) : 0;
      const int lim1 = rl + 8 < it.rows ? sp_limit_at(a, it.nk, it.rel + (rl + 8) / a.G) : 0;
      const int wmin = __reduce_min_sync(0xffffffffu, min(lim0, lim1));
      float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
      float o[D / 8][4];
#pragma unroll
      for (int d = 0; d < D / 8; ++d) o[d][0] = o[d][1] = o[d][2] = o[d][3] = 0.f;
      uint32_t qf[D / 16][4];
      for (int j = grp; j < it.nt; j += 2) {
        const int g = g0 + j, st = g % STAGES;
        if (!mbar_wait(full(st), (g / STAGES) & 1, 665, abort_flag)) { *no_tile = 1; break; }
        const uint32_t kb = s0 + st * C::STAGE, vb = kb + C::TILE, qb = vb + C::TILE;
        if (j == grp) {
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk)
            ldsm4(put(qb, 2048, lane & 15, 2 * kk + (lane >> 4)), qf[kk][0], qf[kk][1], qf[kk][2], qf[kk][3]);
        }
        // two accumulator pairs halve the dependent chain of the products
        float s[2][4], s2[2][4];
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[n][e] = s2[n][e] = 0.f;
#pragma unroll
        for (int kk = 0; kk < D / 16; kk += 2) {
          uint32_t x0, x1, x2, x3;
          ldsm4(put(kb, 8192, wk * 16 + ((lane >> 4) << 3) + (lane & 7), 2 * kk + ((lane >> 3) & 1)), x0, x1, x2, x3);
          mma_bf16(s[0], qf[kk], x0, x1);
          mma_bf16(s[1], qf[kk], x2, x3);
          ldsm4(put(kb, 8192, wk * 16 + ((lane >> 4) << 3) + (lane & 7), 2 * kk + 2 + ((lane >> 3) & 1)), x0, x1, x2,
                x3);
          mma_bf16(s2[0], qf[kk + 1], x0, x1);
          mma_bf16(s2[1], qf[kk + 1], x2, x3);
        }
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[n][e] += s2[n][e];
        const int k0 = (it.t0 + j) * kSpKeys + wk * 16, c0 = k0 + 2 * (lane & 3);
        if (wmin < k0 + 16) {
#pragma unroll
          for (int n = 0; n < 2; ++n) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              if (c0 + 8 * n + e >= lim0) s[n][e] = -INFINITY;
              if (c0 + 8 * n + e >= lim1) s[n][2 + e] = -INFINITY;
            }
          }
        }
        float x0 = fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[1][0], s[1][1]));
        float x1 = fmaxf(fmaxf(s[0][2], s[0][3]), fmaxf(s[1][2], s[1][3]));
#pragma unroll
        for (int w = 1; w <= 2; w <<= 1) {
          x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, w));
          x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, w));
        }
        const float n0 = fmaxf(m0, x0 * a.scale_log2), n1 = fmaxf(m1, x1 * a.scale_log2);
        const float r0 = n0 == -INFINITY ? 0.f : n0, r1 = n1 == -INFINITY ? 0.f : n1;
        const float e0 = m0 == n0 ? 1.f : ex2_fast(m0 - r0), e1 = m1 == n1 ? 1.f : ex2_fast(m1 - r1);
        m0 = n0, m1 = n1;
#pragma unroll
        for (int n = 0; n < 2; ++n) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            s[n][e] = ex2_fast(fmaf(s[n][e], a.scale_log2, -r0));
            s[n][2 + e] = ex2_fast(fmaf(s[n][2 + e], a.scale_log2, -r1));
          }
        }
        l0 = l0 * e0 + ((s[0][0] + s[0][1]) + (s[1][0] + s[1][1]));
        l1 = l1 * e1 + ((s[0][2] + s[0][3]) + (s[1][2] + s[1][3]));
        if (__any_sync(0xffffffffu, e0 != 1.f || e1 != 1.f)) {
#pragma unroll
          for (int d = 0; d < D / 8; ++d) o[d][0] *= e0, o[d][1] *= e0, o[d][2] *= e1, o[d][3] *= e1;
        }
        // P is rounded to bf16 for the product (at most 2^-8 relative, averaged over the keys), its sum is not
        const uint32_t pf[4] = {pack_bf16x2(s[0][0], s[0][1]), pack_bf16x2(s[0][2], s[0][3]),
                                pack_bf16x2(s[1][0], s[1][1]), pack_bf16x2(s[1][2], s[1][3])};
        // rows behind the sequence may hold anything, and a weight of zero does not stop a NaN
        const bool tail = it.nk < k0 + 16;
        uint32_t z0 = 0xffffffffu, z1 = 0xffffffffu;
        if (tail) {
          z0 = (c0 < it.nk ? 0xffffu : 0u) | (c0 + 1 < it.nk ? 0xffff0000u : 0u);
          z1 = (c0 + 8 < it.nk ? 0xffffu : 0u) | (c0 + 9 < it.nk ? 0xffff0000u : 0u);
        }
#pragma unroll
        for (int db = 0; db < D / 16; ++db) {
          uint32_t y0, y1, y2, y3;
          ldsm4_t(put(vb, 8192, wk * 16 + (lane & 15), 2 * db + (lane >> 4)), y0, y1, y2, y3);
          if (tail) y0 &= z0, y2 &= z0, y1 &= z1, y3 &= z1;
          mma_bf16(o[2 * db], pf, y0, y1);
          mma_bf16(o[2 * db + 1], pf, y2, y3);
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(empty(st));
      }
      g0 += it.nt;
#pragma unroll
      for (int w = 1; w <= 2; w <<= 1) {
        l0 += __shfl_xor_sync(0xffffffffu, l0, w);
        l1 += __shfl_xor_sync(0xffffffffu, l1, w);
      }
      if ((lane & 3) == 0) {
        sml[warp * 16 + rl] = make_float2(m0, l0);
        sml[warp * 16 + rl + 8] = make_float2(m1, l1);
      }
      float* mine_o = so + (warp * 16 + rl) * D + 2 * (lane & 3);
#pragma unroll
      for (int d = 0; d < D / 8; ++d) {
        if (rl < it.rows) *reinterpret_cast<float2*>(mine_o + 8 * d) = make_float2(o[d][0], o[d][1]);
        if (rl + 8 < it.rows) *reinterpret_cast<float2*>(mine_o + 8 * D + 8 * d) = make_float2(o[d][2], o[d][3]);
      }
      ss_bar();
      if (*no_tile) break;
      for (int e = tid; e < it.rows * (D / 4); e += 32 * C::WARPS) {
        const int r = e / (D / 4), d = 4 * (e % (D / 4));
        float m = -INFINITY;
#pragma unroll
        for (int w = 0; w < C::WARPS; ++w) m = fmaxf(m, sml[w * 16 + r].x);
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        float l = 0.f;
#pragma unroll
        for (int w = 0; w < C::WARPS; ++w) {
          const float2 ml = sml[w * 16 + r];
          // a share without a visible key has maximum -inf and weight 0 (its sum may be NaN: kept)
          const float f = m == -INFINITY ? 1.f : ex2_fast(ml.x - m);
          l = fmaf(ml.y, f, l);
          const float4 v = *reinterpret_cast<const float4*>(so + (w * 16 + r) * D + d);
          acc.x = fmaf(v.x, f, acc.x);
          acc.y = fmaf(v.y, f, acc.y);
          acc.z = fmaf(v.z, f, acc.z);
          acc.w = fmaf(v.w, f, acc.w);
        }
        const int tok = r / a.G;
        const long at = it.slot < 0 ? ((long)a.prefix_parts * a.N + it.tok0 + tok) * a.H + it.hk * a.G + (r - tok * a.G)
                                    : 0;
        float2* ml_out = it.slot < 0 ? a.part_ml + at : a.cut_ml + it.slot * 16 + r;
        float* o_out = it.slot < 0 ? a.part_o + at * D : a.cut_o + ((long)it.slot * 16 + r) * D;
        if (d == 0) *ml_out = make_float2(m, l);
        *reinterpret_cast<float4*>(o_out + d) = acc;
      }
    }
  }
  __syncwarp();
  if (a.beside) griddep_wait();
}

}  // namespace fcv
