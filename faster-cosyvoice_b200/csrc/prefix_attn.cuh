// prefix_attn.cuh -- attention of a ragged batch whose sequences share one prefix.
//
// Sequence b has query rows [cu[b], cu[b+1]) (nq of them, H heads of D values) and nk own key rows
// kv_base[b] .. kv_base[b] + nk; all sequences see the same P prefix keys before them.  Key heads
// are shared by G = H / Hkv query heads.  For query i of sequence b:
//     o = softmax(scale q [Kp ; Kb]^T) [Vp ; Vb]
// over the whole prefix and the own keys j with (P + j) / chunk <= (P + nk - nq + i) / chunk
// (integer division; chunk 0: every own key).  A row that sees no key is zero.
//
// Query rows are stacked over the heads of a key head: stacked row R = token * G + g.  The prefix
// belongs to no sequence, so its products run over stacked rows of the whole batch -- each prefix
// key is read once for 64 rows, not once for every sequence -- and the own keys run per sequence.
// Each piece of keys leaves a running maximum, sum and unnormalised output in float32; a second
// kernel joins the pieces of a row.
#pragma once

#include <type_traits>

#include "fcv_common.cuh"

namespace fcv {

struct SpArgs {
  const void* q;
  long q_stride;  // elements between query rows; heads are D apart
  const void* k;
  const void* v;
  long k_stride, v_stride;
  long kv_rows;  // rows of k and v
  const void* pk;
  const void* pv;
  long pk_stride, pv_stride;
  int P;
  const int32_t* cu;
  const int32_t* kv_base;  // null: cu
  const int32_t* kv_lens;  // null: cu differences
  int B, N, H, Hkv, G, chunk;
  float scale_log2;  // softmax scale in log2 units
  void* out;
  long out_stride;
  float* part_o;   // (parts, N, H, D)
  float2* part_ml; // (parts, N, H): maximum (log2 units) and sum
  int prefix_parts, own_parts;  // one part in all: written to out, nothing to join
  int prefix_items, own_rows;   // blocks of the prefix; blockIdx.y slots of a sequence's row blocks
};

constexpr int kSpKeys = 64;  // keys of a tile

struct SpSeq {
  int q0, nq, nk;
  long base;
};
// The device arrays of a sequence, checked: rows outside the buffers are never touched.
__device__ __forceinline__ SpSeq sp_sequence(const SpArgs& a, int b) {
  SpSeq s;
  const int c0 = a.cu[b], c1 = a.cu[b + 1];
  s.q0 = c0;
  s.nq = c1 - c0;
  if (c0 < 0 || c1 < c0 || c1 > a.N) {
    if (threadIdx.x == 0) record_error(611);
    s.q0 = 0;
    s.nq = 0;
  }
  s.base = a.kv_base ? a.kv_base[b] : s.q0;
  s.nk = a.kv_lens ? a.kv_lens[b] : s.nq;
  if (s.nk < 0 || s.base < 0 || s.base + s.nk > a.kv_rows) {
    if (s.nk != 0 && threadIdx.x == 0) record_error(612);
    s.base = 0;
    s.nk = 0;
  }
  return s;
}
// Own keys that query i of the sequence sees.
__device__ __forceinline__ int sp_limit(const SpArgs& a, const SpSeq& s, int i) {
  if (a.chunk <= 0) return s.nk;
  const long at = (long)a.P + s.nk - s.nq + i;
  if (at < 0) return 0;
  const long lim = (at / a.chunk + 1) * a.chunk - a.P;
  return lim < 0 ? 0 : (lim < s.nk ? static_cast<int>(lim) : s.nk);
}
// Tiles [t0, t1) of piece `part` out of at most `parts` over `tiles` tiles: pieces of equal size,
// none shorter than four tiles unless it is the last.
__device__ __forceinline__ void sp_piece(int tiles, int parts, int part, int& t0, int& t1) {
  const int n = max(1, min(parts, (tiles + 3) / 4));
  const int each = (tiles + n - 1) / n;
  t0 = min(tiles, part * each);
  t1 = part < n ? min(tiles, t0 + each) : t0;
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool valid) {
  const int n = valid ? 16 : 0;  // 0: the 16 bytes are zeroed, the source is not read
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t& a, uint32_t& b, uint32_t& c, uint32_t& d) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(a), "=r"(b), "=r"(c), "=r"(d)
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t& a, uint32_t& b, uint32_t& c, uint32_t& d) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(a), "=r"(b), "=r"(c), "=r"(d)
               : "r"(addr)
               : "memory");
}
// D (16 x 8, f32) += A (16 x 16, bf16, rows) B (16 x 8, bf16, columns)
__device__ __forceinline__ void mma_bf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Where the results of stacked row R of key head hk go (part p of a row, or the row itself).
struct SpRow {
  long token;
  int head;
};
__device__ __forceinline__ SpRow sp_row(const SpArgs& a, int hk, long R) {
  SpRow r;
  r.token = R / a.G;
  r.head = hk * a.G + static_cast<int>(R - r.token * a.G);
  return r;
}

// ------------------------------------------------------------------ bf16
template <int D>
struct SpMma {
  static constexpr int kStages = D == 64 ? 4 : 3;
  static constexpr int kTile = kSpKeys * D * 2;
  static constexpr int kQ = 64 * D * 2;
  static constexpr int kSmem = kQ + kStages * 2 * kTile;
};

// One piece: stacked rows [R0, R0 + rows) of key head hk (rows <= 16 WM) against key rows
// [0, kend) of K / V, tiles [t0, t1).  4 warps: WM of them along the rows (16 each), 4 / WM along
// the keys of a tile; for WM < 4 the warps' partial results are joined in shared memory.
//   limits: row r of the block sees keys [0, lim(r)).
// K, V tiles come by 16-byte asynchronous copies into a ring; a row of a tile is D / 8 chunks of
// 16 bytes, chunk c of row r at c ^ (r % 8), which keeps ldmatrix free of bank conflicts.
// Rows past kend are zero in shared memory, so stale values behind a sequence never reach a product.
template <int D, int WM, typename Limit>
__device__ __forceinline__ void sp_mma_piece(const SpArgs& a, uint8_t* smem, const bf16* K, const bf16* V,
                                             long k_stride, long v_stride, int hk, long R0, int rows, int kend,
                                             int t0, int t1, int part, Limit limit) {
  using C = SpMma<D>;
  constexpr int WK = 4 / WM;
  constexpr int KW = kSpKeys / WK;  // keys of a tile that a warp takes
  constexpr int CH = D / 8;         // 16-byte chunks of a row
  constexpr int STAGES = C::kStages;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int wm = warp % WM, wk = warp / WM;
  const uint32_t s0 = smem_u32(smem), sQ = s0, sKV = s0 + C::kQ;
  const bool direct = a.prefix_parts + a.own_parts == 1;

  auto put = [&](uint32_t base, int r, int c) { return base + r * (D * 2) + ((c ^ (r & 7)) << 4); };
  __syncthreads();  // an earlier piece of this block has left the buffers
  for (int i = tid; i < 16 * WM * CH; i += 128) {
    const int r = i / CH, c = i % CH;
    const bool ok = r < rows;
    const SpRow x = sp_row(a, hk, R0 + (ok ? r : 0));
    cp_async16(put(sQ, r, c), static_cast<const bf16*>(a.q) + x.token * a.q_stride + (long)x.head * D + 8 * c, ok);
  }
  auto load = [&](int t) {
    const uint32_t kb = sKV + ((t - t0) % STAGES) * 2 * C::kTile, vb = kb + C::kTile;
#pragma unroll
    for (int i = tid; i < kSpKeys * CH; i += 128) {
      const int r = i / CH, c = i % CH;
      const long key = (long)t * kSpKeys + r;
      const bool ok = key < kend;
      const long at = ok ? key : 0;
      cp_async16(put(kb, r, c), K + at * k_stride + 8 * c, ok);
      cp_async16(put(vb, r, c), V + at * v_stride + 8 * c, ok);
    }
  };
#pragma unroll
  for (int i = 0; i < STAGES - 1; ++i) {
    if (t0 + i < t1) load(t0 + i);
    cp_async_commit();
  }

  const int rl = 16 * wm + (lane >> 2);  // this thread's rows of the block: rl and rl + 8
  const int lim0 = rl < rows ? limit(rl) : 0, lim1 = rl + 8 < rows ? limit(rl + 8) : 0;
  const int wmin = __reduce_min_sync(0xffffffffu, min(lim0, lim1));
  float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
  float o[D / 8][4];
#pragma unroll
  for (int i = 0; i < D / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
  uint32_t qf[D / 16][4];

  for (int t = t0; t < t1; ++t) {
    cp_async_wait<STAGES - 2>();
    __syncthreads();
    if (t + STAGES - 1 < t1) load(t + STAGES - 1);
    cp_async_commit();
    if (t == t0) {
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk)
        ldsm4(put(sQ, 16 * wm + (lane & 15), 2 * kk + (lane >> 4)), qf[kk][0], qf[kk][1], qf[kk][2], qf[kk][3]);
    }
    const uint32_t kb = sKV + ((t - t0) % STAGES) * 2 * C::kTile, vb = kb + C::kTile;
    float s[KW / 8][4];
#pragma unroll
    for (int i = 0; i < KW / 8; ++i) s[i][0] = s[i][1] = s[i][2] = s[i][3] = 0.f;
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) {
#pragma unroll
      for (int nb = 0; nb < KW / 16; ++nb) {
        uint32_t b0, b1, b2, b3;
        ldsm4(put(kb, wk * KW + nb * 16 + ((lane >> 4) << 3) + (lane & 7), 2 * kk + ((lane >> 3) & 1)), b0, b1, b2,
              b3);
        mma_bf16(s[2 * nb], qf[kk], b0, b1);
        mma_bf16(s[2 * nb + 1], qf[kk], b2, b3);
      }
    }
    const int k0 = t * kSpKeys + wk * KW;
    if (wmin < k0 + KW) {  // some row of the warp stops inside this warp's keys
      const int c0 = k0 + 2 * (lane & 3);
#pragma unroll
      for (int i = 0; i < KW / 8; ++i) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          if (c0 + 8 * i + j >= lim0) s[i][j] = -INFINITY;
          if (c0 + 8 * i + j >= lim1) s[i][2 + j] = -INFINITY;
        }
      }
    }
    float x0 = -INFINITY, x1 = -INFINITY;
#pragma unroll
    for (int i = 0; i < KW / 8; ++i) {
      x0 = fmaxf(x0, fmaxf(s[i][0], s[i][1]));
      x1 = fmaxf(x1, fmaxf(s[i][2], s[i][3]));
    }
#pragma unroll
    for (int w = 1; w <= 2; w <<= 1) {
      x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, w));
      x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, w));
    }
    const float n0 = fmaxf(m0, x0 * a.scale_log2), n1 = fmaxf(m1, x1 * a.scale_log2);
    // a row without a visible key so far keeps the reference 0: its exponentials are all 2^-inf = 0
    const float r0 = n0 == -INFINITY ? 0.f : n0, r1 = n1 == -INFINITY ? 0.f : n1;
    const float e0 = ex2_fast(m0 - r0), e1 = ex2_fast(m1 - r1);
    m0 = n0, m1 = n1;
    float y0 = 0.f, y1 = 0.f;
#pragma unroll
    for (int i = 0; i < KW / 8; ++i) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        s[i][j] = ex2_fast(fmaf(s[i][j], a.scale_log2, -r0));
        s[i][2 + j] = ex2_fast(fmaf(s[i][2 + j], a.scale_log2, -r1));
        y0 += s[i][j];
        y1 += s[i][2 + j];
      }
    }
    l0 = l0 * e0 + y0;
    l1 = l1 * e1 + y1;
#pragma unroll
    for (int i = 0; i < D / 8; ++i) o[i][0] *= e0, o[i][1] *= e0, o[i][2] *= e1, o[i][3] *= e1;
    // P is rounded to bf16 for the product (half a step, 2^-9 relative, averaged over the keys);
    // its sum stays in float32
#pragma unroll
    for (int kk = 0; kk < KW / 16; ++kk) {
      const uint32_t pf[4] = {pack_bf16x2(s[2 * kk][0], s[2 * kk][1]), pack_bf16x2(s[2 * kk][2], s[2 * kk][3]),
                              pack_bf16x2(s[2 * kk + 1][0], s[2 * kk + 1][1]),
                              pack_bf16x2(s[2 * kk + 1][2], s[2 * kk + 1][3])};
#pragma unroll
      for (int db = 0; db < D / 16; ++db) {
        uint32_t b0, b1, b2, b3;
        ldsm4_t(put(vb, wk * KW + kk * 16 + (lane & 15), 2 * db + (lane >> 4)), b0, b1, b2, b3);
        mma_bf16(o[2 * db], pf, b0, b1);
        mma_bf16(o[2 * db + 1], pf, b2, b3);
      }
    }
  }
#pragma unroll
  for (int w = 1; w <= 2; w <<= 1) {
    l0 += __shfl_xor_sync(0xffffffffu, l0, w);
    l1 += __shfl_xor_sync(0xffffffffu, l1, w);
  }
  cp_async_wait<0>();
  if constexpr (WK > 1) {
    // join the key shares of a row group: maxima first, then each warp adds its scaled share in turn
    float* sml = reinterpret_cast<float*>(smem);          // [warp][16] maxima
    float* ssum = sml + 64;                               // [row of the block] sums
    float* so = reinterpret_cast<float*>(smem + C::kQ);   // [row of the block][D]
    __syncthreads();
    if ((lane & 3) == 0) {
      sml[warp * 16 + (lane >> 2)] = m0;
      sml[warp * 16 + (lane >> 2) + 8] = m1;
    }
    __syncthreads();
    float g0 = -INFINITY, g1 = -INFINITY;
#pragma unroll
    for (int w = 0; w < WK; ++w) {
      g0 = fmaxf(g0, sml[(w * WM + wm) * 16 + (lane >> 2)]);
      g1 = fmaxf(g1, sml[(w * WM + wm) * 16 + (lane >> 2) + 8]);
    }
    const float f0 = g0 == -INFINITY ? 0.f : ex2_fast(m0 - g0), f1 = g1 == -INFINITY ? 0.f : ex2_fast(m1 - g1);
    m0 = g0, m1 = g1;
    l0 *= f0, l1 *= f1;
#pragma unroll
    for (int i = 0; i < D / 8; ++i) o[i][0] *= f0, o[i][1] *= f0, o[i][2] *= f1, o[i][3] *= f1;
#pragma unroll 1
    for (int w = WK - 1; w >= 0; --w) {  // a fixed order: the last share writes, the others add, the first keeps
      if (wk == w) {
#pragma unroll
        for (int i = 0; i < D / 8; ++i) {
          float2* p0 = reinterpret_cast<float2*>(so + (long)rl * D + 8 * i + 2 * (lane & 3));
          float2* p1 = reinterpret_cast<float2*>(so + (long)(rl + 8) * D + 8 * i + 2 * (lane & 3));
          if (w != WK - 1) {
            const float2 u0 = *p0, u1 = *p1;
            o[i][0] += u0.x, o[i][1] += u0.y, o[i][2] += u1.x, o[i][3] += u1.y;
          }
          if (w != 0) {
            *p0 = make_float2(o[i][0], o[i][1]);
            *p1 = make_float2(o[i][2], o[i][3]);
          }
        }
        if (w != WK - 1) l0 += ssum[rl], l1 += ssum[rl + 8];
        if (w != 0) {
          __syncwarp();
          if ((lane & 3) == 0) ssum[rl] = l0, ssum[rl + 8] = l1;
        }
      }
      __syncthreads();
    }
  }
  if (wk != 0) return;
  auto emit = [&](int r, float m, float l, int half) {
    if (r >= rows) return;
    const SpRow x = sp_row(a, hk, R0 + r);
    if (direct) {
      const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
      bf16* dst = static_cast<bf16*>(a.out) + x.token * a.out_stride + (long)x.head * D + 2 * (lane & 3);
#pragma unroll
      for (int i = 0; i < D / 8; ++i)
        *reinterpret_cast<uint32_t*>(dst + 8 * i) = pack_bf16x2(o[i][2 * half] * inv, o[i][2 * half + 1] * inv);
    } else {
      const long at = ((long)part * a.N + x.token) * a.H + x.head;
      if ((lane & 3) == 0) a.part_ml[at] = make_float2(m, l);
      if (m == -INFINITY && l == 0.f) return;  // saw no key: joined as nothing
      float* dst = a.part_o + at * D + 2 * (lane & 3);
#pragma unroll
      for (int i = 0; i < D / 8; ++i)
        *reinterpret_cast<float2*>(dst + 8 * i) = make_float2(o[i][2 * half], o[i][2 * half + 1]);
    }
  };
  emit(rl, m0, l0, 0);
  emit(rl + 8, m1, l1, 1);
}

// ------------------------------------------------------------------ fp32 (CUDA cores)
// 256 threads, 16 x 16: thread (ty, tx) has rows RPT ty .. and, of S, keys tx + 16 j, of O,
// columns 4 tx + 64 c.  Rows in shared memory are padded by 4 floats, so the 16-byte reads of 8
// neighbouring rows fall into different banks.
template <int D, int RPT>
struct SpF32 {
  static constexpr int kRows = 16 * RPT;
  static constexpr int kLd = D + 4;
  static constexpr int kStages = 2;
  static constexpr int kSmem = 4 * (kRows * kLd + kStages * 2 * kSpKeys * kLd + kRows * (kSpKeys + 4));
};
template <int D, int RPT, typename Limit>
__device__ __forceinline__ void sp_f32_piece(const SpArgs& a, uint8_t* smem, const float* K, const float* V,
                                             long k_stride, long v_stride, int hk, long R0, int rows, int kend,
                                             int t0, int t1, int part, Limit limit) {
  using C = SpF32<D, RPT>;
  constexpr int LD = C::kLd, CH = D / 4, PLD = kSpKeys + 4;
  float* sQ = reinterpret_cast<float*>(smem);
  float* sKV = sQ + C::kRows * LD;
  float* sP = sKV + C::kStages * 2 * kSpKeys * LD;
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
  const bool direct = a.prefix_parts + a.own_parts == 1;
  __syncthreads();
  for (int i = tid; i < C::kRows * CH; i += 256) {
    const int r = i / CH, c = i % CH;
    const bool ok = r < rows;
    const SpRow x = sp_row(a, hk, R0 + (ok ? r : 0));
    cp_async16(smem_u32(sQ + r * LD + 4 * c),
               static_cast<const float*>(a.q) + x.token * a.q_stride + (long)x.head * D + 4 * c, ok);
  }
  auto load = [&](int t) {
    float* kb = sKV + ((t - t0) & 1) * 2 * kSpKeys * LD;
    float* vb = kb + kSpKeys * LD;
    for (int i = tid; i < kSpKeys * CH; i += 256) {
      const int r = i / CH, c = i % CH;
      const long key = (long)t * kSpKeys + r;
      const bool ok = key < kend;
      const long at = ok ? key : 0;
      cp_async16(smem_u32(kb + r * LD + 4 * c), K + at * k_stride + 4 * c, ok);
      cp_async16(smem_u32(vb + r * LD + 4 * c), V + at * v_stride + 4 * c, ok);
    }
  };
  if (t0 < t1) load(t0);
  cp_async_commit();
  int lim[RPT];
  float m[RPT], l[RPT];
  float o[RPT][D / 16];
#pragma unroll
  for (int i = 0; i < RPT; ++i) {
    lim[i] = RPT * ty + i < rows ? limit(RPT * ty + i) : 0;
    m[i] = -INFINITY;
    l[i] = 0.f;
#pragma unroll
    for (int d = 0; d < D / 16; ++d) o[i][d] = 0.f;
  }
  for (int t = t0; t < t1; ++t) {
    cp_async_wait<0>();
    __syncthreads();
    if (t + 1 < t1) load(t + 1);
    cp_async_commit();
    const float* kb = sKV + ((t - t0) & 1) * 2 * kSpKeys * LD;
    const float* vb = kb + kSpKeys * LD;
    float s[RPT][4];
#pragma unroll
    for (int i = 0; i < RPT; ++i) s[i][0] = s[i][1] = s[i][2] = s[i][3] = 0.f;
#pragma unroll 4
    for (int d = 0; d < D; d += 4) {
      float4 kv[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) kv[j] = *reinterpret_cast<const float4*>(kb + (tx + 16 * j) * LD + d);
#pragma unroll
      for (int i = 0; i < RPT; ++i) {
        const float4 qv = *reinterpret_cast<const float4*>(sQ + (RPT * ty + i) * LD + d);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          s[i][j] = fmaf(qv.x, kv[j].x, s[i][j]);
          s[i][j] = fmaf(qv.y, kv[j].y, s[i][j]);
          s[i][j] = fmaf(qv.z, kv[j].z, s[i][j]);
          s[i][j] = fmaf(qv.w, kv[j].w, s[i][j]);
        }
      }
    }
    const int k0 = t * kSpKeys + tx;
#pragma unroll
    for (int i = 0; i < RPT; ++i) {
      float x = -INFINITY;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        s[i][j] = k0 + 16 * j < lim[i] ? s[i][j] * a.scale_log2 : -INFINITY;
        x = fmaxf(x, s[i][j]);
      }
#pragma unroll
      for (int w = 1; w < 16; w <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, w));
      const float mn = fmaxf(m[i], x), ref = mn == -INFINITY ? 0.f : mn;
      const float e = exp2f(m[i] - ref);
      m[i] = mn;
      float y = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float p = exp2f(s[i][j] - ref);
        y += p;
        sP[(RPT * ty + i) * PLD + tx + 16 * j] = p;
      }
      l[i] = l[i] * e + y;
#pragma unroll
      for (int d = 0; d < D / 16; ++d) o[i][d] *= e;
    }
    __syncwarp();  // a row's 16 threads are half of one warp
#pragma unroll 2
    for (int k = 0; k < kSpKeys; k += 4) {
      float4 p[RPT];
#pragma unroll
      for (int i = 0; i < RPT; ++i) p[i] = *reinterpret_cast<const float4*>(sP + (RPT * ty + i) * PLD + k);
#pragma unroll
      for (int u = 0; u < 4; ++u) {
#pragma unroll
        for (int c = 0; c < D / 64; ++c) {
          const float4 vv = *reinterpret_cast<const float4*>(vb + (k + u) * LD + 64 * c + 4 * tx);
#pragma unroll
          for (int i = 0; i < RPT; ++i) {
            const float pu = u == 0 ? p[i].x : u == 1 ? p[i].y : u == 2 ? p[i].z : p[i].w;
            o[i][4 * c] = fmaf(pu, vv.x, o[i][4 * c]);
            o[i][4 * c + 1] = fmaf(pu, vv.y, o[i][4 * c + 1]);
            o[i][4 * c + 2] = fmaf(pu, vv.z, o[i][4 * c + 2]);
            o[i][4 * c + 3] = fmaf(pu, vv.w, o[i][4 * c + 3]);
          }
        }
      }
    }
    __syncwarp();
  }
  cp_async_wait<0>();
#pragma unroll
  for (int i = 0; i < RPT; ++i) {
#pragma unroll
    for (int w = 1; w < 16; w <<= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], w);
    const int r = RPT * ty + i;
    if (r >= rows) continue;
    const SpRow x = sp_row(a, hk, R0 + r);
    if (direct) {
      const float inv = l[i] > 0.f || l[i] != l[i] ? 1.f / l[i] : 0.f;
      float* dst = static_cast<float*>(a.out) + x.token * a.out_stride + (long)x.head * D + 4 * tx;
#pragma unroll
      for (int c = 0; c < D / 64; ++c)
        *reinterpret_cast<float4*>(dst + 64 * c) =
            make_float4(o[i][4 * c] * inv, o[i][4 * c + 1] * inv, o[i][4 * c + 2] * inv, o[i][4 * c + 3] * inv);
    } else {
      const long at = ((long)part * a.N + x.token) * a.H + x.head;
      if (tx == 0) a.part_ml[at] = make_float2(m[i], l[i]);
      if (m[i] == -INFINITY && l[i] == 0.f) continue;
      float* dst = a.part_o + at * D + 4 * tx;
#pragma unroll
      for (int c = 0; c < D / 64; ++c)
        *reinterpret_cast<float4*>(dst + 64 * c) =
            make_float4(o[i][4 * c], o[i][4 * c + 1], o[i][4 * c + 2], o[i][4 * c + 3]);
    }
  }
}

// ------------------------------------------------------------------ the pieces of a call
// Blocks [0, prefix_items): (row block, key head, part) of the prefix over the stacked rows of the
// batch.  The others: (sequence, key head, part) of the own keys, blockIdx.y striding over the row
// blocks of the sequence.  RP / RO: rows of a block of the prefix / of a sequence; they set the
// shape of the block (see the piece functions).
template <typename T, int D, int RP, int RO>
__global__ void __launch_bounds__(sizeof(T) == 2 ? 128 : 256) sp_pieces_kernel(const SpArgs a) {
  griddep_wait();
  griddep_launch();
  extern __shared__ __align__(128) uint8_t smem[];
  auto piece = [&](auto rows_c, const void* K, const void* V, long ks, long vs, int hk, long R0, int rows, int kend,
                   int t0, int t1, int part, auto limit) {
    constexpr int R = decltype(rows_c)::value;
    const T* k = static_cast<const T*>(K) + (long)hk * D;
    const T* v = static_cast<const T*>(V) + (long)hk * D;
    if constexpr (sizeof(T) == 2)
      sp_mma_piece<D, R / 16>(a, smem, k, v, ks, vs, hk, R0, rows, kend, t0, t1, part, limit);
    else
      sp_f32_piece<D, R / 16>(a, smem, k, v, ks, vs, hk, R0, rows, kend, t0, t1, part, limit);
  };
  int it = blockIdx.x;
  if (it < a.prefix_items) {
    if (blockIdx.y != 0) return;
    const int part = it % a.prefix_parts;
    it /= a.prefix_parts;
    const int hk = it % a.Hkv;
    const long R0 = (long)(it / a.Hkv) * RP;
    const long first = (long)max(0, min(a.N, a.cu[0])) * a.G, end = (long)max(0, min(a.N, a.cu[a.B])) * a.G;
    const long r0 = R0 > first ? R0 : first;
    const long r1 = min(R0 + RP, end);
    if (r0 >= r1) return;
    int t0, t1;
    sp_piece((a.P + kSpKeys - 1) / kSpKeys, a.prefix_parts, part, t0, t1);
    const int P = a.P;
    piece(std::integral_constant<int, RP>(), a.pk, a.pv, a.pk_stride, a.pv_stride, hk, r0, static_cast<int>(r1 - r0),
          P, t0, t1, part, [P](int) { return P; });
    return;
  }
  it -= a.prefix_items;
  const int part = it % a.own_parts;
  it /= a.own_parts;
  const int hk = it % a.Hkv, b = it / a.Hkv;
  const SpSeq s = sp_sequence(a, b);
  const long nrows = (long)s.nq * a.G;
  for (long r = (long)blockIdx.y * RO; r < nrows; r += (long)gridDim.y * RO) {
    const int rows = static_cast<int>(min((long)RO, nrows - r));
    const int seen = sp_limit(a, s, static_cast<int>((r + rows - 1) / a.G));  // limits grow along the rows
    int t0, t1;
    sp_piece((seen + kSpKeys - 1) / kSpKeys, a.own_parts, part, t0, t1);
    piece(std::integral_constant<int, RO>(), static_cast<const T*>(a.k) + s.base * a.k_stride,
          static_cast<const T*>(a.v) + s.base * a.v_stride, a.k_stride, a.v_stride, hk, (long)s.q0 * a.G + r, rows,
          s.nk, t0, t1, a.prefix_parts + part,
          [&](int i) { return sp_limit(a, s, static_cast<int>((r + i) / a.G)); });
  }
}

// Joins the parts of a row: one warp per (token, head).
template <typename T, int D>
__global__ void __launch_bounds__(256) sp_join_kernel(const SpArgs a) {
  griddep_wait();
  griddep_launch();
  const int lane = threadIdx.x & 31;
  const long w = (long)blockIdx.x * 8 + (threadIdx.x >> 5);
  const long token = w / a.H;
  if (token >= a.N || token < a.cu[0] || token >= a.cu[a.B]) return;  // rows behind the last sequence stay
  const int parts = a.prefix_parts + a.own_parts;
  const long step = (long)a.N * a.H;
  float m = -INFINITY;
  for (int p = 0; p < parts; ++p) m = fmaxf(m, a.part_ml[p * step + w].x);
  constexpr int V = D / 32;
  float acc[V];
#pragma unroll
  for (int i = 0; i < V; ++i) acc[i] = 0.f;
  float l = 0.f;
  for (int p = 0; p < parts; ++p) {
    const float2 ml = a.part_ml[p * step + w];
    if (ml.x == -INFINITY && ml.y == 0.f) continue;
    const float f = exp2f(ml.x - m);
    l = fmaf(ml.y, f, l);
    const float* src = a.part_o + (p * step + w) * D + V * lane;
#pragma unroll
    for (int i = 0; i < V; ++i) acc[i] = fmaf(src[i], f, acc[i]);
  }
  const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
  T* dst = static_cast<T*>(a.out) + token * a.out_stride + (w - token * a.H) * D + V * lane;
#pragma unroll
  for (int i = 0; i < V; ++i) dst[i] = from_f<T>(acc[i] * inv);
}

}  // namespace fcv
