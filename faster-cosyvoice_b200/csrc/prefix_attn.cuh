// prefix_attn.cuh -- attention of a ragged batch whose sequences share one prefix.
//
// Sequence b has query rows [cu[b], cu[b+1]) (nq of them, H heads of D values) and nk own key rows
// kv_base[b] .. kv_base[b] + nk; all sequences see the same P prefix keys before them.  Key heads
// are shared by G = H / Hkv query heads.  For query i of sequence b:
//     o = softmax(scale q [Kp ; Kb]^T) [Vp ; Vb]
// over the whole prefix and the own keys j with (P + j) / chunk <= (P + nk - nq + i) / chunk
// (integer division; chunk 0: every own key).  A row that sees no key is zero.
//
// Query rows are stacked over the heads of a key head: stacked row R = token * G + g.  Cut into parts,
// the prefix, which belongs to no sequence, takes stacked rows of the whole batch -- each of its keys
// is read once for 64 rows or more, not once for every sequence -- and the own keys run per sequence.
// Each piece of keys leaves a running maximum, sum and unnormalised output in float32; a second
// kernel joins the pieces of a row.  Whole, a block takes rows of one sequence through the prefix and
// its own keys in one go, so every sequence reads the prefix again and nothing is joined; short
// prefixes and long queries are faster that way.
//
// This file has the kernel for few rows in bf16 (mma.sync: 16 to 64 rows to a block, bound by the
// latency of a key tile, 0.43 us for 16 rows of 64 values, 0.74 us of 128) and for all of float32 (CUDA
// cores, bound by the FMA pipe: 354 us for 8 documents of 243 to 600 rows behind 250 keys, 16 heads of
// 64, 30 TFLOP/s), and the join.  prefix_fa.cuh has the tensor-core kernel for many rows,
// prefix_stream.cuh the one for the own keys of decode steps.
#pragma once

#include <type_traits>

#include "fcv_common.cuh"

namespace fcv {

// How the SMs are shared between the prefix parts (tensor-core kernel) and the own keys
// (sp_stream_kernel) of a decode step: the choices that the host worked out, each with the blocks and
// parts of the former and its time.  The own keys are known on the device only, so each kernel picks
// the same choice from their number (sp_pick).
constexpr int kSplits = 12;
struct SpSplit {
  int n;                 // 0: prefix_parts and cuts are fixed
  int sms;
  int ctas[kSplits], parts[kSplits];
  float fa_us[kSplits];  // time of the prefix parts
  float own_us[kSplits]; // time of a unit of own keys beside them (0: no SM is left, they come after)
  float unit_us;         // a unit of own keys on one SM,
  float floor_us;        // and on the whole GPU (memory bandwidth)
};

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
  int prefix_parts, own_parts;
  int prefix_items;  // blocks of the prefix
  int own_rows;      // blockIdx.y slots of a sequence's row blocks
  int whole;         // a sequence's rows take the prefix and their own keys in one go: nothing to join
  int beside;        // runs beside the kernel launched before it (see sp_pieces_kernel)
  // own keys by sp_stream_kernel (prefix_stream.cuh): cuts > 0 stretches, the tiles before every
  // sequence (B + 1), and two boundary slots of 16 rows for every stretch
  int cuts;
  long* tile_start;
  float* cut_o;
  float2* cut_ml;
  SpSplit split;
};

constexpr int kSpKeys = 64;  // keys of a tile
// Fewest tiles of a part: a part's join costs about as much as four tiles in bf16, as one in fp32
// (16 streams behind 1000 keys, parts of at least 4 and 1 tiles: 28.8 and 15.9 us).
template <typename T>
__host__ __device__ constexpr int sp_least() {
  return sizeof(T) == 2 ? 4 : 1;
}

struct SpSeq {
  int q0, nq, nk;
  long base;
};
// The device arrays of a sequence, checked: rows outside the buffers are never touched.
__device__ __forceinline__ SpSeq sp_sequence(const SpArgs& a, int b, bool report) {
  SpSeq s;
  const int c0 = a.cu[b], c1 = a.cu[b + 1];
  s.q0 = c0;
  s.nq = c1 - c0;
  if (c0 < 0 || c1 < c0 || c1 > a.N) {
    if (report) record_error(611);
    s.q0 = 0;
    s.nq = 0;
  }
  s.base = a.kv_base ? a.kv_base[b] : s.q0;
  s.nk = a.kv_lens ? a.kv_lens[b] : s.nq;
  if (s.nk < 0 || s.base < 0 || s.base + s.nk > a.kv_rows) {
    if (s.nk != 0 && report) record_error(612);
    s.base = 0;
    s.nk = 0;
  }
  return s;
}
// Own keys, of nk, that a query at own position `at` sees (negative: before the first own key).
__device__ __forceinline__ int sp_limit_at(const SpArgs& a, int nk, int at) {
  if (a.chunk <= 0) return nk;
  const long pos = (long)a.P + at;
  if (pos < 0) return 0;
  const long lim = a.chunk == 1 ? (long)at + 1 : (pos / a.chunk + 1) * a.chunk - a.P;
  return lim < 0 ? 0 : (lim < nk ? static_cast<int>(lim) : nk);
}
// Own keys that query i of the sequence sees.
__device__ __forceinline__ int sp_limit(const SpArgs& a, const SpSeq& s, int i) {
  return sp_limit_at(a, s.nk, s.nk - s.nq + i);
}
// Tiles [t0, t1) of piece `part` out of at most `parts` over `tiles` tiles: pieces of equal size,
// none shorter than `least` tiles unless it is the last.
__device__ __forceinline__ void sp_piece(int tiles, int parts, int least, int part, int& t0, int& t1) {
  const int n = max(1, min(parts, (tiles + least - 1) / least));
  const int each = (tiles + n - 1) / n;
  t0 = min(tiles, part * each);
  t1 = part < n ? min(tiles, t0 + each) : t0;
}

// A stretch of keys of one key head: tiles [t0, t1) of the rows of k / v, of which the first kend exist.
template <typename T>
struct SpKeys {
  const T* k;
  const T* v;
  long ks, vs;  // row strides
  int kend, t0, t1;
};

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

// One piece: stacked rows [R0, R0 + rows) of key head hk (rows <= 16 WM) against the tiles of `pre`
// (keys that every row sees) and then of `own` (row r of the block sees keys [0, limit(r))).  The
// result is part `part` of the rows, or final for part < 0.  4 warps: WM of them along the rows (16
// each), 4 / WM along the keys of a tile; for WM < 4 the warps' partial results are joined in shared
// memory.
// K, V tiles come by 16-byte asynchronous copies into a ring; a row of a tile is D / 8 chunks of
// 16 bytes, chunk c of row r at c ^ (r % 8), which keeps ldmatrix free of bank conflicts.
// Rows past the last key are zero in shared memory, so stale values behind a sequence never reach a product.
template <int D, int WM, typename Limit>
__device__ __forceinline__ void sp_mma_piece(const SpArgs& a, uint8_t* smem, const SpKeys<bf16>& pre,
                                             const SpKeys<bf16>& own, int hk, long R0, int rows, int part,
                                             Limit limit) {
  using C = SpMma<D>;
  constexpr int WK = 4 / WM;
  constexpr int KW = kSpKeys / WK;  // keys of a tile that a warp takes
  constexpr int CH = D / 8;         // 16-byte chunks of a row
  constexpr int STAGES = C::kStages;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int wm = warp % WM, wk = warp / WM;
  const uint32_t s0 = smem_u32(smem), sQ = s0, sKV = s0 + C::kQ;
  const bool direct = part < 0;
  const int n_pre = pre.t1 - pre.t0, tiles = n_pre + own.t1 - own.t0;

  auto put = [&](uint32_t base, int r, int c) { return base + r * (D * 2) + ((c ^ (r & 7)) << 4); };
  __syncthreads();  // an earlier piece of this block has left the buffers
  for (int i = tid; i < 16 * WM * CH; i += 128) {
    const int r = i / CH, c = i % CH;
    const bool ok = r < rows;
    const SpRow x = sp_row(a, hk, R0 + (ok ? r : 0));
    cp_async16(put(sQ, r, c), static_cast<const bf16*>(a.q) + x.token * a.q_stride + (long)x.head * D + 8 * c, ok);
  }
  const int lr = tid / CH, lc = tid % CH;  // this thread copies chunk lc of rows lr, lr + 128 / CH, ...
  auto load = [&](int u) {
    const bool first = u < n_pre;
    const SpKeys<bf16>& src = first ? pre : own;
    const int key = (src.t0 + (first ? u : u - n_pre)) * kSpKeys + lr;
    const uint32_t kb = sKV + (u % STAGES) * 2 * C::kTile, vb = kb + C::kTile;
    const bf16* kp = src.k + key * src.ks + 8 * lc;
    const bf16* vp = src.v + key * src.vs + 8 * lc;
#pragma unroll
    for (int j = 0; j < kSpKeys * CH / 128; ++j) {
      constexpr int step = 128 / CH;
      const bool ok = key + j * step < src.kend;
      cp_async16(put(kb, lr + j * step, lc), ok ? kp + j * step * src.ks : src.k, ok);
      cp_async16(put(vb, lr + j * step, lc), ok ? vp + j * step * src.vs : src.v, ok);
    }
  };
#pragma unroll
  for (int i = 0; i < STAGES - 1; ++i) {
    if (i < tiles) load(i);
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

  for (int t = 0; t < tiles; ++t) {
    cp_async_wait<STAGES - 2>();
    __syncthreads();
    if (t + STAGES - 1 < tiles) load(t + STAGES - 1);
    cp_async_commit();
    if (t == 0) {
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk)
        ldsm4(put(sQ, 16 * wm + (lane & 15), 2 * kk + (lane >> 4)), qf[kk][0], qf[kk][1], qf[kk][2], qf[kk][3]);
    }
    const uint32_t kb = sKV + (t % STAGES) * 2 * C::kTile, vb = kb + C::kTile;
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
    const bool first = t < n_pre;
    const int k0 = (first ? pre.t0 + t : own.t0 + t - n_pre) * kSpKeys + wk * KW;
    if ((first ? pre.kend : wmin) < k0 + KW) {  // some row of the warp stops inside this warp's keys
      const int c0 = k0 + 2 * (lane & 3), z0 = first ? pre.kend : lim0, z1 = first ? pre.kend : lim1;
#pragma unroll
      for (int i = 0; i < KW / 8; ++i) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          if (c0 + 8 * i + j >= z0) s[i][j] = -INFINITY;
          if (c0 + 8 * i + j >= z1) s[i][2 + j] = -INFINITY;
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
    // P is rounded to bf16 for the product (at most half a step, 2^-8 relative, averaged over the
    // keys); its sum stays in float32
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
// d (two floats) += a b, as one instruction.
__device__ __forceinline__ void ffma2(float2& d, const float2& a, const float2& b) {
  asm("{\n\t.reg .b64 a, b, d;\n\t"
      "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 d, {%0, %1};\n\t"
      "fma.rn.f32x2 d, a, b, d;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "+f"(d.x), "+f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
}
// 128 threads, 8 x 16: thread (ty, tx) has rows RPT ty .. and, of S, keys tx + 16 j, of O,
// columns 4 tx + 64 c.  Rows in shared memory are padded by 4 floats, so the 16-byte reads of 8
// neighbouring rows fall into different banks.  Bound by the FMA pipe and, beside it, by the
// shared-memory reads: with 8 rows a thread, 12 16-byte reads feed 128 multiply-adds; S keeps two
// partial sums (even and odd d), so that a pair of them is one instruction.
template <int D, int RPT>
struct SpF32 {
  static constexpr int kRows = 8 * RPT;
  static constexpr int kThreads = 128;
  static constexpr int kLd = D + 4;
  static constexpr int kStages = 2;
  static constexpr int kSmem = 4 * (kRows * kLd + kStages * 2 * kSpKeys * kLd + kRows * (kSpKeys + 4));
};
template <int D, int RPT, typename Limit>
__device__ __forceinline__ void sp_f32_piece(const SpArgs& a, uint8_t* smem, const SpKeys<float>& pre,
                                             const SpKeys<float>& own, int hk, long R0, int rows, int part,
                                             Limit limit) {
  using C = SpF32<D, RPT>;
  constexpr int LD = C::kLd, CH = D / 4, PLD = kSpKeys + 4, TH = C::kThreads;
  float* sQ = reinterpret_cast<float*>(smem);
  float* sKV = sQ + C::kRows * LD;
  float* sP = sKV + C::kStages * 2 * kSpKeys * LD;
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
  const bool direct = part < 0;
  const int n_pre = pre.t1 - pre.t0, tiles = n_pre + own.t1 - own.t0;
  __syncthreads();
  for (int i = tid; i < C::kRows * CH; i += TH) {
    const int r = i / CH, c = i % CH;
    const bool ok = r < rows;
    const SpRow x = sp_row(a, hk, R0 + (ok ? r : 0));
    cp_async16(smem_u32(sQ + r * LD + 4 * c),
               static_cast<const float*>(a.q) + x.token * a.q_stride + (long)x.head * D + 4 * c, ok);
  }
  const int lr = tid / CH, lc = tid % CH;  // this thread copies chunk lc of rows lr, lr + TH / CH, ...
  auto load = [&](int u) {
    const bool first = u < n_pre;
    const SpKeys<float>& src = first ? pre : own;
    const int key = (src.t0 + (first ? u : u - n_pre)) * kSpKeys + lr;
    float* kb = sKV + (u & 1) * 2 * kSpKeys * LD + lr * LD + 4 * lc;
    float* vb = kb + kSpKeys * LD;
    const float* kp = src.k + key * src.ks + 4 * lc;
    const float* vp = src.v + key * src.vs + 4 * lc;
#pragma unroll 4
    for (int j = 0; j < kSpKeys * CH / TH; ++j) {
      constexpr int step = TH / CH;
      const bool ok = key + j * step < src.kend;
      cp_async16(smem_u32(kb + j * step * LD), ok ? kp + j * step * src.ks : src.k, ok);
      cp_async16(smem_u32(vb + j * step * LD), ok ? vp + j * step * src.vs : src.v, ok);
    }
  };
  if (tiles > 0) load(0);
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
  for (int t = 0; t < tiles; ++t) {
    cp_async_wait<0>();
    __syncthreads();
    if (t + 1 < tiles) load(t + 1);
    cp_async_commit();
    const float* kb = sKV + (t & 1) * 2 * kSpKeys * LD;
    const float* vb = kb + kSpKeys * LD;
    float2 s2[RPT][4];
#pragma unroll
    for (int i = 0; i < RPT; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) s2[i][j] = make_float2(0.f, 0.f);
#pragma unroll 2
    for (int d = 0; d < D; d += 4) {
      float4 kv[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) kv[j] = *reinterpret_cast<const float4*>(kb + (tx + 16 * j) * LD + d);
#pragma unroll
      for (int i = 0; i < RPT; ++i) {
        const float4 qv = *reinterpret_cast<const float4*>(sQ + (RPT * ty + i) * LD + d);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          ffma2(s2[i][j], make_float2(qv.x, qv.y), make_float2(kv[j].x, kv[j].y));
          ffma2(s2[i][j], make_float2(qv.z, qv.w), make_float2(kv[j].z, kv[j].w));
        }
      }
    }
    const bool first = t < n_pre;
    const int k0 = (first ? pre.t0 + t : own.t0 + t - n_pre) * kSpKeys + tx;
#pragma unroll
    for (int i = 0; i < RPT; ++i) {
      float x = -INFINITY, s[4];
      const int z = first ? pre.kend : lim[i];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        s[j] = k0 + 16 * j < z ? (s2[i][j].x + s2[i][j].y) * a.scale_log2 : -INFINITY;
        x = fmaxf(x, s[j]);
      }
#pragma unroll
      for (int w = 1; w < 16; w <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, w));
      const float mn = fmaxf(m[i], x), ref = mn == -INFINITY ? 0.f : mn;
      const float e = exp2f(m[i] - ref);
      m[i] = mn;
      float y = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float p = exp2f(s[j] - ref);
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
// blocks of the sequence; with `whole` they take the prefix as well.  RP / RO: rows of a block of
// the prefix / of a sequence; they set the shape of the block (see the piece functions).
// `beside`: the tensor-core kernel of the prefix parts was launched just before on a part of the
// SMs, and this kernel fills the others.  Every block of that kernel has waited for the work before
// it when this one starts, and its results are not read here, so the wait moves to the end, where
// it makes this kernel's completion imply the other's.
template <typename T, int D, int RP, int RO>
__device__ __forceinline__ void sp_block(const SpArgs& a, uint8_t* smem) {
  auto piece = [&](auto rows_c, const SpKeys<T>& pre, const SpKeys<T>& own, int hk, long R0, int rows, int part,
                   auto limit) {
    constexpr int R = decltype(rows_c)::value;
    if constexpr (sizeof(T) == 2)
      sp_mma_piece<D, R / 16>(a, smem, pre, own, hk, R0, rows, part, limit);
    else
      sp_f32_piece<D, R / 8>(a, smem, pre, own, hk, R0, rows, part, limit);
  };
  int it = blockIdx.x;
  SpKeys<T> pre{static_cast<const T*>(a.pk), static_cast<const T*>(a.pv), a.pk_stride, a.pv_stride, a.P, 0, 0};
  SpKeys<T> own{static_cast<const T*>(a.k), static_cast<const T*>(a.v), a.k_stride, a.v_stride, 0, 0, 0};
  const int prefix_tiles = (a.P + kSpKeys - 1) / kSpKeys;
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
    sp_piece(prefix_tiles, a.prefix_parts, sp_least<T>(), part, pre.t0, pre.t1);
    pre.k += (long)hk * D;
    pre.v += (long)hk * D;
    piece(std::integral_constant<int, RP>(), pre, own, hk, r0, static_cast<int>(r1 - r0), part,
          [](int) { return 0; });
    return;
  }
  it -= a.prefix_items;
  const int part = it % a.own_parts;
  it /= a.own_parts;
  const int hk = it % a.Hkv, b = it / a.Hkv;
  const SpSeq s = sp_sequence(a, b, threadIdx.x == 0);
  const long nrows = (long)s.nq * a.G;
  pre.k += (long)hk * D;
  pre.v += (long)hk * D;
  own.k += s.base * a.k_stride + (long)hk * D;
  own.v += s.base * a.v_stride + (long)hk * D;
  own.kend = s.nk;
  if (a.whole) pre.t1 = prefix_tiles;
  for (long r = (long)blockIdx.y * RO; r < nrows; r += (long)gridDim.y * RO) {
    const int rows = static_cast<int>(min((long)RO, nrows - r));
    const int seen = sp_limit(a, s, static_cast<int>((r + rows - 1) / a.G));  // limits grow along the rows
    sp_piece((seen + kSpKeys - 1) / kSpKeys, a.own_parts, sp_least<T>(), part, own.t0, own.t1);
    piece(std::integral_constant<int, RO>(), pre, own, hk, (long)s.q0 * a.G + r, rows,
          a.whole ? -1 : a.prefix_parts + part,
          [&](int i) { return sp_limit(a, s, static_cast<int>((r + i) / a.G)); });
  }
}
template <typename T, int D, int RP, int RO>
__global__ void __launch_bounds__(128) sp_pieces_kernel(const SpArgs a) {
  extern __shared__ __align__(128) uint8_t smem[];
  if (!a.beside) griddep_wait();
  griddep_launch();
  sp_block<T, D, RP, RO>(a, smem);
  if (a.beside) griddep_wait();
}

// Own parts left by sp_stream_kernel.  The (sequence, row block, key head) items lie end to end, each
// kSsItem units for its own cost (start, join) and one for every key tile, and are cut into equal
// stretches (64 sequences of 1 to 1023 keys: 79 us when only tiles count, 62 with three units an item).
constexpr int kSsItem = 3;
struct SsCount {
  int blocks, tiles;  // row blocks of 16 / G tokens; key tiles of each item
  __device__ __forceinline__ int units() const { return tiles > 0 ? tiles + kSsItem : 0; }
  __device__ __forceinline__ long all(int Hkv) const { return (long)blocks * Hkv * units(); }
};
__device__ __forceinline__ SsCount ss_count(const SpArgs& a, int nq, int nk) {
  const int per = 16 / a.G;
  SsCount c;
  c.blocks = (nq + per - 1) / per;
  c.tiles = (nk + kSpKeys - 1) / kSpKeys;
  return c;
}
// Stretches of `total` units (none is empty), the first unit of stretch c, the stretch that holds a unit.
__device__ __forceinline__ int ss_stretches(long total, int cuts) {
  return static_cast<int>(min(total, (long)cuts));
}
__device__ __forceinline__ long ss_cut(long total, int n, long c) { return total * c / n; }
__device__ __forceinline__ int ss_stretch(long total, int n, long unit) {
  return static_cast<int>(((unit + 1) * n - 1) / total);
}

// The choice whose slower side is the fastest for `units` of own keys.
__device__ __forceinline__ int sp_pick(const SpSplit& s, long units) {
  int best = 0;
  float best_us = 0.f;
  const float u = static_cast<float>(units);
  for (int i = 0; i < s.n; ++i) {
    // rounded one by one: every kernel has to come to the same figure
    const float us = s.own_us[i] > 0.f ? fmaxf(s.fa_us[i], __fmul_rn(u, s.own_us[i]))
                                       : __fadd_rn(s.fa_us[i], __fmul_rn(u, s.floor_us));
    if (i == 0 || us < best_us) best = i, best_us = us;
  }
  return best;
}
__device__ __forceinline__ int sp_pick_cuts(const SpSplit& s, int i) {
  return s.ctas[i] < s.sms ? s.sms - s.ctas[i] : s.sms;
}

// Joins the parts of a row: one warp per (token, head).  Its loads are a chain of round trips (the
// token's sequence, the parts' maxima and sums, their outputs), so what can be read at once is: part by
// part it took 24 us for 2048 rows of 17 parts, like this 7 us for the 5 parts that they have now.
// REPORT: without own parts no kernel before this one has looked at the sequences, so the first block
// reports those out of range (behind a runtime check it cost every call 0.3 us).
template <typename T, int D, bool REPORT>
__global__ void __launch_bounds__(256) sp_join_kernel(const SpArgs a) {
  const int lane = threadIdx.x & 31;
  const long w = (long)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int token = static_cast<int>(min(w / a.H, (long)a.N));
  const int head = static_cast<int>(w - (long)token * a.H);
  const long step = (long)a.N * a.H;
  // The caller's arrays may be read before the wait: the kernels that leave the parts launch this one
  // after their own wait (or the one beside them did) for whatever was on the stream before the call.
  const int begin = a.cu[0], end = a.cu[a.B];
  int b = 0;
  SpSeq s{};
  if (a.cuts > 0 && token < a.N) {
    // the token's sequence: its own number when every sequence has one query
    b = min(token, a.B - 1);
    s = sp_sequence(a, b, false);
    if (s.q0 > token || s.q0 + s.nq <= token) {
      int lo = 0, hi = a.B - 1;
      while (lo < hi) {
        const int mid = (lo + hi) / 2;
        if (a.cu[mid + 1] > token) hi = mid;
        else lo = mid + 1;
      }
      b = lo;
      s = sp_sequence(a, b, false);
    }
  }
  griddep_wait();
  griddep_launch();
  if (REPORT && blockIdx.x == 0)
    for (int i = threadIdx.x; i < a.B; i += blockDim.x) sp_sequence(a, i, true);
  if (token >= a.N || token < begin || token >= end) return;  // rows behind the last sequence stay
  // own parts: all of them, or (cuts) one in the row's own place or one in each stretch that the item meets
  int own = a.own_parts, first = -1, prefix_parts = a.prefix_parts;
  long slot_row = 0;
  if (a.cuts > 0) {
    own = 0;
    const long total = a.tile_start[a.B];
    long start = a.tile_start[b];
    const SsCount c = ss_count(a, s.nq, s.nk);
    const int i = token - s.q0;
    int cuts = a.cuts;
    if (a.split.n > 0) {
      const int pick = sp_pick(a.split, total);
      cuts = sp_pick_cuts(a.split, pick);
      prefix_parts = a.split.parts[pick];
    }
    if (i >= 0 && i < s.nq && c.tiles > 0) {
      const int per = 16 / a.G, hk = head / a.G, rb = i / per;
      start += (long)(rb * a.Hkv + hk) * c.units() + kSsItem;  // the item's first tile
      const int n = ss_stretches(total, cuts);
      const int c0 = ss_stretch(total, n, start), c1 = ss_stretch(total, n, start + c.tiles - 1);
      own = c1 - c0 + 1;
      if (own > 1) first = c0;
      slot_row = (i - rb * per) * a.G + (head - hk * a.G);
    }
  }
  const int parts = prefix_parts + own;
  // part p of the row: its index among the stored maxima and sums (and, times D, among the outputs)
  auto place = [&](int p, const float2*& ml, const float*& o) {
    if (p >= prefix_parts && first >= 0) {
      const int c = first + p - prefix_parts;
      // a stretch keeps the item that began before it in slot 0, the one that goes on behind it in slot 1
      const long at = (2L * c + (c == first ? 1 : 0)) * 16 + slot_row;
      ml = a.cut_ml + at;
      o = a.cut_o + at * D;
    } else {
      // own part 0 stands behind the places of a.prefix_parts parts, of which fewer may be in use
      const long at = (p < prefix_parts ? p : a.prefix_parts + p - prefix_parts) * step + w;
      ml = a.part_ml + at;
      o = a.part_o + at * D;
    }
  };
  // 32 parts at a time: lane p has part p's maximum, sum and place; the outputs are then read by the
  // whole warp, eight parts in flight
  constexpr int V = D / 32;
  float acc[V];
#pragma unroll
  for (int i = 0; i < V; ++i) acc[i] = 0.f;
  float m = -INFINITY, l = 0.f;
  for (int p0 = 0; p0 < parts; p0 += 32) {
    const int n = min(32, parts - p0);
    float2 ml = make_float2(-INFINITY, 0.f);
    const float* o = nullptr;
    if (lane < n) {
      const float2* at;
      place(p0 + lane, at, o);
      ml = *at;
    }
    float top = ml.x;
#pragma unroll
    for (int i = 16; i > 0; i >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, i));
    const float m_new = fmaxf(m, top);
    if (m_new > m) {  // rescale what the parts before left
      const float f = exp2f(m - m_new);
      l *= f;
#pragma unroll
      for (int i = 0; i < V; ++i) acc[i] *= f;
      m = m_new;
    }
    // a part that saw no key (maximum -inf, sum 0) holds no output; a sum that is NaN is kept
    const bool some = ml.x != -INFINITY || ml.y != 0.f;
    const float f = !some ? 0.f : (m == -INFINITY ? 1.f : exp2f(ml.x - m));
    float part = some ? ml.y * f : 0.f;
#pragma unroll
    for (int i = 16; i > 0; i >>= 1) part += __shfl_xor_sync(0xffffffffu, part, i);
    l += part;
    uint32_t todo = __ballot_sync(0xffffffffu, some);
    while (todo) {
      float v[8][V], g[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int p = todo ? __ffs(todo) - 1 : 0;
        const bool have = todo != 0;
        todo &= todo - 1;
        g[u] = __shfl_sync(0xffffffffu, f, p);
        const unsigned long long at = __shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(o), p);
        const float* src = reinterpret_cast<const float*>(at) + V * lane;
#pragma unroll
        for (int i = 0; i < V; ++i) v[u][i] = have ? src[i] : 0.f;
        if (!have) g[u] = 0.f;
      }
#pragma unroll
      for (int u = 0; u < 8; ++u)
#pragma unroll
        for (int i = 0; i < V; ++i) acc[i] = fmaf(v[u][i], g[u], acc[i]);
    }
  }
  const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
  T* dst = static_cast<T*>(a.out) + token * a.out_stride + (long)head * D + V * lane;
#pragma unroll
  for (int i = 0; i < V; ++i) dst[i] = from_f<T>(acc[i] * inv);
}

}  // namespace fcv
