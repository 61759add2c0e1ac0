// qknorm.cuh -- per-head RMS norm of queries and keys with the position rotation.
//
// For every token n of packed [Q | K | V] rows and every head x (D values) of Q and K:
//     y = x * rsqrt(mean(x^2) + eps) * w            (w: one D-vector for Q, one for K)
//     (y_a, y_b) -> (y_a c - y_b s, y_b c + y_a s)   c, s = cos/sin[position[n]][i], i < half
// over the pairs (2i, 2i + 1) (interleaved) or (i, i + half); values past 2 half only get the
// norm.  Values V are copied when the keys go to a cache.  Sums and products are float32; each
// output is rounded once.
//
// Bound by memory: every value is read and written once.  On a B200 (copy: 6.54 TB/s), calls one after
// another: 96000 tokens of 16/16 heads of 64 in bf16, 788 MB, 146 us (5.4 TB/s); 6577 tokens of 32/8 heads
// of 128 into scattered cache rows, 164 MB, 31.6 us (5.2 TB/s); 20914 tokens of 16/16 heads of 64 in
// float32, 343 MB, 55.7 us (6.2 TB/s).  Two, three and six steps in flight and three or four blocks on an SM
// measure the same within 1 %; a warp that loops over tokens, the next one's loads ahead, 147 us.
#pragma once

#include "fcv_common.cuh"

namespace fcv {

struct QkNormArgs {
  const void* qkv;
  long row_stride;  // elements
  int N, heads, kv_heads;
  const float* q_weight;  // null: 1
  const float* k_weight;
  float eps;
  const float* cos;  // (rope_rows, half)
  const float* sin;
  int rope_rows, half;
  const int32_t* positions;
  void* q_out;
  long q_stride;
  void* k_out;
  long k_stride;
  void* v_out;  // null: values are not copied
  long v_stride;
  const int32_t* kv_rows;  // null: token n's keys go to row n; an entry < 0 stores nothing
  long kv_limit;           // rows of k_out / v_out
  int warps_per_row;
};

template <typename T>
struct Vec8;
template <>
struct Vec8<bf16> {
  uint4 u;
  __device__ __forceinline__ void load(const bf16* p) { u = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void store(bf16* p) const { *reinterpret_cast<uint4*>(p) = u; }
  __device__ __forceinline__ void get(float (&x)[8]) const {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
  __device__ __forceinline__ void set(const float (&x)[8]) {
    u = make_uint4(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]),
                   pack_bf16x2(x[6], x[7]));
  }
};
template <>
struct Vec8<float> {
  float4 a, b;
  __device__ __forceinline__ void load(const float* p) {
    a = *reinterpret_cast<const float4*>(p);
    b = *reinterpret_cast<const float4*>(p + 4);
  }
  __device__ __forceinline__ void store(float* p) const {
    *reinterpret_cast<float4*>(p) = a;
    *reinterpret_cast<float4*>(p + 4) = b;
  }
  __device__ __forceinline__ void get(float (&x)[8]) const {
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w;
    x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
  }
  __device__ __forceinline__ void set(const float (&x)[8]) {
    a = make_float4(x[0], x[1], x[2], x[3]);
    b = make_float4(x[4], x[5], x[6], x[7]);
  }
};

// A warp takes (a share of) one token's heads, 256 / D heads at a time: D / 8 lanes hold a head,
// 8 values each, so loads and stores are 16 bytes wide (32 in float32) and the sum of squares is a
// few shuffles.  The token's cos / sin values and the weights stay in registers over its heads; U
// steps are loaded before any is finished, the first of them before the token's position is known.
template <typename T, int D, bool INTERLEAVED>
__global__ void __launch_bounds__(256, sizeof(T) == 2 ? 3 : 2) qk_norm_rope_kernel(const QkNormArgs a) {
  griddep_wait();
  griddep_launch();
  constexpr int L = D / 8;          // lanes of a head
  constexpr int HPW = 32 / L;       // heads of one step of the warp
  constexpr int U = sizeof(T) == 2 ? 4 : 2;  // steps in flight
  const int lane = threadIdx.x & 31;
  const long w = (long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  const long n = w / a.warps_per_row;
  const int part = static_cast<int>(w - n * a.warps_per_row);
  if (n >= a.N) return;
  const int sub = lane / L, l = lane % L, d0 = 8 * l;
  const T* row = static_cast<const T*>(a.qkv) + n * a.row_stride + d0;
  const int step = HPW * a.warps_per_row;
  const int units = a.heads + a.kv_heads;
  Vec8<T> v[U];
  auto load = [&](int base, int end) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int h = base + u * step + sub;
      if (h < end) v[u].load(row + (long)h * D);
    }
  };
  load(part * HPW, units);
  const int pos = a.positions[n];
  long kv_row = a.kv_rows ? a.kv_rows[n] : n;
  if (pos < 0 || pos >= a.rope_rows) {
    if (lane == 0) record_error(601);
    return;
  }
  if (kv_row >= a.kv_limit) {
    if (lane == 0) record_error(602);
    kv_row = -1;
  }
  // rotation of this lane's values: INTERLEAVED uses pairs 4l .. 4l+3 (cs[0..3]); halves use table
  // entries d0 mod half, the partner values sitting half / 8 lanes away
  float cs[8], sn[8];
  const bool rot = d0 < 2 * a.half;
  int src = lane;
  if (rot) {
    const long at = (long)pos * a.half;
    if (INTERLEAVED) {
      const float4 c4 = *reinterpret_cast<const float4*>(a.cos + at + 4 * l);
      const float4 s4 = *reinterpret_cast<const float4*>(a.sin + at + 4 * l);
      cs[0] = c4.x, cs[1] = c4.y, cs[2] = c4.z, cs[3] = c4.w;
      sn[0] = s4.x, sn[1] = s4.y, sn[2] = s4.z, sn[3] = s4.w;
    } else {
      const bool low = d0 < a.half;
      const long i = at + (low ? d0 : d0 - a.half);
      Vec8<float> t;
      t.load(a.cos + i), t.get(cs);
      t.load(a.sin + i), t.get(sn);
      src = lane + (low ? a.half / 8 : -a.half / 8);
      if (low) {
#pragma unroll
        for (int j = 0; j < 8; ++j) sn[j] = -sn[j];
      }
    }
  }
  // queries, then keys (a step may hold the last of the one and the first of the other)
  float wt[8];
  auto weights = [&](const float* p) {
    if (p) {
      Vec8<float> t;
      t.load(p + d0), t.get(wt);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) wt[i] = 1.f;
    }
  };
  bool of_q = part * HPW + sub < a.heads;
  weights(of_q ? a.q_weight : a.k_weight);
  for (int base = part * HPW; base < units; base += U * step) {
    if (base != part * HPW) load(base, units);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int h0 = base + u * step;
      if (h0 >= units) break;  // warp-uniform
      const int h = h0 + sub;
      const bool is_q = h < a.heads;
      if (is_q != of_q) {  // the lane's last query head is behind it
        weights(a.k_weight);
        of_q = false;
      }
      float x[8];
      v[u].get(x);
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) ss = fmaf(x[i], x[i], ss);
#pragma unroll
      for (int o = L / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      const float r = rsqrtf(ss * (1.f / D) + a.eps);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = x[i] * r * wt[i];
      if (INTERLEAVED) {
        if (rot) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float p = x[2 * i], q = x[2 * i + 1];
            x[2 * i] = p * cs[i] - q * sn[i];
            x[2 * i + 1] = q * cs[i] + p * sn[i];
          }
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float other = __shfl_sync(0xffffffffu, x[i], src);
          if (rot) x[i] = x[i] * cs[i] + other * sn[i];
        }
      }
      v[u].set(x);
      if (is_q)
        v[u].store(static_cast<T*>(a.q_out) + n * a.q_stride + (long)h * D + d0);
      else if (h < units && kv_row >= 0)
        v[u].store(static_cast<T*>(a.k_out) + kv_row * a.k_stride + (long)(h - a.heads) * D + d0);
    }
  }
  if (a.v_out == nullptr || kv_row < 0) return;
  row += (long)units * D;
  for (int base = part * HPW; base < a.kv_heads; base += U * step) {
    load(base, a.kv_heads);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int h = base + u * step + sub;
      if (h < a.kv_heads) v[u].store(static_cast<T*>(a.v_out) + kv_row * a.v_stride + (long)h * D + d0);
    }
  }
}

}  // namespace fcv
