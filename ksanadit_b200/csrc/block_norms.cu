// Norms on both sides of a block's half, with its gate, its residual scale and the residual sum between them:
//
//   r = x + a * gate * N(y) * wp          N(v) = v * rsqrt(mean(v^2) + eps), or the same of v - mean(v)
//   h = N(r) * wn * (1 + scale) + shift
//
// and the gradients of both.  With yh = N(y), rh = N(r), A = a gate wp, B = (1 + scale) wn, t = dh B and D = dr + the gradient of r through h:
//
//   D  = dr + rstd_r (t - rh mean(t rh) - mean(t))      dx = D            (mean(t) and mean(e) only where N subtracts the mean)
//   dy = rstd_y (e - yh mean(e yh) - mean(e)), e = D A
//   dgate = a wp sum(D yh)   dwp = a sum(D gate yh)   dscale = wn sum(dh rh)   dwn = sum(dh (1 + scale) rh)   dshift = sum(dh)
//
// where the sums run over the rows that share a modulation row, or all.  Bound by HBM: x, y in and r, h out, 8 C bytes a row; x, y,
// dr, dh in and dx, dy out, 12 C bytes.  r is formed anew from x and y in the backward pass, which costs no more bytes than reading it
// would and is not rounded.  All arithmetic is fp32, each result is rounded once: h is the norm of the unrounded r.
//
// Columns are taken in chunks of 8 (one 128-bit access per tensor); a row is owned by a group of warps whose threads hold one chunk
// or two, and the next row's loads are issued before the present row's sums are exchanged.
#include <algorithm>

#include "../../include/ksana_b200.h"
#include "common.cuh"
#include "host_utils.h"

namespace ksb {
namespace norms {

constexpr int MAX_WARPS = 32, MAX_GROUPS = 12;

struct Params {
  const void* x;
  const void* y;  // null: r = x
  int64_t ldx, ldy, M;
  int C;
  float eps, a;
  // modulation row of row m: rows m / rows_per_mod, `stride` elements apart; each may be null
  const void* gate;
  const void* scale;
  const void* shift;
  int64_t gate_stride, scale_stride, shift_stride, rows_per_mod;
  const float* post_w;  // or null
  const float* pre_w;
  float4* stats;  // per row: mean and 1 / std of y, of r; or null
  void* r;
  void* h;        // null: no norm behind the sum
};

struct Grads {
  const void* dr;  // or null
  const void* dh;  // or null
  int64_t lddr, lddh;
  void* dx;        // or null
  void* dy;        // or null
  void* dgate;     // [M / rows_per_mod, C] halves each, or null
  void* dscale;
  void* dshift;
  float* dpost_w;  // [C] or null
  float* dpre_w;
  float* parts;    // workspace
  int64_t chunk_rows;
  int chunks;      // of the rows that share a modulation row
  int samples;     // modulation rows
};

__device__ __forceinline__ uint4 load8(const void* base, int64_t offset_bytes) { return *reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(base) + offset_bytes); }

template <typename T> __device__ __forceinline__ void unpack8(const uint4& v, float (&f)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 p = HalfOps<T>::unpack2(w[i]);
    f[2 * i] = p.x;
    f[2 * i + 1] = p.y;
  }
}
template <typename T> __device__ __forceinline__ uint4 pack8(const float (&f)[8]) {
  return make_uint4(HalfOps<T>::pack2(make_float2(f[0], f[1])), HalfOps<T>::pack2(make_float2(f[2], f[3])), HalfOps<T>::pack2(make_float2(f[4], f[5])),
                    HalfOps<T>::pack2(make_float2(f[6], f[7])));
}
__device__ __forceinline__ void weight8(const float* w, int c, float (&f)[8]) {
  if (!w) {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = 1.f;
    return;
  }
  const float4 a = *reinterpret_cast<const float4*>(w + c * 8), b = *reinterpret_cast<const float4*>(w + c * 8 + 4);
  f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
  f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
}
// A = a gate wp of chunk c
template <typename T> __device__ __forceinline__ void post_factor(const Params& p, int64_t mod, int c, float (&f)[8]) {
  weight8(p.post_w, c, f);
  if (p.gate) {
    float g[8];
    unpack8<T>(load8(p.gate, (mod * p.gate_stride + c * 8) * 2), g);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] *= p.a * g[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] *= p.a;
  }
}
// B = (1 + scale) wn of chunk c
template <typename T> __device__ __forceinline__ void pre_factor(const Params& p, int64_t mod, int c, float (&f)[8]) {
  weight8(p.pre_w, c, f);
  if (p.scale) {
    float s[8];
    unpack8<T>(load8(p.scale, (mod * p.scale_stride + c * 8) * 2), s);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] *= 1.f + s[i];
  }
}

// A group of warps that owns a row: sums over its threads.  Each of a row's sums has its own place, and rows take turns between two
// sets of places, so that one barrier per sum is enough.
struct Group {
  float2* red;  // [2][4][warps]
  int id, warps, warp, lane, par;
  __device__ __forceinline__ float2 sum(float2 v, int place) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
      v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
    }
    if (warps == 1) return v;
    float2* at = red + (par * 4 + place) * warps;
    if (lane == 0) at[warp] = v;
    asm volatile("bar.sync %0, %1;" ::"r"(id + 1), "r"(warps * 32) : "memory");
    v = at[0];
    for (int w = 1; w < warps; ++w) {
      const float2 o = at[w];
      v.x += o.x;
      v.y += o.y;
    }
    return v;
  }
  __device__ __forceinline__ float sum(float v, int place) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (warps == 1) return v;
    float2* at = red + (par * 4 + place) * warps;
    if (lane == 0) at[warp].x = v;
    asm volatile("bar.sync %0, %1;" ::"r"(id + 1), "r"(warps * 32) : "memory");
    v = at[0].x;
    for (int w = 1; w < warps; ++w) v += at[w].x;
    return v;
  }
};

// 1 / std of a row of which this thread holds NC chunks, and the row's mean
template <int NC, bool LAYER>
__device__ __forceinline__ float2 row_stats(Group& g, const float (&v)[NC][8], const bool (&live)[NC], float inv_c, float eps, int place) {
  float mean = 0.f;
  if (LAYER) {
    float s = 0.f;
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int i = 0; i < 8; ++i) s += v[c][i];
    mean = g.sum(s, place) * inv_c;
  }
  float s = 0.f;
#pragma unroll
  for (int c = 0; c < NC; ++c)
    if (live[c]) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float d = LAYER ? v[c][i] - mean : v[c][i];
        s = fmaf(d, d, s);
      }
    }
  return make_float2(mean, rsqrtf(g.sum(s, place + 1) * inv_c + eps));
}

template <typename T, int NC, bool LAYER, int THREADS, int CTAS>
__global__ void __launch_bounds__(THREADS, CTAS) forward_kernel(const __grid_constant__ Params p) {
  __shared__ float2 red[2 * 4 * MAX_WARPS];
  const int t = threadIdx.x, nt = blockDim.x, chunks = p.C / 8;
  Group g{red + threadIdx.y * (2 * 4 * (nt / 32)), (int)threadIdx.y, nt / 32, t >> 5, t & 31, 0};
  const float inv_c = 1.f / static_cast<float>(p.C);
  bool live[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c) live[c] = t + c * nt < chunks;
  const int64_t step = static_cast<int64_t>(gridDim.x) * blockDim.y;
  uint4 nx[NC], ny[NC];
  auto fetch = [&](int64_t row) {
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      nx[c] = ny[c] = make_uint4(0, 0, 0, 0);
      if (row < p.M && live[c]) {
        nx[c] = load8(p.x, (row * p.ldx + (t + c * nt) * 8) * 2);
        if (p.y) ny[c] = load8(p.y, (row * p.ldy + (t + c * nt) * 8) * 2);
      }
    }
  };
  int64_t row = static_cast<int64_t>(blockIdx.x) * blockDim.y + threadIdx.y;
  fetch(row);
  for (; row < p.M; row += step, g.par ^= 1) {
    float x[NC][8], y[NC][8];
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      unpack8<T>(nx[c], x[c]);
      unpack8<T>(ny[c], y[c]);
    }
    fetch(row + step);
    const int64_t mod = row / p.rows_per_mod;
    float4 st = make_float4(0.f, 0.f, 0.f, 0.f);
    if (p.y) {
      const float2 s = row_stats<NC, LAYER>(g, y, live, inv_c, p.eps, 0);
      st.x = s.x;
      st.y = s.y;
#pragma unroll
      for (int c = 0; c < NC; ++c)
        if (live[c]) {
          float f[8];
          post_factor<T>(p, mod, t + c * nt, f);
#pragma unroll
          for (int i = 0; i < 8; ++i) x[c][i] = fmaf(f[i], (LAYER ? y[c][i] - s.x : y[c][i]) * s.y, x[c][i]);
          *reinterpret_cast<uint4*>(static_cast<T*>(p.r) + row * p.C + (t + c * nt) * 8) = pack8<T>(x[c]);
        }
    }
    if (p.h) {
      const float2 s = row_stats<NC, LAYER>(g, x, live, inv_c, p.eps, 2);
      st.z = s.x;
      st.w = s.y;
#pragma unroll
      for (int c = 0; c < NC; ++c)
        if (live[c]) {
          float f[8], b[8];
          pre_factor<T>(p, mod, t + c * nt, f);
#pragma unroll
          for (int i = 0; i < 8; ++i) b[i] = 0.f;
          if (p.shift) unpack8<T>(load8(p.shift, (mod * p.shift_stride + (t + c * nt) * 8) * 2), b);
#pragma unroll
          for (int i = 0; i < 8; ++i) b[i] = fmaf((LAYER ? x[c][i] - s.x : x[c][i]) * s.y, f[i], b[i]);
          *reinterpret_cast<uint4*>(static_cast<T*>(p.h) + row * p.C + (t + c * nt) * 8) = pack8<T>(b);
        }
    }
    if (p.stats && t == 0) p.stats[row] = st;
  }
}

// Sums over rows that a thread keeps for its chunk: of D yh, dh rh and dh.
struct Sums {
  float p[8], q[8], s[8];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] = q[i] = s[i] = 0.f;
  }
};

// One chunk per thread.  WHOLE: a group takes all rows of a modulation row, and writes the modulation's gradients itself; else a CTA takes
// a stretch of them and leaves its sums to finish_kernel.
template <typename T, bool LAYER, bool WHOLE, int THREADS>
__global__ void __launch_bounds__(THREADS, 1) backward_kernel(const __grid_constant__ Params p, const __grid_constant__ Grads q) {
  extern __shared__ __align__(16) float shared_sums[];  // [3][C], [2][C] with WHOLE
  __shared__ float2 red[2 * 4 * MAX_WARPS];
  const int t = threadIdx.x, nt = blockDim.x;
  Group g{red + threadIdx.y * (2 * 4 * (nt / 32)), (int)threadIdx.y, nt / 32, t >> 5, t & 31, 0};
  const float inv_c = 1.f / static_cast<float>(p.C);
  const bool live = t < p.C / 8;
  Sums acc;
  acc.clear();
  float wp[8], wn[8];  // WHOLE: of the weights' gradients
#pragma unroll
  for (int i = 0; i < 8; ++i) wp[i] = wn[i] = 0.f;

  uint4 nx, ny, ndr, ndh;
  float4 nst;
  auto fetch = [&](int64_t row, int64_t end) {
    nx = ny = ndr = ndh = make_uint4(0, 0, 0, 0);
    nst = make_float4(0.f, 0.f, 0.f, 0.f);
    if (row < end && live) {
      nx = load8(p.x, (row * p.ldx + t * 8) * 2);
      if (p.y) ny = load8(p.y, (row * p.ldy + t * 8) * 2);
      if (q.dr) ndr = load8(q.dr, (row * q.lddr + t * 8) * 2);
      if (q.dh) ndh = load8(q.dh, (row * q.lddh + t * 8) * 2);
      nst = p.stats[row];
    }
  };
  auto rows = [&](int64_t row, int64_t step, int64_t end, int64_t mod) {
    float A[8], B[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) A[i] = B[i] = 0.f;
    if (live) {
      if (p.y) post_factor<T>(p, mod, t, A);
      if (q.dh) pre_factor<T>(p, mod, t, B);
    }
    fetch(row, end);
    for (; row < end; row += step, g.par ^= 1) {
      float yh[8], r[8], d[8], dh[8];
      unpack8<T>(nx, r);
      unpack8<T>(ny, yh);
      unpack8<T>(ndr, d);
      unpack8<T>(ndh, dh);
      const float4 st = nst;
      fetch(row + step, end);
      if (p.y) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          yh[i] = (LAYER ? yh[i] - st.x : yh[i]) * st.y;
          r[i] = fmaf(A[i], yh[i], r[i]);
        }
      }
      if (q.dh) {
        float2 s = make_float2(0.f, 0.f);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          r[i] = (LAYER ? r[i] - st.z : r[i]) * st.w;
          acc.q[i] = fmaf(dh[i], r[i], acc.q[i]);
          acc.s[i] += dh[i];
          dh[i] *= B[i];
          s.x = fmaf(dh[i], r[i], s.x);
          if (LAYER) s.y += dh[i];
        }
        if (LAYER) s = g.sum(s, 0);
        else s.x = g.sum(s.x, 0);
        s.x *= inv_c;
        s.y *= inv_c;
#pragma unroll
        for (int i = 0; i < 8; ++i) d[i] = fmaf(st.w, dh[i] - r[i] * s.x - (LAYER ? s.y : 0.f), d[i]);
      }
      if (q.dx && live) *reinterpret_cast<uint4*>(static_cast<T*>(q.dx) + row * p.C + t * 8) = pack8<T>(d);
      if (p.y) {
        float2 s = make_float2(0.f, 0.f);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          acc.p[i] = fmaf(d[i], yh[i], acc.p[i]);
          d[i] *= A[i];
          s.x = fmaf(d[i], yh[i], s.x);
          if (LAYER) s.y += d[i];
        }
        if (q.dy) {
          if (LAYER) s = g.sum(s, 1);
          else s.x = g.sum(s.x, 1);
          s.x *= inv_c;
          s.y *= inv_c;
#pragma unroll
          for (int i = 0; i < 8; ++i) d[i] = st.y * (d[i] - yh[i] * s.x - (LAYER ? s.y : 0.f));
          if (live) *reinterpret_cast<uint4*>(static_cast<T*>(q.dy) + row * p.C + t * 8) = pack8<T>(d);
        }
      }
    }
  };
  // the groups' sums of one kind, added up in the order of the groups
  auto add_up = [&](float* to, const float (&v)[8]) {
    if (!live) return;
#pragma unroll
    for (int i = 0; i < 8; ++i) to[t * 8 + i] = threadIdx.y == 0 ? v[i] : to[t * 8 + i] + v[i];
  };
  auto write_sums = [&](float* to, const float (&v)[8]) {
    *reinterpret_cast<float4*>(to + t * 8) = make_float4(v[0], v[1], v[2], v[3]);
    *reinterpret_cast<float4*>(to + t * 8 + 4) = make_float4(v[4], v[5], v[6], v[7]);
  };

  if constexpr (WHOLE) {
    for (int64_t b = static_cast<int64_t>(blockIdx.x) * blockDim.y + threadIdx.y; b < q.samples; b += static_cast<int64_t>(gridDim.x) * blockDim.y) {
      acc.clear();
      rows(b * p.rows_per_mod, 1, (b + 1) * p.rows_per_mod, b);
      if (!live) continue;
      float f[8], o[8];
      auto out = [&](void* to) { *reinterpret_cast<uint4*>(static_cast<T*>(to) + b * p.C + t * 8) = pack8<T>(o); };
      if (p.y) {
        if (q.dpost_w) {
#pragma unroll
          for (int i = 0; i < 8; ++i) f[i] = 1.f;
          if (p.gate) unpack8<T>(load8(p.gate, (b * p.gate_stride + t * 8) * 2), f);
#pragma unroll
          for (int i = 0; i < 8; ++i) wp[i] = fmaf(p.a * f[i], acc.p[i], wp[i]);
        }
        if (q.dgate) {
          weight8(p.post_w, t, f);
#pragma unroll
          for (int i = 0; i < 8; ++i) o[i] = p.a * f[i] * acc.p[i];
          out(q.dgate);
        }
      }
      if (q.dh) {
        if (q.dpre_w) {
#pragma unroll
          for (int i = 0; i < 8; ++i) f[i] = 0.f;
          if (p.scale) unpack8<T>(load8(p.scale, (b * p.scale_stride + t * 8) * 2), f);
#pragma unroll
          for (int i = 0; i < 8; ++i) wn[i] = fmaf(1.f + f[i], acc.q[i], wn[i]);
        }
        if (q.dscale) {
          weight8(p.pre_w, t, f);
#pragma unroll
          for (int i = 0; i < 8; ++i) o[i] = f[i] * acc.q[i];
          out(q.dscale);
        }
        if (q.dshift) {
#pragma unroll
          for (int i = 0; i < 8; ++i) o[i] = acc.s[i];
          out(q.dshift);
        }
      }
    }
    if (!q.dpost_w && !q.dpre_w) return;
    float* to = q.parts + static_cast<int64_t>(blockIdx.x) * 2 * p.C;
    if (blockDim.y == 1) {
      if (live) {
        write_sums(to, wp);
        write_sums(to + p.C, wn);
      }
      return;
    }
    for (int k = 0; k < (int)blockDim.y; ++k) {
      __syncthreads();
      if (k == (int)threadIdx.y) {
        add_up(shared_sums, wp);
        add_up(shared_sums + p.C, wn);
      }
    }
    __syncthreads();
    for (int i = threadIdx.y * nt + t; i < 2 * p.C; i += nt * blockDim.y) to[i] = shared_sums[i];
  } else {
    const int64_t b = blockIdx.x / q.chunks, first = b * p.rows_per_mod, from = first + (blockIdx.x - b * q.chunks) * q.chunk_rows;
    const int64_t last = first + p.rows_per_mod, end = from + q.chunk_rows < last ? from + q.chunk_rows : last;
    rows(from + threadIdx.y, blockDim.y, end, b);
    float* to = q.parts + static_cast<int64_t>(blockIdx.x) * 3 * p.C;
    if (blockDim.y == 1) {
      if (live) {
        write_sums(to, acc.p);
        write_sums(to + p.C, acc.q);
        write_sums(to + 2 * p.C, acc.s);
      }
      return;
    }
    for (int k = 0; k < (int)blockDim.y; ++k) {
      __syncthreads();
      if (k == (int)threadIdx.y) {
        add_up(shared_sums, acc.p);
        add_up(shared_sums + p.C, acc.q);
        add_up(shared_sums + 2 * p.C, acc.s);
      }
    }
    __syncthreads();
    for (int i = threadIdx.y * nt + t; i < 3 * p.C; i += nt * blockDim.y) to[i] = shared_sums[i];
  }
}

// Adds up the stretches' sums, in order: 32 columns per CTA, 16 threads per column, which take turns over the stretches of a
// modulation row, or over the modulation rows where there are many.
constexpr int FINISH = 16;
template <typename T> __global__ void __launch_bounds__(32 * FINISH) finish_kernel(const __grid_constant__ Params p, const __grid_constant__ Grads q) {
  __shared__ float part[3][FINISH][33];
  const int lane = threadIdx.x, j = threadIdx.y, col = blockIdx.x * 32 + lane;
  const bool live = col < p.C;
  pdl_wait();
  const bool by_sample = q.samples >= FINISH;
  const float wp = p.post_w && live ? p.post_w[col] : 1.f, wn = p.pre_w && live ? p.pre_w[col] : 1.f;
  float dwp = 0.f, dwn = 0.f;
  auto write = [&](int b, float sp, float sq, float ss) {
    if (!live) return;
    const float gate = p.gate ? HalfOps<T>::to_f(static_cast<const T*>(p.gate)[b * p.gate_stride + col]) : 1.f;
    const float scale = p.scale ? HalfOps<T>::to_f(static_cast<const T*>(p.scale)[b * p.scale_stride + col]) : 0.f;
    const int64_t at = static_cast<int64_t>(b) * p.C + col;
    if (q.dgate) static_cast<T*>(q.dgate)[at] = HalfOps<T>::from_f(p.a * wp * sp);
    if (q.dscale) static_cast<T*>(q.dscale)[at] = HalfOps<T>::from_f(wn * sq);
    if (q.dshift) static_cast<T*>(q.dshift)[at] = HalfOps<T>::from_f(ss);
    dwp = fmaf(p.a * gate, sp, dwp);
    dwn = fmaf(1.f + scale, sq, dwn);
  };
  auto sums = [&](int b, int first, int step, float (&s)[3]) {
    const float* from = q.parts + (static_cast<int64_t>(b) * q.chunks + first) * 3 * p.C + col;
    s[0] = s[1] = s[2] = 0.f;
    if (!live) return;
    for (int c = first; c < q.chunks; c += step, from += static_cast<int64_t>(step) * 3 * p.C) {
      s[0] += from[0];
      s[1] += from[p.C];
      s[2] += from[2 * p.C];
    }
  };
  float s[3];
  if (by_sample) {
    for (int b = j; b < q.samples; b += FINISH) {
      sums(b, 0, 1, s);
      write(b, s[0], s[1], s[2]);
    }
    part[0][j][lane] = dwp;
    part[1][j][lane] = dwn;
    __syncthreads();
    if (j != 0 || !live) return;
    dwp = dwn = 0.f;
    for (int k = 0; k < FINISH; ++k) {
      dwp += part[0][k][lane];
      dwn += part[1][k][lane];
    }
  } else {
    for (int b = 0; b < q.samples; ++b) {
      sums(b, j, FINISH, s);
#pragma unroll
      for (int i = 0; i < 3; ++i) part[i][j][lane] = s[i];
      __syncthreads();
      if (j == 0) {
        s[0] = s[1] = s[2] = 0.f;
        for (int k = 0; k < FINISH; ++k)
#pragma unroll
          for (int i = 0; i < 3; ++i) s[i] += part[i][k][lane];
        write(b, s[0], s[1], s[2]);
      }
      __syncthreads();
    }
    if (j != 0 || !live) return;
  }
  if (q.dpost_w) q.dpost_w[col] = dwp;
  if (q.dpre_w) q.dpre_w[col] = dwn;
}

// The weights' gradients from the CTAs' sums of a WHOLE launch.
__global__ void __launch_bounds__(32 * FINISH) finish_weights_kernel(const __grid_constant__ Params p, const __grid_constant__ Grads q, int count) {
  __shared__ float part[2][FINISH][33];
  const int lane = threadIdx.x, j = threadIdx.y, col = blockIdx.x * 32 + lane;
  pdl_wait();
  float a = 0.f, b = 0.f;
  if (col < p.C)
    for (int c = j; c < count; c += FINISH) {
      a += q.parts[static_cast<int64_t>(c) * 2 * p.C + col];
      b += q.parts[static_cast<int64_t>(c) * 2 * p.C + p.C + col];
    }
  part[0][j][lane] = a;
  part[1][j][lane] = b;
  __syncthreads();
  if (j != 0 || col >= p.C) return;
  a = b = 0.f;
  for (int k = 0; k < FINISH; ++k) {
    a += part[0][k][lane];
    b += part[1][k][lane];
  }
  if (q.dpost_w) q.dpost_w[col] = a;
  if (q.dpre_w) q.dpre_w[col] = b;
}

// How the backward pass shares out the rows.
struct Plan {
  int threads, groups, ctas, chunks;
  int64_t chunk_rows;
  bool whole;
  int64_t floats(int C) const { return static_cast<int64_t>(ctas) * (whole ? 2 : 3) * C; }
};
static Plan plan_backward(int64_t M, int64_t C, int64_t rows_per_mod) {
  Plan s{};
  const int chunks = static_cast<int>(C / 8);
  s.threads = (chunks + 31) / 32 * 32;
  s.groups = std::min(MAX_GROUPS, std::max(1, 512 / s.threads));
  const int64_t samples = M / rows_per_mod;
  const int per_sm = s.threads * s.groups <= 512 ? 2 : 1;
  const int64_t room = static_cast<int64_t>(sm_count()) * per_sm;
  s.whole = samples >= room;
  if (s.whole) {
    s.ctas = static_cast<int>(std::min<int64_t>(room, (samples + s.groups - 1) / s.groups));
    s.chunks = 1;
    s.chunk_rows = rows_per_mod;
  } else {
    const int64_t most = std::max<int64_t>(1, room / samples), rows = (rows_per_mod + most - 1) / most;
    s.chunk_rows = std::max<int64_t>(rows, std::min<int64_t>(s.groups, rows_per_mod));
    s.chunks = static_cast<int>((rows_per_mod + s.chunk_rows - 1) / s.chunk_rows);
    s.ctas = static_cast<int>(samples * s.chunks);
  }
  return s;
}

template <typename T, int NC, bool LAYER, int THREADS, int CTAS> static int forward_as(const Params& p, int threads, int groups, cudaStream_t st) {
  const int64_t need = (p.M + groups - 1) / groups, room = static_cast<int64_t>(sm_count()) * CTAS;
  return launch_kernel("sandwich norm", reinterpret_cast<const void*>(forward_kernel<T, NC, LAYER, THREADS, CTAS>), dim3((unsigned)std::min(need, room)),
                       dim3(threads, groups), 0, st, 1, false, p);
}
template <typename T, bool LAYER> static int forward(const Params& p, cudaStream_t st) {
  const int chunks = p.C / 8;
  if (chunks <= 64) {
    const int threads = (chunks + 31) / 32 * 32;
    return forward_as<T, 1, LAYER, 256, 4>(p, threads, std::min(MAX_GROUPS, 256 / threads), st);
  }
  const int threads = (chunks + 63) / 64 * 32;
  if (threads <= 384) return forward_as<T, 2, LAYER, 384, 2>(p, threads, std::min(MAX_GROUPS, 384 / threads), st);
  return forward_as<T, 2, LAYER, 1024, 1>(p, threads, 1, st);
}

template <typename T, bool LAYER, bool WHOLE, int THREADS> static int backward_as(const Params& p, const Grads& q, const Plan& s, cudaStream_t st) {
  const size_t smem = s.groups > 1 ? (size_t)(WHOLE ? 2 : 3) * p.C * 4 : 0;
  return launch_kernel("sandwich norm gradient", reinterpret_cast<const void*>(backward_kernel<T, LAYER, WHOLE, THREADS>), dim3((unsigned)s.ctas), dim3(s.threads, s.groups),
                       smem, st, 1, false, p, q);
}
template <typename T, bool LAYER, bool WHOLE> static int backward_of(const Params& p, const Grads& q, const Plan& s, cudaStream_t st) {
  const int threads = s.threads * s.groups;
  if (threads <= 512) return backward_as<T, LAYER, WHOLE, 512>(p, q, s, st);
  if (threads <= 640) return backward_as<T, LAYER, WHOLE, 640>(p, q, s, st);
  return backward_as<T, LAYER, WHOLE, 1024>(p, q, s, st);
}
template <typename T> static int backward(const Params& p, const Grads& q, const Plan& s, bool layer, cudaStream_t st) {
  int rc;
  if (layer) rc = s.whole ? backward_of<T, true, true>(p, q, s, st) : backward_of<T, true, false>(p, q, s, st);
  else rc = s.whole ? backward_of<T, false, true>(p, q, s, st) : backward_of<T, false, false>(p, q, s, st);
  if (rc) return rc;
  const dim3 grid((unsigned)((p.C + 31) / 32)), block(32, FINISH);
  if (!s.whole) {
    if (!q.dgate && !q.dscale && !q.dshift && !q.dpost_w && !q.dpre_w) return 0;
    return launch_kernel("sandwich norm sums", reinterpret_cast<const void*>(finish_kernel<T>), grid, block, 0, st, 1, true, p, q);
  }
  if (!q.dpost_w && !q.dpre_w) return 0;
  return launch_kernel("sandwich norm sums", reinterpret_cast<const void*>(finish_weights_kernel), grid, block, 0, st, 1, true, p, q, s.ctas);
}

static int check(const Params& p, int dtype, int64_t C, int64_t mod_rows) {
  if (dtype != KSB_BF16 && dtype != KSB_FP16) return fail(KSB_ERR_INVALID, "dtype must be KSB_BF16 or KSB_FP16");
  if (p.M < 0 || C <= 0 || C % 8 != 0 || p.M > INT32_MAX) return fail(KSB_ERR_INVALID, "bad shape M=%lld C=%lld (C %% 8 == 0)", (long long)p.M, (long long)C);
  if (C > KSB_NORM_MAX_C) return fail(KSB_ERR_UNSUPPORTED, "C=%lld is above %d", (long long)C, KSB_NORM_MAX_C);
  if (mod_rows < 1 || (p.M > 0 && p.M % mod_rows != 0)) return fail(KSB_ERR_INVALID, "mod_rows must divide M");
  const bool strides = (p.M <= 1 || (p.ldx >= C && (!p.y || p.ldy >= C))) && p.ldx % 8 == 0 && p.ldy % 8 == 0 && p.gate_stride % 8 == 0 && p.scale_stride % 8 == 0 && p.shift_stride % 8 == 0;
  const bool aligned = aligned16(p.x) && aligned16(p.y) && aligned16(p.gate) && aligned16(p.scale) && aligned16(p.shift) && aligned16(p.post_w) && aligned16(p.pre_w) && aligned16(p.stats);
  if (!strides || !aligned) return fail(KSB_ERR_INVALID, "tensors must be 16-byte aligned, their rows multiples of 8 elements apart");
  if (p.M > 0 && !p.y && (p.gate || p.post_w)) return fail(KSB_ERR_INVALID, "gate and post_w belong to y");
  return 0;
}

}  // namespace norms
}  // namespace ksb

using namespace ksb;

static int norm_params(norms::Params& p, const ksb_sandwich_norm_args* a) {
  if (!a) return fail(KSB_ERR_INVALID, "null pointer");
  p.x = a->x; p.y = a->y; p.ldx = a->ldx; p.ldy = a->y ? a->ldy : 0; p.M = a->M; p.C = (int)a->C; p.eps = a->eps; p.a = a->residual_scale;
  p.gate = a->gate; p.scale = a->scale; p.shift = a->shift;
  p.gate_stride = a->gate_stride; p.scale_stride = a->scale_stride; p.shift_stride = a->shift_stride;
  p.post_w = a->post_w; p.pre_w = a->pre_w; p.stats = reinterpret_cast<float4*>(a->stats);
  if (int rc = norms::check(p, a->dtype, a->C, a->mod_rows)) return rc;
  p.rows_per_mod = p.M > 0 ? p.M / a->mod_rows : 1;
  return 0;
}

extern "C" int ksb_sandwich_norm(const ksb_sandwich_norm_args* a, void* r, void* h, ksb_stream_t stream) {
  norms::Params p{};
  if (int rc = norm_params(p, a)) return rc;
  if (p.M == 0) return 0;
  if (!p.x || (p.y && !r) || (!p.y && !h) || !aligned16(r) || !aligned16(h)) return fail(KSB_ERR_INVALID, "null or unaligned pointer");
  if (!h && (p.scale || p.shift || p.pre_w)) return fail(KSB_ERR_INVALID, "scale, shift and pre_w belong to h");
  p.r = r; p.h = h;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  int rc;
  if (a->dtype == KSB_BF16) rc = a->layer ? norms::forward<__nv_bfloat16, true>(p, st) : norms::forward<__nv_bfloat16, false>(p, st);
  else rc = a->layer ? norms::forward<__half, true>(p, st) : norms::forward<__half, false>(p, st);
  return rc ? rc : 1;
}

extern "C" int64_t ksb_sandwich_norm_workspace(int64_t M, int64_t C, int64_t mod_rows) {
  if (M <= 0 || C <= 0 || C % 8 != 0 || C > KSB_NORM_MAX_C || mod_rows < 1 || M % mod_rows != 0) return 0;
  return norms::plan_backward(M, C, M / mod_rows).floats((int)C) * 4;
}

extern "C" int ksb_sandwich_norm_backward(const ksb_sandwich_norm_args* a, const ksb_sandwich_norm_grads* g, void* workspace, ksb_stream_t stream) {
  norms::Params p{};
  if (int rc = norm_params(p, a)) return rc;
  if (!g) return fail(KSB_ERR_INVALID, "null pointer");
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (p.M == 0) {  // sums over no rows
    if ((g->dpost_w && cudaMemsetAsync(g->dpost_w, 0, p.C * 4, st) != cudaSuccess) || (g->dpre_w && cudaMemsetAsync(g->dpre_w, 0, p.C * 4, st) != cudaSuccess))
      return fail(KSB_ERR_CUDA, "cannot clear the sums");
    for (void* m : {g->dgate, g->dscale, g->dshift})
      if (m && cudaMemsetAsync(m, 0, (size_t)a->mod_rows * p.C * 2, st) != cudaSuccess) return fail(KSB_ERR_CUDA, "cannot clear the sums");
    return 0;
  }
  norms::Grads q{};
  q.dr = g->dr; q.dh = g->dh; q.lddr = g->dr ? g->lddr : 0; q.lddh = g->dh ? g->lddh : 0;
  q.dx = g->dx; q.dy = g->dy; q.dgate = g->dgate; q.dscale = g->dscale; q.dshift = g->dshift; q.dpost_w = g->dpost_w; q.dpre_w = g->dpre_w;
  q.parts = static_cast<float*>(workspace);
  if (!p.x || !p.stats || !workspace || (!q.dr && !q.dh)) return fail(KSB_ERR_INVALID, "null pointer");
  for (const void* t : {q.dr, q.dh, (const void*)q.dx, (const void*)q.dy, (const void*)q.dgate, (const void*)q.dscale, (const void*)q.dshift, (const void*)workspace})
    if (!aligned16(t)) return fail(KSB_ERR_INVALID, "unaligned pointer");
  if (q.lddr % 8 != 0 || q.lddh % 8 != 0 || (p.M > 1 && ((q.dr && q.lddr < p.C) || (q.dh && q.lddh < p.C)))) return fail(KSB_ERR_INVALID, "rows of dr and dh must be multiples of 8 elements apart");
  if (!p.y && (q.dy || q.dgate || q.dpost_w)) return fail(KSB_ERR_INVALID, "dy, dgate and dpost_w belong to y");
  if (!q.dh && (q.dscale || q.dshift || q.dpre_w)) return fail(KSB_ERR_INVALID, "dscale, dshift and dpre_w belong to dh");
  const norms::Plan s = norms::plan_backward(p.M, p.C, p.rows_per_mod);
  q.chunk_rows = s.chunk_rows;
  q.chunks = s.chunks;
  q.samples = (int)a->mod_rows;
  const int before = launch_count();
  if (int rc = a->dtype == KSB_BF16 ? norms::backward<__nv_bfloat16>(p, q, s, a->layer != 0, st) : norms::backward<__half>(p, q, s, a->layer != 0, st)) return rc;
  return launch_count() - before;
}
