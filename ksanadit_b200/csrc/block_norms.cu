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
// Columns are taken in chunks of 8 (one 128-bit access per tensor).  A row is owned by a group of warps whose threads hold one chunk or
// two, always the same columns, so that what the modulation and the weights make of them stays in registers as long as the modulation
// row does.  A thread copies what it will read itself (cp.async) some rows ahead into a ring in shared memory: HBM is kept busy
// through the exchanges of a row's sums, of which there are two to four, one after the other.
//
// Measured (bf16, RMS): forward 2 x 32760 x 1536 134 us (6.0 TB/s), 75600 x 5120 485 us (6.4 TB/s); backward 242 us (5.0) and 889 us (5.2 TB/s: without
// the barrier of a row's exchange, as a probe, 762; two exchanges, other numbers of warps and chunks, a barrier in two halves were slower).  One
// row 6 us, all of it launch.
#include <algorithm>

#include "../../include/ksana_b200.h"
#include "common.cuh"
#include "host_utils.h"

namespace ksb {
namespace norms {

// Rows of the backward pass's ring.  Of 5120 columns, three and four: 30000 rows 401 and 369 us, layer norm 380 and 396.
template <int NC, bool LAYER> constexpr int backward_depth = NC == 4 ? 2 : LAYER ? 3 : 4;
template <int NC> constexpr int backward_threads = NC == 4 ? 256 : 640;  // of a CTA, one per SM

struct Params {
  const void* x;
  const void* y;  // null: r = x
  int64_t ldx, ldy;
  int M, C;
  float eps, a;
  // modulation row of row m: rows m / rows_per_mod, `stride` elements apart; each may be null
  const void* gate;
  const void* scale;
  const void* shift;
  int64_t gate_stride, scale_stride, shift_stride;
  int rows_per_mod;
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
  int chunk_rows;
  int chunks;      // of the rows that share a modulation row
  int samples;     // modulation rows
  int one_row;     // KSB_NORM_ONE_*: gradients that are sums over all rows, of tensors with one row beside others that have several
};
// Whether a launch has sums over all rows to make, besides those over a modulation row's.
__host__ __device__ __forceinline__ bool sums_all(const Grads& q) {
  return q.dpost_w || q.dpre_w || ((q.one_row & KSB_NORM_ONE_GATE) && q.dgate) || ((q.one_row & KSB_NORM_ONE_SCALE) && q.dscale) || ((q.one_row & KSB_NORM_ONE_SHIFT) && q.dshift);
}

__device__ __forceinline__ uint4 load8(const void* base, int64_t offset_bytes) { return *reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(base) + offset_bytes); }

// Two fp32 numbers in one register pair; one instruction works on both (backward pass of 75600 x 5120: 0.8 % less than one by one).
typedef unsigned long long F2;
__device__ __forceinline__ F2 pair(float x, float y) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ F2 both(float x) { return pair(x, x); }
__device__ __forceinline__ float2 split(F2 v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ F2 add(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ F2 mul(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ float total(F2 v) {
  const float2 f = split(v);
  return f.x + f.y;
}
// a thread's chunk: eight columns
struct V8 {
  F2 v[4];
  __device__ __forceinline__ F2& operator[](int i) { return v[i]; }
  __device__ __forceinline__ const F2& operator[](int i) const { return v[i]; }
};
__device__ __forceinline__ V8 fill8(float x) { return {both(x), both(x), both(x), both(x)}; }

template <typename T> __device__ __forceinline__ V8 unpack8(const uint4& v) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  V8 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 p = HalfOps<T>::unpack2(w[i]);
    r[i] = pair(p.x, p.y);
  }
  return r;
}
template <typename T> __device__ __forceinline__ uint4 pack8(const V8& f) {
  return make_uint4(HalfOps<T>::pack2(split(f[0])), HalfOps<T>::pack2(split(f[1])), HalfOps<T>::pack2(split(f[2])), HalfOps<T>::pack2(split(f[3])));
}
__device__ __forceinline__ V8 weight8(const float* w, int c) {
  if (!w) return fill8(1.f);
  const float4 a = *reinterpret_cast<const float4*>(w + c * 8), b = *reinterpret_cast<const float4*>(w + c * 8 + 4);
  return {pair(a.x, a.y), pair(a.z, a.w), pair(b.x, b.y), pair(b.z, b.w)};
}
// A = a gate wp of chunk c
template <typename T> __device__ __forceinline__ V8 post_factor(const Params& p, int64_t mod, int c) {
  V8 f = weight8(p.post_w, c);
  const F2 a = both(p.a);
  if (p.gate) {
    const V8 g = unpack8<T>(load8(p.gate, (mod * p.gate_stride + c * 8) * 2));
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = mul(f[i], mul(a, g[i]));
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = mul(f[i], a);
  }
  return f;
}
// B = (1 + scale) wn of chunk c
template <typename T> __device__ __forceinline__ V8 pre_factor(const Params& p, int64_t mod, int c) {
  V8 f = weight8(p.pre_w, c);
  if (p.scale) {
    const V8 s = unpack8<T>(load8(p.scale, (mod * p.scale_stride + c * 8) * 2));
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = mul(f[i], add(both(1.f), s[i]));
  }
  return f;
}

__device__ __forceinline__ void copy8(uint32_t dst, const void* base, int64_t offset_bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(static_cast<const uint8_t*>(base) + offset_bytes) : "memory");
}
// Where every row has a modulation row of its own, the L2 asks for it with the row's copies, some rows ahead of its use.  us without and with:
// forward 75600 x 1 x 1536 397 and 355, 32760 x 1 x 5120 609 and 583 (1560 rows, which lie in the L2: 35.7 and 38.0, so of many rows only);
// backward 747 and 669, 1172 and 1066, 97.8 and 93.5.
__device__ __forceinline__ void ask_for(const void* base, int64_t offset_bytes) {
  if (base) asm volatile("prefetch.global.L2 [%0];" ::"l"(static_cast<const uint8_t*>(base) + offset_bytes));
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// A group of warps that owns a row: sums over its threads.  Each of a row's sums has its own place, and rows take turns between two
// sets of places, so that one barrier per exchange is enough.  The places behind the last warp's hold zeros.
constexpr int PLACES = 8;
constexpr int RED_FLOATS = 2 * PLACES * 64;  // groups x warps, in fours, are at most 64
// Every lane's v, all the same, for the compiler to know it: counts and addresses then leave the vector registers, and branches take one
// instruction.  It is asked for (of the rows' counts, of the warps') where it gained.  us without and with: forward 30000 x 1536 70.9 and 65.0, x 4096
// 169 and 155, 5000 x 5120 40.9 and 37.7, 75600 x 768 95 and 87, x 2056 232 and 213, x 4616 504 and 470, layer norm 2 x 32760 x 5120 646 and 582.  RMS norms
// by CTAs of all 320 threads whose lanes all have columns come to the copy's rate without it, and with many rows lose a tenth: 75600 x 5120 483 and 530,
// x 2560 244 and 277, x 1024 106 and 116; so much from some 25000 rows of 1024 columns, 16000 of 2560, 11000 of 5120.  (After a tenth of a second
// of nothing but such calls the two forms change places at 75600 x 5120, 531 and 490; the cause is not known.)
// Backward: four chunks, 20000 x 8192 442 and 365, 75600 x 1 x 1536 877 and 744, layer norm 2 x 32760 x 5120 875 and (of the warps alone) 832; but
// 75600 x 5120 889 and 1081, 30000 x 1536 123 and 134.
template <bool ASKED> __device__ __forceinline__ int uniform(int v) { return ASKED ? __shfl_sync(0xffffffffu, v, 0) : v; }

template <bool UNIFORM> struct Group {
  float* red;  // [2][PLACES][warps, in fours]
  int id, warps, warp, lane, par;
  __device__ __forceinline__ Group(float* all, int group, int threads, int t)
      : id(uniform<UNIFORM>(group)), warps(threads / 32), warp(uniform<UNIFORM>(t >> 5)), lane(t & 31), par(0) {
    red = all + id * 2 * PLACES * four();
    if (warps > 1)
      for (int i = t; i < 2 * PLACES * four(); i += threads) red[i] = 0.f;
    barrier();
  }
  __device__ __forceinline__ int four() const { return (warps + 3) / 4 * 4; }
  __device__ __forceinline__ void barrier() const {
    if (warps > 1) asm volatile("bar.sync %0, %1;" ::"r"(id + 1), "r"(warps * 32) : "memory");
  }
  __device__ __forceinline__ float collect(const float* at) const {
    float v = 0.f;
#pragma unroll
    for (int i = 0; i < 5; ++i)  // at most 20 warps
      if (i * 4 < warps) {
        const float4 f = reinterpret_cast<const float4*>(at)[i];
        v += (f.x + f.y) + (f.z + f.w);
      }
    return v;
  }
  __device__ __forceinline__ float sum(float v, int place) const {
    v = warp_sum(v);
    if (warps == 1) return v;
    float* at = red + (par * PLACES + place) * four();
    if (lane == 0) at[warp] = v;
    barrier();
    return collect(at);
  }
  // N sums in one exchange.  Of eight, lanes first share out the sums and only then add up one each, the warps' sums as well: 9 and 2 shuffles
  // instead of 40, and 5 loads instead of 40 (32760 x 2 x 5120: a seventh less).  Of three that would only lengthen the way (75600 x 5120: a quarter more).
  template <int N> __device__ __forceinline__ void sums(float (&v)[N]) const {
    constexpr bool SHARED_OUT = N == 8;
    if (SHARED_OUT) {
      int off = 16;
#pragma unroll
      for (int n = 4; n > 0; n /= 2, off /= 2) {
        const bool upper = lane & off;
#pragma unroll
        for (int i = 0; i < n; ++i) {
          const float keep = upper ? v[i + n] : v[i], give = upper ? v[i] : v[i + n];
          v[i] = keep + __shfl_xor_sync(0xffffffffu, give, off);
        }
      }
#pragma unroll
      for (int o = 2; o > 0; o /= 2) v[0] += __shfl_xor_sync(0xffffffffu, v[0], o);
    } else {
#pragma unroll
      for (int o = 16; o > 0; o /= 2)
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
    }
    if (warps > 1) {
      float* at = red + par * PLACES * four();
      if (SHARED_OUT) {
        if ((lane & 3) == 0) at[(lane >> 2) * four() + warp] = v[0];
      } else if (lane == 0) {
#pragma unroll
        for (int i = 0; i < N; ++i) at[i * four() + warp] = v[i];
      }
      barrier();
      if (SHARED_OUT) {
        v[0] = 0.f;
#pragma unroll
        for (int w = 0; w < 20; w += 4)
          if (w < four()) v[0] += at[(lane >> 2) * four() + w + (lane & 3)];
#pragma unroll
        for (int o = 2; o > 0; o /= 2) v[0] += __shfl_xor_sync(0xffffffffu, v[0], o);
      } else {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = collect(at + i * four());
      }
    }
    if (SHARED_OUT) {
      const float mine = v[0];
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = __shfl_sync(0xffffffffu, mine, i * 4);
    }
  }
};

// 1 / std of a row of which this thread holds NC chunks, and the row's mean; `chunk`(c) gives chunk c (zeros where there is none)
template <int NC, bool LAYER, typename Of, typename Chunk>
__device__ __forceinline__ float2 row_stats(Of& g, const Chunk& chunk, const bool (&live)[NC], float inv_c, float eps, int place) {
  float mean = 0.f;
  if (LAYER) {
    F2 s = both(0.f);
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const V8 f = chunk(c);
#pragma unroll
      for (int i = 0; i < 4; ++i) s = add(s, f[i]);
    }
    mean = g.sum(total(s), place) * inv_c;
  }
  F2 s = both(0.f);
  const F2 minus = both(-mean);
#pragma unroll
  for (int c = 0; c < NC; ++c)
    if (live[c]) {
      const V8 f = chunk(c);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const F2 d = LAYER ? add(f[i], minus) : f[i];
        s = fma2(d, d, s);
      }
    }
  return make_float2(mean, rsqrtf(g.sum(total(s), place + 1) * inv_c + eps));
}

constexpr int FORWARD_DEPTH = 4;
template <typename T, int NC, bool LAYER, int THREADS, int CTAS, bool UNIFORM, bool APART>
__global__ void __launch_bounds__(THREADS, CTAS) forward_kernel(const __grid_constant__ Params p) {
  extern __shared__ __align__(16) uint8_t ring_bytes[];  // [FORWARD_DEPTH][x, y][NC][threads] 16 bytes
  __shared__ __align__(16) float red[RED_FLOATS];
  constexpr int DEPTH = FORWARD_DEPTH;
  const int t = threadIdx.x, nt = blockDim.x, chunks = p.C / 8, all = nt * blockDim.y;
  const int y = uniform<UNIFORM>(threadIdx.y);
  Group<UNIFORM> g(red, y, nt, t);
  const float inv_c = 1.f / static_cast<float>(p.C);
  bool live[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c) live[c] = t + c * nt < chunks;
  const int step = gridDim.x * blockDim.y;  // rows are below 2^31, and so is a row and DEPTH steps: see the launch
  const uint32_t mine = smem_u32(ring_bytes) + (y * nt + t) * 16;
  int ahead = blockIdx.x * blockDim.y + y;
  auto fetch = [&](int slot) {
    if (ahead < p.M) {
#pragma unroll
      for (int c = 0; c < NC; ++c)
        if (live[c]) {
          copy8(mine + ((slot * 2) * NC + c) * all * 16, p.x, (static_cast<int64_t>(ahead) * p.ldx + (t + c * nt) * 8) * 2);
          if (p.y) copy8(mine + ((slot * 2 + 1) * NC + c) * all * 16, p.y, (static_cast<int64_t>(ahead) * p.ldy + (t + c * nt) * 8) * 2);
          if (APART) {
            ask_for(p.gate, (ahead * p.gate_stride + (t + c * nt) * 8) * 2);
            ask_for(p.scale, (ahead * p.scale_stride + (t + c * nt) * 8) * 2);
            ask_for(p.shift, (ahead * p.shift_stride + (t + c * nt) * 8) * 2);
          }
        }
    }
    ahead += step;
    copies_commit();
  };
  int row = ahead;
  pdl_wait();  // whatever ran ahead, the caller's kernels too
  pdl_release();
#pragma unroll
  for (int d = 0; d < DEPTH - 1; ++d) fetch(d);
  V8 A[NC], B[NC];
  uint4 S[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    S[c] = make_uint4(0, 0, 0, 0);
    A[c] = B[c] = fill8(0.f);
  }
  int mod_end = 0, slot = 0;
  for (; row < p.M; row += step, g.par ^= 1) {
    if (row >= mod_end) {
      const int mod = row / p.rows_per_mod;
      mod_end = (mod + 1) * p.rows_per_mod;
#pragma unroll
      for (int c = 0; c < NC; ++c)
        if (live[c]) {
          if (p.y) A[c] = post_factor<T>(p, mod, t + c * nt);
          if (p.h) {
            B[c] = pre_factor<T>(p, mod, t + c * nt);
            if (p.shift) S[c] = load8(p.shift, (mod * p.shift_stride + (t + c * nt) * 8) * 2);
          }
        }
    }
    copies_wait<DEPTH - 2>();
    // as halves for as long as that will do: registers are what limits the rows in flight
    uint4 vx[NC], vy[NC];
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      vx[c] = vy[c] = make_uint4(0, 0, 0, 0);
      if (live[c]) {
        vx[c] = ld_shared_v4(mine + ((slot * 2) * NC + c) * all * 16);
        if (p.y) vy[c] = ld_shared_v4(mine + ((slot * 2 + 1) * NC + c) * all * 16);
      }
    }
    fetch(slot == 0 ? DEPTH - 1 : slot - 1);  // the slot that was read one row ago
    if (++slot == DEPTH) slot = 0;
    float4 st = make_float4(0.f, 0.f, 0.f, 0.f);
    V8 x[NC];
    if (p.y) {
      const float2 s = row_stats<NC, LAYER>(g, [&](int c) { return unpack8<T>(vy[c]); }, live, inv_c, p.eps, 0);
      st.x = s.x;
      st.y = s.y;
      const F2 minus = both(-s.x), rstd = both(s.y);
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const V8 y = unpack8<T>(vy[c]);
        x[c] = unpack8<T>(vx[c]);
#pragma unroll
        for (int i = 0; i < 4; ++i) x[c][i] = fma2(A[c][i], mul(LAYER ? add(y[i], minus) : y[i], rstd), x[c][i]);
        if (live[c]) *reinterpret_cast<uint4*>(static_cast<T*>(p.r) + static_cast<int64_t>(row) * p.C + (t + c * nt) * 8) = pack8<T>(x[c]);
      }
    } else {
#pragma unroll
      for (int c = 0; c < NC; ++c) x[c] = unpack8<T>(vx[c]);
    }
    if (p.h) {
      const float2 s = row_stats<NC, LAYER>(g, [&](int c) { return x[c]; }, live, inv_c, p.eps, 2);
      st.z = s.x;
      st.w = s.y;
      const F2 minus = both(-s.x), rstd = both(s.y);
#pragma unroll
      for (int c = 0; c < NC; ++c)
        if (live[c]) {
          V8 o = unpack8<T>(S[c]);
#pragma unroll
          for (int i = 0; i < 4; ++i) o[i] = fma2(mul(LAYER ? add(x[c][i], minus) : x[c][i], rstd), B[c][i], o[i]);
          *reinterpret_cast<uint4*>(static_cast<T*>(p.h) + static_cast<int64_t>(row) * p.C + (t + c * nt) * 8) = pack8<T>(o);
        }
    }
    if (p.stats && t == 0) p.stats[row] = st;
  }
}

// Sums over rows that a thread keeps for a chunk: of D yh, dh rh and dh.
struct Sums {
  V8 p, q, s;
};

// NC chunks per thread.  WHOLE: a group takes all rows of some modulation rows, and writes the modulation's gradients itself; else a CTA takes
// a stretch of the rows of one and leaves its sums to finish_kernel.  ONE (WHOLE): some of gate, scale and shift have one row for all (a form of its
// own, since the other one lost 1 - 2 % to the questions: 32760 x 1 x 5120 1050 and 1063 us, layer norm 20000 x 1 x 8192 1784 and 1814).
//
// With w = dr + rstd_r t and z = A yh, D = w - a1 rh - a0 is linear in its row's a1 = rstd_r mean(t rh) and a0 = rstd_r mean(t), and so are the sums
// that dy takes: sum(e yh) = sum(w z) - a1 sum(rh z) - a0 sum(z), sum(e) = sum(w A) - a1 sum(rh A) - a0 sum(A).  So a row has one exchange, of
// three sums for RMS norms (a0 = 0) and of eight for layer norms, instead of two, one after the other.
//
// Up to 5120 columns a thread has one chunk and up to twenty warps share a row: eight warps of three chunks, which leaves the exchanges less to do
// but the schedulers two warps each, took 15 % longer for 75600 x 5120 than twenty of one (889 us now), twelve of two 17 %.  NC = 4 with WHOLE has 240 - 376
// bytes of spills at 255 registers: 20000 x 1 x 8192 1745 us, layer norm 1784.
template <typename T, int NC, bool LAYER, bool WHOLE, bool ONE>
__global__ void __launch_bounds__(backward_threads<NC>, 1) backward_kernel(const __grid_constant__ Params p, const __grid_constant__ Grads q) {
  extern __shared__ __align__(16) uint8_t ring_bytes[];  // [DEPTH][x, y, dr, dh][NC][threads] 16 bytes and the factors; in the end the groups' sums
  __shared__ __align__(16) float red[RED_FLOATS];
  constexpr int DEPTH = backward_depth<NC, LAYER>;
  const int t = threadIdx.x, nt = blockDim.x, all = nt * blockDim.y;
  constexpr bool ROWS = NC == 4 || WHOLE, WARPS = LAYER && !ROWS;
  const int y = uniform<WARPS>(threadIdx.y), group_row = uniform<ROWS>(threadIdx.y);
  Group<WARPS> g(red, y, nt, t);
  const float inv_c = 1.f / static_cast<float>(p.C);
  bool live[NC];
  Sums acc[NC];
  V8 wp[NC], wn[NC];  // WHOLE: of the weights' gradients
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    live[c] = t + c * nt < p.C / 8;
    acc[c].p = acc[c].q = acc[c].s = wp[c] = wn[c] = fill8(0.f);
  }

  // the group's rows: row, row + step, .. below end
  int row, step, end;
  if (WHOLE) {
    const int64_t groups = static_cast<int64_t>(gridDim.x) * blockDim.y, id = static_cast<int64_t>(blockIdx.x) * blockDim.y + group_row;
    row = static_cast<int>(q.samples * id / groups) * p.rows_per_mod;
    end = static_cast<int>(q.samples * (id + 1) / groups) * p.rows_per_mod;
    step = 1;
  } else {
    const int b = blockIdx.x / q.chunks, of = b * p.rows_per_mod, from = of + (blockIdx.x - b * q.chunks) * q.chunk_rows;
    end = min(from + q.chunk_rows, of + p.rows_per_mod);
    row = from + group_row;
    step = blockDim.y;
  }
  const uint32_t mine = smem_u32(ring_bytes) + (y * nt + t) * 16;
  auto place = [&](int slot, int which, int c) { return mine + ((slot * 4 + which) * NC + c) * all * 16; };
  int ahead = row;
  auto fetch = [&](int slot) {
    if (ahead < end) {
      const int64_t at = ahead;
      const uint8_t* px = static_cast<const uint8_t*>(p.x) + (at * p.ldx + t * 8) * 2;
      const uint8_t* py = static_cast<const uint8_t*>(p.y) + (at * p.ldy + t * 8) * 2;
      const uint8_t* pr = static_cast<const uint8_t*>(q.dr) + (at * q.lddr + t * 8) * 2;
      const uint8_t* ph = static_cast<const uint8_t*>(q.dh) + (at * q.lddh + t * 8) * 2;
#pragma unroll
      for (int c = 0; c < NC; ++c)
        if (live[c]) {
          copy8(place(slot, 0, c), px, c * nt * 16);
          if (p.y) copy8(place(slot, 1, c), py, c * nt * 16);
          if (q.dr) copy8(place(slot, 2, c), pr, c * nt * 16);
          if (q.dh) copy8(place(slot, 3, c), ph, c * nt * 16);
          if (WHOLE && p.rows_per_mod == 1) {
            ask_for(p.gate, (at * p.gate_stride + (t + c * nt) * 8) * 2);
            ask_for(p.scale, (at * p.scale_stride + (t + c * nt) * 8) * 2);
          }
        }
    }
    ahead += step;
    copies_commit();
  };
  pdl_wait();
  pdl_release();
#pragma unroll
  for (int d = 0; d < DEPTH - 1; ++d) fetch(d);
  float4 next_st = row < end ? p.stats[row] : make_float4(0.f, 0.f, 0.f, 0.f);
  int mod = row / p.rows_per_mod, mod_end = 0;
  // A and B wait in shared memory
  auto factor_at = [&](int which, int c, int i) { return place(DEPTH, which * 2 + i, c); };
  auto put_factor = [&](int which, int c, const V8& f) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
      asm volatile("st.shared.v2.b64 [%0], {%1, %2};" ::"r"(factor_at(which, c, i)), "l"(f[2 * i]), "l"(f[2 * i + 1]) : "memory");
  };
  auto factor = [&](int which, int c) {
    V8 f;
#pragma unroll
    for (int i = 0; i < 2; ++i)
      asm volatile("ld.shared.v2.b64 {%0, %1}, [%2];" : "=l"(f[2 * i]), "=l"(f[2 * i + 1]) : "r"(factor_at(which, c, i)) : "memory");
    return f;
  };
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    put_factor(0, c, fill8(0.f));
    put_factor(1, c, fill8(0.f));
  }
  // WHOLE: a modulation row's gradients, and its part of the weights'.  What a tensor with one row takes (acc.p: the gate and the weight
  // behind it, acc.q: the scale and the weight ahead, acc.s: the shift) runs on instead, through all rows.
  const bool one_gate = ONE && q.one_row & KSB_NORM_ONE_GATE, one_scale = ONE && q.one_row & KSB_NORM_ONE_SCALE, one_shift = ONE && q.one_row & KSB_NORM_ONE_SHIFT;
  auto flush = [&]() {
    const F2 a = both(p.a);
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      if (live[c]) {
        const int ch = t + c * nt;
        V8 f, o;
        auto out = [&](void* to) { *reinterpret_cast<uint4*>(static_cast<T*>(to) + static_cast<int64_t>(mod) * p.C + ch * 8) = pack8<T>(o); };
        if (p.y && !one_gate) {
          if (q.dpost_w) {
            f = p.gate ? unpack8<T>(load8(p.gate, (mod * p.gate_stride + ch * 8) * 2)) : fill8(1.f);
#pragma unroll
            for (int i = 0; i < 4; ++i) wp[c][i] = fma2(mul(a, f[i]), acc[c].p[i], wp[c][i]);
          }
          if (q.dgate) {
            f = weight8(p.post_w, ch);
#pragma unroll
            for (int i = 0; i < 4; ++i) o[i] = mul(mul(a, f[i]), acc[c].p[i]);
            out(q.dgate);
          }
        }
        if (q.dh) {
          if (q.dpre_w && !one_scale) {
            f = p.scale ? unpack8<T>(load8(p.scale, (mod * p.scale_stride + ch * 8) * 2)) : fill8(0.f);
#pragma unroll
            for (int i = 0; i < 4; ++i) wn[c][i] = fma2(add(both(1.f), f[i]), acc[c].q[i], wn[c][i]);
          }
          if (q.dscale && !one_scale) {
            f = weight8(p.pre_w, ch);
#pragma unroll
            for (int i = 0; i < 4; ++i) o[i] = mul(f[i], acc[c].q[i]);
            out(q.dscale);
          }
          if (q.dshift && !one_shift) {
            o = acc[c].s;
            out(q.dshift);
          }
        }
      }
      if (!one_gate) acc[c].p = fill8(0.f);
      if (!one_scale) acc[c].q = fill8(0.f);
      if (!one_shift) acc[c].s = fill8(0.f);
    }
  };
  int slot = 0;
  for (; row < end; row += step, g.par ^= 1) {
    if (row >= mod_end) {
      if (WHOLE && mod_end != 0) {
        flush();
        ++mod;
      }
      mod_end = (mod + 1) * p.rows_per_mod;
#pragma unroll
      for (int c = 0; c < NC; ++c)
        if (live[c]) {
          if (p.y) put_factor(0, c, post_factor<T>(p, mod, t + c * nt));
          if (q.dh) put_factor(1, c, pre_factor<T>(p, mod, t + c * nt));
        }
    }
    const float4 st = next_st;
    if (row + step < end) next_st = p.stats[row + step];
    copies_wait<DEPTH - 2>();
    const uint4 none = make_uint4(0, 0, 0, 0);
    const F2 y_minus = both(-st.x), y_rstd = both(st.y), r_minus = both(-st.z), r_rstd = both(st.w);
    V8 yh[NC], w[NC], rh[NC];
    constexpr int N = LAYER ? 8 : 3;
    float m[N];  // the sums of t rh, w z, rh z, (t, z, w A, rh A, A)
    F2 tr = both(0.f), wz = tr, rz = tr, ts = tr, zs = tr, wa = tr, ra = tr, as = tr;
    const uint32_t src = mine + slot * 4 * NC * all * 16;
    auto from = [&](int which, int c, bool there) { return unpack8<T>(live[c] && there ? ld_shared_v4(src + (which * NC + c) * all * 16) : none); };
    // the factors are read where they are used: held, they would push others out of the registers (75600 x 5120: 23 % more)
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      yh[c] = from(1, c, p.y != nullptr);
      w[c] = from(2, c, q.dr != nullptr);
      rh[c] = fill8(0.f);
      if (p.y) {
#pragma unroll
        for (int i = 0; i < 4; ++i) yh[c][i] = mul(LAYER ? add(yh[c][i], y_minus) : yh[c][i], y_rstd);
      }
      if (q.dh) {
        rh[c] = from(0, c, true);
        const V8 dh = from(3, c, true);
        V8 f = factor(0, c);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          rh[c][i] = fma2(f[i], yh[c][i], rh[c][i]);
          rh[c][i] = mul(LAYER ? add(rh[c][i], r_minus) : rh[c][i], r_rstd);
          acc[c].q[i] = fma2(dh[i], rh[c][i], acc[c].q[i]);
          acc[c].s[i] = add(acc[c].s[i], dh[i]);
        }
        f = factor(1, c);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const F2 tv = mul(dh[i], f[i]);
          tr = fma2(tv, rh[c][i], tr);
          if (LAYER) ts = add(ts, tv);
          w[c][i] = fma2(r_rstd, tv, w[c][i]);
        }
      }
    }
    fetch(slot == 0 ? DEPTH - 1 : slot - 1);  // the slot that was read one row ago
    if (++slot == DEPTH) slot = 0;
    if (p.y) {
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const V8 f = factor(0, c);  // zeros where there is no column
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const F2 z = mul(f[i], yh[c][i]);
          wz = fma2(w[c][i], z, wz);
          rz = fma2(rh[c][i], z, rz);
          if (LAYER) {
            zs = add(zs, z);
            wa = fma2(w[c][i], f[i], wa);
            ra = fma2(rh[c][i], f[i], ra);
            as = add(as, f[i]);
          }
        }
      }
    }
    m[0] = total(tr);
    m[1] = total(wz);
    m[2] = total(rz);
    if (LAYER) {
      m[N - 5] = total(ts);
      m[N - 4] = total(zs);
      m[N - 3] = total(wa);
      m[N - 2] = total(ra);
      m[N - 1] = total(as);
    }
    g.sums<N>(m);
    const float a1 = m[0] * inv_c * st.w, a0 = LAYER ? m[N - 5] * inv_c * st.w : 0.f;
    const float e1 = m[1] - a1 * m[2] - (LAYER ? a0 * m[N - 4] : 0.f), e0 = LAYER ? m[N - 3] - a1 * m[N - 2] - a0 * m[N - 1] : 0.f;
    const F2 xa1 = both(-a1), xa0 = both(-a0), xe1 = both(-e1 * inv_c), xe0 = both(-e0 * inv_c);
#pragma unroll
    for (int c = 0; c < NC; ++c) {
#pragma unroll
      for (int i = 0; i < 4; ++i) w[c][i] = fma2(rh[c][i], xa1, LAYER ? add(w[c][i], xa0) : w[c][i]);  // D
      const int64_t at = static_cast<int64_t>(row) * p.C + (t + c * nt) * 8;
      if (q.dx && live[c]) *reinterpret_cast<uint4*>(static_cast<T*>(q.dx) + at) = pack8<T>(w[c]);
      if (p.y) {
        const V8 A = factor(0, c);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          acc[c].p[i] = fma2(w[c][i], yh[c][i], acc[c].p[i]);
          w[c][i] = fma2(yh[c][i], xe1, mul(w[c][i], A[i]));
          w[c][i] = mul(y_rstd, LAYER ? add(w[c][i], xe0) : w[c][i]);
        }
        if (q.dy && live[c]) *reinterpret_cast<uint4*>(static_cast<T*>(q.dy) + at) = pack8<T>(w[c]);
      }
    }
  }
  if (WHOLE && mod_end != 0) flush();
  copies_wait<0>();

  // What is left to the second kernel: the groups' sums, added up in the order of the groups where there are several.
  constexpr int KINDS = WHOLE && !ONE ? 2 : 3;
  if (WHOLE && !sums_all(q)) return;
  float* to = q.parts + static_cast<int64_t>(blockIdx.x) * KINDS * p.C;
  float* sums = blockDim.y == 1 ? to : reinterpret_cast<float*>(ring_bytes);
  for (int y = 0; y < (int)blockDim.y; ++y) {
    if (blockDim.y > 1) __syncthreads();
    if (y != (int)threadIdx.y) continue;
#pragma unroll
    for (int c = 0; c < NC; ++c)
      if (live[c]) {
#pragma unroll
        for (int k = 0; k < KINDS; ++k) {
          const V8& v = WHOLE && !ONE ? (k == 0 ? wp[c] : wn[c]) : k == 0 ? (!WHOLE || one_gate ? acc[c].p : wp[c]) : k == 1 ? (!WHOLE || one_scale ? acc[c].q : wn[c]) : acc[c].s;
          F2* at = reinterpret_cast<F2*>(sums + k * p.C + (t + c * nt) * 8);
#pragma unroll
          for (int i = 0; i < 4; ++i) at[i] = y == 0 ? v[i] : add(at[i], v[i]);
        }
      }
  }
  if (blockDim.y == 1) return;
  __syncthreads();
  for (int i = threadIdx.y * nt + t; i < KINDS * p.C; i += all) to[i] = sums[i];
}

// Adds up the stretches' sums, in order: 32 columns per CTA, 16 threads per column, which take turns over the stretches of a
// modulation row, or over the modulation rows where there are many.  Without gradients of the weights, which are sums over all of them, the
// modulation rows have CTAs of their own (backward pass of 3 x 777 x 2056 25.0 and 22.4 us, of 8 x 777 x 2048 51.4 and 42.9).
constexpr int FINISH = 16;
template <typename T> __global__ void __launch_bounds__(32 * FINISH) finish_kernel(const __grid_constant__ Params p, const __grid_constant__ Grads q) {
  __shared__ float part[5][FINISH][33];
  const int lane = threadIdx.x, j = threadIdx.y, col = blockIdx.x * 32 + lane;
  const bool live = col < p.C;
  pdl_wait();
  pdl_release();
  const bool by_sample = q.samples >= FINISH;
  const float wp = p.post_w && live ? p.post_w[col] : 1.f, wn = p.pre_w && live ? p.pre_w[col] : 1.f;
  const bool one_gate = q.one_row & KSB_NORM_ONE_GATE, one_scale = q.one_row & KSB_NORM_ONE_SCALE, one_shift = q.one_row & KSB_NORM_ONE_SHIFT;
  float all[5] = {0.f, 0.f, 0.f, 0.f, 0.f};  // over all rows: of the two weights', and of gate, scale and shift where they have one row
  auto write = [&](int b, float sp, float sq, float ss) {
    if (!live) return;
    const float gate = p.gate ? HalfOps<T>::to_f(static_cast<const T*>(p.gate)[b * p.gate_stride + col]) : 1.f;
    const float scale = p.scale ? HalfOps<T>::to_f(static_cast<const T*>(p.scale)[b * p.scale_stride + col]) : 0.f;
    const int64_t at = static_cast<int64_t>(b) * p.C + col;
    if (q.dgate && !one_gate) static_cast<T*>(q.dgate)[at] = HalfOps<T>::from_f(p.a * wp * sp);
    if (q.dscale && !one_scale) static_cast<T*>(q.dscale)[at] = HalfOps<T>::from_f(wn * sq);
    if (q.dshift && !one_shift) static_cast<T*>(q.dshift)[at] = HalfOps<T>::from_f(ss);
    all[0] = fmaf(p.a * gate, sp, all[0]);
    all[1] = fmaf(1.f + scale, sq, all[1]);
    all[2] += sp;
    all[3] += sq;
    all[4] += ss;
  };
  auto sums = [&](int b, int first, int step, float (&s)[3]) {
    const float* from = q.parts + (static_cast<int64_t>(b) * q.chunks + first) * 3 * p.C + col;
    s[0] = s[1] = s[2] = 0.f;
    if (!live) return;
#pragma unroll 4
    for (int c = first; c < q.chunks; c += step, from += static_cast<int64_t>(step) * 3 * p.C) {
      s[0] += from[0];
      s[1] += from[p.C];
      s[2] += from[2 * p.C];
    }
  };
  float s[3];
  if (by_sample) {
    for (int b = blockIdx.y * FINISH + j; b < q.samples; b += gridDim.y * FINISH) {
      sums(b, 0, 1, s);
      write(b, s[0], s[1], s[2]);
    }
#pragma unroll
    for (int i = 0; i < 5; ++i) part[i][j][lane] = all[i];
    __syncthreads();
    if (j != 0 || !live) return;
#pragma unroll
    for (int i = 0; i < 5; ++i) all[i] = 0.f;
    for (int k = 0; k < FINISH; ++k)
#pragma unroll
      for (int i = 0; i < 5; ++i) all[i] += part[i][k][lane];
  } else {
    for (int b = blockIdx.y; b < q.samples; b += gridDim.y) {
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
  if (q.dpost_w) q.dpost_w[col] = all[0];
  if (q.dpre_w) q.dpre_w[col] = all[1];
  if (q.dgate && one_gate) static_cast<T*>(q.dgate)[col] = HalfOps<T>::from_f(p.a * wp * all[2]);
  if (q.dscale && one_scale) static_cast<T*>(q.dscale)[col] = HalfOps<T>::from_f(wn * all[3]);
  if (q.dshift && one_shift) static_cast<T*>(q.dshift)[col] = HalfOps<T>::from_f(all[4]);
}

// What is summed over all rows, from the CTAs' sums of a WHOLE launch (ONE: as there, a third sum among them).
template <typename T, bool ONE> __global__ void __launch_bounds__(32 * FINISH) finish_all_kernel(const __grid_constant__ Params p, const __grid_constant__ Grads q, int count) {
  constexpr int KINDS = ONE ? 3 : 2;
  __shared__ float part[KINDS][FINISH][33];
  const int lane = threadIdx.x, j = threadIdx.y, col = blockIdx.x * 32 + lane;
  pdl_wait();
  pdl_release();
  float v[KINDS];
#pragma unroll
  for (int k = 0; k < KINDS; ++k) v[k] = 0.f;
  if (col < p.C)
#pragma unroll 4
    for (int c = j; c < count; c += FINISH) {
      const float* from = q.parts + static_cast<int64_t>(c) * KINDS * p.C + col;
      v[0] += from[0];
      v[1] += from[p.C];
      if (ONE) v[KINDS - 1] += from[2 * p.C];
    }
#pragma unroll
  for (int k = 0; k < KINDS; ++k) part[k][j][lane] = v[k];
  __syncthreads();
  if (j != 0 || col >= p.C) return;
#pragma unroll
  for (int k = 0; k < KINDS; ++k) v[k] = 0.f;
#pragma unroll
  for (int i = 0; i < FINISH; ++i)
#pragma unroll
    for (int k = 0; k < KINDS; ++k) v[k] += part[k][i][lane];
  if constexpr (ONE) {  // a gate or scale with one row has waited until here: see flush
    const bool one_gate = q.one_row & KSB_NORM_ONE_GATE, one_scale = q.one_row & KSB_NORM_ONE_SCALE, one_shift = q.one_row & KSB_NORM_ONE_SHIFT;
    if (q.dgate && one_gate) static_cast<T*>(q.dgate)[col] = HalfOps<T>::from_f(p.a * (p.post_w ? p.post_w[col] : 1.f) * v[0]);
    if (q.dscale && one_scale) static_cast<T*>(q.dscale)[col] = HalfOps<T>::from_f((p.pre_w ? p.pre_w[col] : 1.f) * v[1]);
    if (q.dshift && one_shift) static_cast<T*>(q.dshift)[col] = HalfOps<T>::from_f(v[KINDS - 1]);
    if (one_gate) v[0] *= p.a * HalfOps<T>::to_f(static_cast<const T*>(p.gate)[col]);
    if (one_scale) v[1] *= 1.f + HalfOps<T>::to_f(static_cast<const T*>(p.scale)[col]);
  }
  if (q.dpost_w) q.dpost_w[col] = v[0];
  if (q.dpre_w) q.dpre_w[col] = v[1];
}

// How the backward pass shares out the rows: a CTA per SM, of as many groups as its threads hold.
struct Plan {
  int each, threads, groups, ctas, chunks;  // each: chunks per thread
  int64_t chunk_rows;
  bool whole;
  int64_t floats(int C) const { return static_cast<int64_t>(ctas) * 3 * C; }
};
static Plan plan_backward(int64_t M, int64_t C, int64_t rows_per_mod) {
  Plan s{};
  s.each = C <= 5120 ? 1 : 4;
  s.threads = static_cast<int>((C / 8 + 32 * s.each - 1) / (32 * s.each) * 32);
  s.groups = s.each == 4 ? 1 : std::min(15, backward_threads<1> / s.threads);  // a named barrier each
  const int64_t samples = M / rows_per_mod, room = sm_count();
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

template <typename T, int NC, bool LAYER, int THREADS, int CTAS, bool UNIFORM, bool APART> static int forward_kind(const Params& p, int threads, int groups, cudaStream_t st) {
  auto kernel = forward_kernel<T, NC, LAYER, THREADS, CTAS, UNIFORM, APART>;
  static DeviceOnce limit;
  if (int rc = limit.raise_smem(reinterpret_cast<const void*>(kernel), FORWARD_DEPTH * 2 * NC * THREADS * 16)) return rc;
  const int need = (p.M + groups - 1) / groups, room = sm_count() * CTAS;
  return launch_kernel("sandwich norm", reinterpret_cast<const void*>(kernel), dim3((unsigned)std::min(need, room)), dim3(threads, groups),
                       FORWARD_DEPTH * 2 * NC * threads * groups * 16, st, 1, true, p);
}
template <typename T, int NC, bool LAYER, int THREADS, int CTAS> static int forward_as(const Params& p, int threads, int groups, cudaStream_t st) {
  if (p.rows_per_mod == 1 && p.M > 4096 && (p.gate || p.scale || p.shift)) return forward_kind<T, NC, LAYER, THREADS, CTAS, true, true>(p, threads, groups, st);
  // see uniform; a 32nd of the lanes may be idle (75600 x 992 100 and 114 us, x 896 98 and 90)
  if (!LAYER && THREADS == 320 && groups * threads == 320 && p.C / 8 * 32 >= 31 * NC * threads && p.M > 16384)
    return forward_kind<T, NC, LAYER, THREADS, CTAS, LAYER || THREADS != 320, false>(p, threads, groups, st);
  return forward_kind<T, NC, LAYER, THREADS, CTAS, true, false>(p, threads, groups, st);
}
template <typename T, bool LAYER> static int forward(const Params& p, cudaStream_t st) {
  const int chunks = p.C / 8;
  if (chunks <= 64) {
    const int threads = (chunks + 31) / 32 * 32;
    return forward_as<T, 1, LAYER, 256, 4>(p, threads, 256 / threads, st);
  }
  const int threads = (chunks + 63) / 64 * 32;
  if (threads <= 320) return forward_as<T, 2, LAYER, 320, 2>(p, threads, 320 / threads, st);
  return forward_as<T, 2, LAYER, 512, 1>(p, threads, 1, st);
}

template <typename T, int NC, bool LAYER, bool WHOLE, bool ONE> static int backward_as(const Params& p, const Grads& q, const Plan& s, cudaStream_t st) {
  auto kernel = backward_kernel<T, NC, LAYER, WHOLE, ONE>;
  constexpr int bytes = (backward_depth<NC, LAYER> + 1) * 64 * NC;  // a thread: the ring, and the factors
  static DeviceOnce limit;
  if (int rc = limit.raise_smem(reinterpret_cast<const void*>(kernel), bytes * backward_threads<NC>)) return rc;
  return launch_kernel("sandwich norm gradient", reinterpret_cast<const void*>(kernel), dim3((unsigned)s.ctas), dim3(s.threads, s.groups), bytes * s.threads * s.groups, st, 1, true, p, q);
}
template <typename T, bool LAYER, bool WHOLE, bool ONE> static int backward_of(const Params& p, const Grads& q, const Plan& s, cudaStream_t st) {
  return s.each == 1 ? backward_as<T, 1, LAYER, WHOLE, ONE>(p, q, s, st) : backward_as<T, 4, LAYER, WHOLE, ONE>(p, q, s, st);
}
template <typename T, bool LAYER> static int backward_form(const Params& p, const Grads& q, const Plan& s, cudaStream_t st) {
  if (!s.whole) return backward_of<T, LAYER, false, false>(p, q, s, st);
  return q.one_row ? backward_of<T, LAYER, true, true>(p, q, s, st) : backward_of<T, LAYER, true, false>(p, q, s, st);
}
template <typename T> static int backward(const Params& p, const Grads& q, const Plan& s, bool layer, cudaStream_t st) {
  if (int rc = layer ? backward_form<T, true>(p, q, s, st) : backward_form<T, false>(p, q, s, st)) return rc;
  const dim3 grid((unsigned)((p.C + 31) / 32)), block(32, FINISH);
  if (!s.whole) {
    if (!q.dgate && !q.dscale && !q.dshift && !q.dpost_w && !q.dpre_w) return 0;
    const unsigned apart = sums_all(q) ? 1 : q.samples < FINISH ? q.samples : (q.samples + FINISH - 1) / FINISH;
    return launch_kernel("sandwich norm sums", reinterpret_cast<const void*>(finish_kernel<T>), dim3(grid.x, apart), block, 0, st, 1, true, p, q);
  }
  if (!sums_all(q)) return 0;
  return launch_kernel("sandwich norm sums", q.one_row ? reinterpret_cast<const void*>(finish_all_kernel<T, true>) : reinterpret_cast<const void*>(finish_all_kernel<T, false>), grid, block, 0, st, 1, true, p, q, s.ctas);
}

static int check(const Params& p, int dtype, int64_t C, int64_t mod_rows) {
  if (dtype != KSB_BF16 && dtype != KSB_FP16) return fail(KSB_ERR_INVALID, "dtype must be KSB_BF16 or KSB_FP16");
  if (C <= 0 || C % 8 != 0) return fail(KSB_ERR_INVALID, "bad shape M=%d C=%lld (C %% 8 == 0)", p.M, (long long)C);
  if (C > KSB_NORM_MAX_C) return fail(KSB_ERR_UNSUPPORTED, "C=%lld is above %d", (long long)C, KSB_NORM_MAX_C);
  if (mod_rows < 1 || (p.M > 0 && p.M % mod_rows != 0)) return fail(KSB_ERR_INVALID, "mod_rows must divide M");
  // the distance between rows of a tensor that has one row, or none, is nobody's
  const bool strides = (p.M <= 1 || (p.ldx >= C && (!p.y || p.ldy >= C) && p.ldx % 8 == 0 && p.ldy % 8 == 0)) && p.gate_stride % 8 == 0 && p.scale_stride % 8 == 0 && p.shift_stride % 8 == 0;
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
  p.x = a->x; p.y = a->y; p.ldx = a->ldx; p.ldy = a->y ? a->ldy : 0; p.C = (int)a->C; p.eps = a->eps; p.a = a->residual_scale;
  p.gate = a->gate; p.scale = a->scale; p.shift = a->shift;
  p.gate_stride = a->gate_stride; p.scale_stride = a->scale_stride; p.shift_stride = a->shift_stride;
  p.post_w = a->post_w; p.pre_w = a->pre_w; p.stats = reinterpret_cast<float4*>(a->stats);
  if (a->M < 0 || a->M > KSB_NORM_MAX_M) return fail(KSB_ERR_INVALID, "bad shape M=%lld", (long long)a->M);
  p.M = (int)a->M;
  if (int rc = norms::check(p, a->dtype, a->C, a->mod_rows)) return rc;
  p.rows_per_mod = p.M > 0 ? (int)(p.M / a->mod_rows) : 1;
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
  // one row of a tensor is all of its rows: what a call with a single modulation row does anyway
  const int one_row = a->mod_rows > 1 ? g->one_row : 0;
  if ((g->one_row & ~(KSB_NORM_ONE_GATE | KSB_NORM_ONE_SCALE | KSB_NORM_ONE_SHIFT)) != 0 || ((one_row & KSB_NORM_ONE_GATE) && (!p.gate || p.gate_stride != 0)) ||
      ((one_row & KSB_NORM_ONE_SCALE) && (!p.scale || p.scale_stride != 0)) || ((one_row & KSB_NORM_ONE_SHIFT) && (!p.shift || p.shift_stride != 0)))
    return fail(KSB_ERR_INVALID, "one_row names a tensor that is not there or has several rows");
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (p.M == 0) {  // sums over no rows
    if ((g->dpost_w && cudaMemsetAsync(g->dpost_w, 0, p.C * 4, st) != cudaSuccess) || (g->dpre_w && cudaMemsetAsync(g->dpre_w, 0, p.C * 4, st) != cudaSuccess))
      return fail(KSB_ERR_CUDA, "cannot clear the sums");
    void* const mods[3] = {g->dgate, g->dscale, g->dshift};
    for (int i = 0; i < 3; ++i)
      if (mods[i] && cudaMemsetAsync(mods[i], 0, (size_t)(one_row >> i & 1 ? 1 : a->mod_rows) * p.C * 2, st) != cudaSuccess)
        return fail(KSB_ERR_CUDA, "cannot clear the sums");
    return 0;
  }
  norms::Grads q{};
  q.dr = g->dr; q.dh = g->dh; q.lddr = g->dr ? g->lddr : 0; q.lddh = g->dh ? g->lddh : 0;
  q.dx = g->dx; q.dy = g->dy; q.dgate = g->dgate; q.dscale = g->dscale; q.dshift = g->dshift; q.dpost_w = g->dpost_w; q.dpre_w = g->dpre_w;
  q.parts = static_cast<float*>(workspace);
  if (!p.x || !p.stats || !workspace || (!q.dr && !q.dh)) return fail(KSB_ERR_INVALID, "null pointer");
  for (const void* t : {q.dr, q.dh, (const void*)q.dx, (const void*)q.dy, (const void*)q.dgate, (const void*)q.dscale, (const void*)q.dshift, (const void*)workspace})
    if (!aligned16(t)) return fail(KSB_ERR_INVALID, "unaligned pointer");
  if (p.M > 1 && (q.lddr % 8 != 0 || q.lddh % 8 != 0 || (q.dr && q.lddr < p.C) || (q.dh && q.lddh < p.C))) return fail(KSB_ERR_INVALID, "rows of dr and dh must be multiples of 8 elements apart");
  if (!p.y && (q.dy || q.dgate || q.dpost_w)) return fail(KSB_ERR_INVALID, "dy, dgate and dpost_w belong to y");
  if (!q.dh && (q.dscale || q.dshift || q.dpre_w)) return fail(KSB_ERR_INVALID, "dscale, dshift and dpre_w belong to dh");
  const norms::Plan s = norms::plan_backward(p.M, p.C, p.rows_per_mod);
  q.chunk_rows = (int)s.chunk_rows;
  q.chunks = s.chunks;
  q.samples = (int)a->mod_rows;
  q.one_row = one_row;
  const int before = launch_count();
  if (int rc = a->dtype == KSB_BF16 ? norms::backward<__nv_bfloat16>(p, q, s, a->layer != 0, st) : norms::backward<__half>(p, q, s, a->layer != 0, st)) return rc;
  return launch_count() - before;
}
