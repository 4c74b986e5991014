// Products of a few rows with a weight held in 4 bits:
//
//   out[m, n] = sum_g s[n, g] * (sum_{k in group g} (q[n, k] - z[n, g]) * x[m, k]) + bias[n]
//
// Bound by the weight's way from memory: N K / 2 bytes + a scale (and a zero point) per group, 2 M N K flop.  The weight is
// packed once, in tiles of 16 rows x 64 columns (512 bytes): lane 4 r + t of a warp finds in its 16 bytes the eight columns 8 t of
// both 32-column blocks of rows r and r + 8, as the A fragment of mma.m16n8k16 wants them.  (q - z) is an integer of
// at most 15 in magnitude, exact in bf16 and fp16, so the products are exact and their sums are fp32 per group; the scale
// multiplies a group's fp32 sum, it is never rounded into the weight.
//
// One CTA of sixteen warps per SM takes an even share of the row tiles, each warp an even share of that share's tiles.  A lane copies the
// tiles' bytes that it will read itself (cp.async), and lanes of the warp the scales and zero points, into a ring of the warp's own, so no
// warp waits for another until the end, when the sums of row tiles that several warps share are added up, in the order of the warps.  x
// waits in shared memory.  Where it leaves no room for the rings, or there are few row tiles, the CTAs of a cluster share K: each
// keeps its row tiles' sums, and in the end they are added up in the order of K through distributed shared memory.
//
// Close to bound by issue slots, so a slot of the ring is four tiles, whose copies and products are unrolled, and what a warp keeps of its
// place is one count.  1 x 5120 -> 30720 (81 MB): 16.3 us, without half the products 15.1, HBM's rate 12.5; with a step to a
// slot (89 instructions a tile) 18.7, with bulk copies and mbarriers 18.4, and there deeper rings gained nothing.  8 rows 19.0 us, 16 rows 28.3; 4 x 13824
// -> 30720 (222 MB) 40.2 us, 5.5 TB/s.  5 x 1536 -> 9216 in groups of 32 6.2 us and 16 x 8960 -> 1533 9.3 us, where launch, x's way into
// shared memory and the last sums come one after the other.
#include <algorithm>

#include "../../include/ksana_b200.h"
#include "common.cuh"
#include "host_utils.h"

namespace ksb {
namespace w4 {

constexpr int TILE_N = 16, TILE_K = 64, TILE_BYTES = 512;
constexpr int WARPS = 16, THREADS = WARPS * 32;
constexpr int SMEM_LIMIT = 232448;
// A step: the tiles of a group of 128 columns, or one tile.  A slot of a warp's ring: up to four tiles, their scales and zero points.
constexpr int SLOT_TILES = 4;
// Slots of a ring: a third one gains 4 % (1 x 5120 -> 30720 17.1 -> 16.3 us), and costs more where sixteen rows of x then need a cluster (28.3 -> 37.3 us).
__host__ __device__ constexpr int depth(int nt) { return nt == 1 ? 3 : 2; }
__host__ __device__ constexpr int step_tiles(int group) { return group == 128 ? 2 : 1; }
__host__ __device__ constexpr int slot_bytes(int group, bool zeros) { return SLOT_TILES * TILE_BYTES + SLOT_TILES * TILE_K / group * (zeros ? 48 : 32); }

struct Params {
  const void* x;
  const uint8_t* weight;
  const uint8_t* scale;  // halves
  const uint8_t* zero;   // or null
  const void* bias;      // or null
  void* out;
  int64_t ldx, ldo;
  int M, N, K;
  int split;             // CTAs of a cluster, which share K
  int units_each, units_over;  // row tiles per cluster; the first clusters have one more
  int steps, groups;     // of a row tile (a step: GT tiles)
  int pitch;             // bytes between rows of x in shared memory: 64 more than a multiple of 128, so that the eight 16-byte
                         // reads of a quarter warp (two rows, four neighbours each) are in different banks
  int x_at, sums_at;     // in shared memory, behind the rings
};

// Eight weights of a word as four pairs, (q - z) times UNIT: an AND (or one lop3) and one fma each, and one shift for the word; shifting every
// pair into place held up the integer pipe (1 x 5120 -> 30720: 8 % more).
__device__ __forceinline__ uint32_t and_or(uint32_t w, uint32_t mask, uint32_t c) {
  uint32_t v;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(v) : "r"(w), "r"(mask), "r"(c));
  return v;
}
template <typename T> struct Nibbles;
// The low eight bits of a bf16 count in steps of 2^-133, through the subnormal numbers and the first normal ones (bf16 arithmetic keeps
// both): a nibble in bits 0 - 3 is q 2^-133, in bits 4 - 7 q 2^-129.  Brought to q / 64, since 2^127 is as far as a factor goes.
template <> struct Nibbles<__nv_bfloat16> {
  typedef uint16_t IsHalf;
  static constexpr float UNIT = 1.f / 64;
  uint32_t minus;  // -z / 64 twice
  __device__ __forceinline__ explicit Nibbles(uint32_t z) {
    const uint32_t n = (0x4300u | z) * 0x10001u;  // 128 + z
    minus = fma(n, 0xbc80bc80u, 0x40004000u);     // (128 + z) (-1 / 64) + 2
  }
  static __device__ __forceinline__ uint32_t fma(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t d;
    asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
    return d;
  }
  __device__ __forceinline__ uint32_t low(uint32_t w) const { return fma(w & 0x000f000fu, 0x7f007f00u, minus); }
  __device__ __forceinline__ uint32_t high(uint32_t w) const { return fma(w & 0x00f000f0u, 0x7d007d00u, minus); }
};
// 1024 + q and 1024 + 16 q are the fp16 numbers 0x6400 | q and 0x6400 | q << 4 (integers in the lowest bits of a large half: Kim, Henry, Fahim and Awadalla,
// "Who Says Elephants Can't Run: Bringing Large Scale MoE Models into Cloud Scale Production", 2022).
template <> struct Nibbles<__half> {
  typedef uint8_t IsHalf;
  static constexpr float UNIT = 1.f;
  uint32_t minus, minus16;  // -(1024 + z), -(64 + z)
  __device__ __forceinline__ explicit Nibbles(uint32_t z) : minus((0xe400u | z) * 0x10001u), minus16((0xd400u | z << 4) * 0x10001u) {}
  static __device__ __forceinline__ uint32_t fma(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t d;
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
    return d;
  }
  __device__ __forceinline__ uint32_t low(uint32_t w) const { return fma(and_or(w, 0x000f000fu, 0x64006400u), 0x3c003c00u, minus); }
  __device__ __forceinline__ uint32_t high(uint32_t w) const { return fma(and_or(w, 0x00f000f0u, 0x64006400u), 0x2c002c00u, minus16); }
};

// c = a * b + c; the first of a group's products starts from zeros
#define KSB_MMA16(NAME, TYPE)                                                                                                              \
  __device__ __forceinline__ void NAME(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, float c0, float c1, float c2, float c3) { \
    asm("mma.sync.aligned.m16n8k16.row.col.f32." TYPE "." TYPE ".f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %12, %13};"    \
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])                                                                                    \
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));                                \
  }
KSB_MMA16(mma_bf16, "bf16")
KSB_MMA16(mma_f16, "f16")
#undef KSB_MMA16
template <typename T> __device__ __forceinline__ void mma16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, bool first) {
  const float c0 = first ? 0.f : c[0], c1 = first ? 0.f : c[1], c2 = first ? 0.f : c[2], c3 = first ? 0.f : c[3];
  if constexpr (sizeof(typename Nibbles<T>::IsHalf) == 1) mma_f16(c, a, b0, b1, c0, c1, c2, c3);
  else mma_bf16(c, a, b0, b1, c0, c1, c2, c3);
}

// 16 bytes, or zeros
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool there) {
  const int bytes = there ? 16 : 0;
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ float load_cluster(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}

// NT: blocks of eight rows of x.  G: columns of a group.
template <typename T, int NT, bool ZEROS, int G>
__global__ void __launch_bounds__(THREADS, 1) w4_kernel(const __grid_constant__ Params p) {
  extern __shared__ __align__(128) uint8_t smem[];
  constexpr int GT = step_tiles(G), SCALES = G == 32 ? 2 : 1;  // tiles and groups per step
  constexpr int SLOT = slot_bytes(G, ZEROS), SLOT_STEPS = SLOT_TILES / GT, GROUPS = SLOT_STEPS * SCALES, DEPTH = depth(NT);
  constexpr int SLOT_BYTES = SLOT_TILES * TILE_BYTES, SCALE_AT = SLOT_BYTES, ZERO_AT = SCALE_AT + GROUPS * 32;
  constexpr int SUMS = TILE_N * 8 * NT;       // of a row tile: [row of x][row of the weight]
  // [0]: of the row tile that a warp comes into midway.  [1]: of the one it leaves midway, and on its way to memory any other's
  __shared__ __align__(16) float parts[2][WARPS][SUMS];
  __shared__ __align__(16) uint8_t nothing[256];  // x of the rows there are not
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31, r = lane >> 2, t = lane & 3;
  const int split = p.split, rank = split > 1 ? (int)cluster_ctarank() : 0, cta = blockIdx.x, cluster = cta / split;
  const int k0 = p.steps * rank / split, steps = p.steps * (rank + 1) / split - k0;  // this CTA's steps of every row tile
  const int u0 = cluster * p.units_each + min(cluster, p.units_over), units = p.units_each + (cluster < p.units_over);
  const int64_t share = static_cast<int64_t>(units) * steps;
  const int begin = static_cast<int>(share * warp / WARPS), end = static_cast<int>(share * (warp + 1) / WARPS);
  const uint8_t* ring = smem + warp * (DEPTH * SLOT);
  uint8_t* xs = smem + p.x_at;
  float* sums = reinterpret_cast<float*>(smem + p.sums_at);  // split: [row tile][SUMS]
  const uint32_t ring_at = smem_u32(ring);
  int u = begin / steps, k = begin - u * steps;
  // Of the next steps to ask for: row tile, how many the warp has of it from there on, and the lane's place in them.  Lanes bring the scales and
  // zero points too, 16 bytes each.
  int ahead_u = u, ahead_left = min(steps - k, end - begin);
  const uint8_t* weight = p.weight + (static_cast<int64_t>(u0 + u) * p.steps + k0 + k) * (GT * TILE_BYTES) + lane * 16;
  const bool is_zero = ZEROS && lane >= 2 * GROUPS, has_scale = lane < (ZEROS ? 3 : 2) * GROUPS;
  const int group = is_zero ? lane - 2 * GROUPS : lane >> 1;  // in the slot
  auto scale_place = [&](int at_k) {
    const int64_t g = static_cast<int64_t>(u0 + ahead_u) * p.groups + static_cast<int64_t>(k0 + at_k) * SCALES + group;
    return is_zero ? p.zero + g * 16 : p.scale + g * 32 + (lane & 1) * 16;
  };
  const uint8_t* scale = scale_place(k);
  const int last_u = (end - 1) / steps, last_steps = end - last_u * steps;
  // a row's last half tile may be behind K: it has no group of its own (zeros here), and zeros in x
  const bool lone = SCALES == 2 && (p.groups & 1) && k0 + steps == p.steps;
  const int x0 = k0 * GT * TILE_K, width = min(p.K - x0, steps * GT * TILE_K);  // this CTA's columns of x
  const uint32_t scale_to = ring_at + (is_zero ? ZERO_AT + group * 16 : SCALE_AT + lane * 16), tiles_to = ring_at + lane * 16;
  // Up to a slot of steps, not past a row tile's end.
  auto fetch = [&](int slot) {  // its place in bytes
    if (ahead_left > SLOT_STEPS - (lone ? 0 : 1)) {
#pragma unroll
      for (int g = 0; g < SLOT_TILES; ++g) copy16(tiles_to + slot + g * TILE_BYTES, weight + g * TILE_BYTES, true);
      if (has_scale) copy16(scale_to + slot, scale, true);
      ahead_left -= SLOT_STEPS;
      weight += SLOT_BYTES;
      scale += is_zero ? GROUPS * 16 : GROUPS * 32;
    } else if (ahead_left > 0) {
      const int n = min(SLOT_STEPS, ahead_left), groups = n * SCALES - (lone && n == ahead_left && (ahead_u < last_u || last_steps == steps) ? 1 : 0);
#pragma unroll 1
      for (int g = 0; g < n * GT; ++g) copy16(tiles_to + slot + g * TILE_BYTES, weight + g * TILE_BYTES, true);
      if (has_scale) copy16(scale_to + slot, group < groups ? scale : p.scale, group < groups);
      ahead_left -= n;
      weight += n * (GT * TILE_BYTES);
      scale += n * SCALES * (is_zero ? 16 : 32);
    }
    if (ahead_left == 0 && ahead_u < last_u) {
      ++ahead_u;
      ahead_left = ahead_u == last_u ? last_steps : steps;
      weight += static_cast<int64_t>(p.steps - steps) * (GT * TILE_BYTES);
      scale = scale_place(0);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  pdl_wait();  // whatever ran ahead, the caller's kernels too
  pdl_release();
  // x, ahead of the weight, whose slots it would have to wait for; zeros behind its last column, and in place of its missing rows
  {
    const int units16 = steps * GT * 8, full = width / 8;  // 16-byte units of a row
    const int each = WARPS / p.M, m = warp / each;  // warps per row (at most 16 rows); the last may have none
    if (m < p.M) {
      const T* row = static_cast<const T*>(p.x) + m * p.ldx + x0;
      for (int i = (warp - m * each) * 32 + lane; i < units16; i += each * 32) copy16(smem_u32(xs) + m * p.pitch + i * 16, row + (i < full ? i * 8 : 0), i < full);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    if (threadIdx.x < 16) reinterpret_cast<uint4*>(nothing)[threadIdx.x] = make_uint4(0, 0, 0, 0);
  }
#pragma unroll
  for (int d = 0; d < DEPTH - 1; ++d) fetch(d * SLOT);
  asm volatile("cp.async.wait_group %0;" ::"n"(DEPTH - 1) : "memory");  // x, asked for first
  __syncthreads();

  float acc[NT][4];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[nt][i] = 0.f;
  // a row tile's sums on their way out
  auto put = [&](int which) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        parts[which][warp][(nt * 8 + 2 * t + (i & 1)) * TILE_N + r + (i >> 1) * 8] = acc[nt][i] * (1.f / Nibbles<T>::UNIT);
        acc[nt][i] = 0.f;
      }
    __syncwarp();
  };
  auto store = [&](int row_tile, int j, float v) {
    const int m = j >> 4, n = (u0 + row_tile) * TILE_N + (j & 15);
    if (n >= p.N) return;
    if (p.bias) v += HalfOps<T>::to_f(static_cast<const T*>(p.bias)[n]);
    static_cast<T*>(p.out)[m * p.ldo + n] = HalfOps<T>::from_f(v);
  };
  auto keep = [&](int row_tile, int j, float v) {
    if (split > 1) sums[row_tile * SUMS + j] = v;
    else store(row_tile, j, v);
  };
  const int live = p.M * TILE_N;  // sums that there are
  // a lane's x: of a row that there is not, the same zeros at every step
  const uint8_t *x_row[NT], *xk[NT];
  int x_step[NT];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const bool there = nt * 8 + r < p.M;
    x_step[nt] = there ? GT * 128 : 0;
    x_row[nt] = (there ? xs + (nt * 8 + r) * p.pitch : nothing) + t * 16;
    xk[nt] = x_row[nt] + k * x_step[nt];
  }
  bool entered = k != 0;  // the row tile was begun by an earlier warp
  int slot = 0, free_slot = (DEPTH - 1) * SLOT;
  int left = min(steps - k, end - begin);  // of the row tile
  while (left > 0) {
    asm volatile("cp.async.wait_group %0;" ::"n"(DEPTH - 2) : "memory");
    __syncwarp();  // every lane's part of the slot is there, and the slot before has been read
    fetch(free_slot);
    free_slot = slot;
    const uint8_t* tiles = ring + slot + lane * 16;
    const T* scales = reinterpret_cast<const T*>(ring + slot + SCALE_AT) + r;
    const uint8_t* zeros = ring + slot + ZERO_AT + r;
    slot = slot == (DEPTH - 1) * SLOT ? 0 : slot + SLOT;
    auto step = [&](int j) {
      float part[NT][4];
#pragma unroll
      for (int half = 0; half < 2 * GT; ++half) {
        const uint4 a4 = *reinterpret_cast<const uint4*>(tiles + (j * GT + (half >> 1)) * TILE_BYTES);
        const uint32_t w0 = half & 1 ? a4.z : a4.x, w1 = half & 1 ? a4.w : a4.y;
        const bool first = SCALES == 2 || half == 0, done = SCALES == 2 || half == 2 * GT - 1;
        const int g = (j * SCALES + (SCALES == 2 ? half : 0)) * TILE_N;
        uint32_t z0 = 8, z1 = 8;
        if (ZEROS) {
          z0 = zeros[g] & 15u;
          z1 = zeros[g + 8] & 15u;
        }
        const Nibbles<T> n0(z0), n1(z1);
        uint32_t a[2][4];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const uint32_t v0 = w0 >> (8 * c), v1 = w1 >> (8 * c);
          a[c][0] = n0.low(v0);
          a[c][1] = n1.low(v1);
          a[c][2] = n0.high(v0);
          a[c][3] = n1.high(v1);
        }
        float s0 = 0.f, s1 = 0.f;
        if (done) {
          s0 = HalfOps<T>::to_f(scales[g]);  // over UNIT: see put
          s1 = HalfOps<T>::to_f(scales[g + 8]);
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const uint4 b = *reinterpret_cast<const uint4*>(xk[nt] + j * x_step[nt] + half * 64);
          mma16<T>(part[nt], a[0], b.x, b.y, first);
          mma16<T>(part[nt], a[1], b.z, b.w, false);
          if (done) {
            acc[nt][0] = fmaf(s0, part[nt][0], acc[nt][0]);
            acc[nt][1] = fmaf(s0, part[nt][1], acc[nt][1]);
            acc[nt][2] = fmaf(s1, part[nt][2], acc[nt][2]);
            acc[nt][3] = fmaf(s1, part[nt][3], acc[nt][3]);
          }
        }
      }
    };
    if (left >= SLOT_STEPS) {
#pragma unroll
      for (int j = 0; j < SLOT_STEPS; ++j) step(j);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) xk[nt] += SLOT_STEPS * x_step[nt];
      left -= SLOT_STEPS;
    } else {
#pragma unroll 1
      for (int j = 0; j < left; ++j) step(j);
      left = 0;
    }
    if (left > 0) continue;
    if (u == last_u && last_steps != steps) {  // left midway
      k = last_steps;
      break;
    }
    put(entered ? 0 : 1);
    if (!entered) {
#pragma unroll 1
      for (int j = lane; j < live; j += 32) keep(u, j, parts[1][warp][j]);
      __syncwarp();
    }
    entered = false;
    k = 0;
    if (++u > last_u) break;
    left = u == last_u ? last_steps : steps;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) xk[nt] = x_row[nt];
    if (p.bias && lane == 0) asm volatile("prefetch.global.L1 [%0];" ::"l"(static_cast<const T*>(p.bias) + min((u0 + u) * TILE_N, p.N - 1)));
  }
  if (begin == end || k != 0) put(begin == end || entered ? 0 : 1);  // without a share: zeros
  __syncthreads();
  // Row tiles that several warps share, each known by the warp that has begun it and left it to others: 32 sums at a time, by all warps in
  // turn (by one warp, a row tile of sixteen pieces and 16 rows took 5 us).
  const int batches = (live + 31) / 32;
#pragma unroll 1
  for (int i = warp; i < WARPS * batches; i += WARPS) {
    const int w0 = i / batches, j = (i - w0 * batches) * 32 + lane;
    const int first = static_cast<int>(share * w0 / WARPS), left = static_cast<int>(share * (w0 + 1) / WARPS), tail = left / steps, start = tail * steps;
    if (left == start || first == left || first > start || j >= live) continue;
    float v = parts[1][w0][j];
#pragma unroll 4
    for (int w = w0 + 1; w < WARPS && static_cast<int>(share * w / WARPS) < start + steps; ++w) v += parts[0][w][j];
    keep(tail, j, v);
  }
  if (split > 1) {
    cluster_sync_all();  // every CTA's sums are there
    const uint32_t mine = smem_u32(sums);
    for (int i = rank * THREADS + threadIdx.x; i < units * live; i += split * THREADS) {
      const int row_tile = i / live, j = i - row_tile * live;
      float v = 0.f;
      for (int c = 0; c < split; ++c) v += load_cluster(mapa_shared(mine, c) + (row_tile * SUMS + j) * 4);
      store(row_tile, j, v);
    }
    cluster_sync_all();  // none leaves while another reads it
  }
}

constexpr int fixed_bytes(int nt) { return 2 * WARPS * TILE_N * 8 * nt * 4 + 256 + 128; }
template <typename T, int NT, bool ZEROS, int G> static int launch(const Params& p, int grid, size_t smem, cudaStream_t st) {
  auto kernel = w4_kernel<T, NT, ZEROS, G>;
  static DeviceOnce limit;
  if (int rc = limit.raise_smem(reinterpret_cast<const void*>(kernel), SMEM_LIMIT - fixed_bytes(NT))) return rc;
  return launch_kernel("w4 linear", reinterpret_cast<const void*>(kernel), dim3((unsigned)grid), dim3(THREADS), smem, st, p.split, true, p);
}
template <typename T, int NT, bool ZEROS> static int with_group(const Params& p, int group, int grid, size_t smem, cudaStream_t st) {
  return group == 32 ? launch<T, NT, ZEROS, 32>(p, grid, smem, st) : group == 64 ? launch<T, NT, ZEROS, 64>(p, grid, smem, st) : launch<T, NT, ZEROS, 128>(p, grid, smem, st);
}
template <typename T> static int dispatch(const Params& p, int group, int grid, size_t smem, cudaStream_t st) {
  if (p.M > 8) return p.zero ? with_group<T, 2, true>(p, group, grid, smem, st) : with_group<T, 2, false>(p, group, grid, smem, st);
  return p.zero ? with_group<T, 1, true>(p, group, grid, smem, st) : with_group<T, 1, false>(p, group, grid, smem, st);
}

}  // namespace w4
}  // namespace ksb

using namespace ksb;

extern "C" int ksb_w4_linear(const void* x, int dtype, int64_t M, int64_t K, int64_t ldx, const void* weight, const void* scale, const void* zero,
                             int group, const void* bias, int64_t N, void* out, int64_t ldo, ksb_stream_t stream) {
  if (dtype != KSB_BF16 && dtype != KSB_FP16) return fail(KSB_ERR_INVALID, "dtype must be KSB_BF16 or KSB_FP16");
  if (group != 32 && group != 64 && group != 128) return fail(KSB_ERR_INVALID, "groups of 32, 64 or 128 columns, not %d", group);
  if (M < 0 || N <= 0 || K <= 0 || M > INT32_MAX || N > INT32_MAX - 16 || K % group != 0)
    return fail(KSB_ERR_INVALID, "bad shape M=%lld N=%lld K=%lld (K in whole groups of %d)", (long long)M, (long long)N, (long long)K, group);
  if (K > KSB_W4_MAX_K) return fail(KSB_ERR_UNSUPPORTED, "K=%lld is above %d", (long long)K, KSB_W4_MAX_K);
  if (M == 0) return 0;
  if (!x || !weight || !scale || !out) return fail(KSB_ERR_INVALID, "null pointer");
  if (!aligned16(x) || !aligned16(weight) || !aligned16(scale) || (zero && !aligned16(zero)) || (M > 1 && (ldx < K || ldx % 8 != 0)) || (M > 1 && ldo < N))
    return fail(KSB_ERR_INVALID, "x, the packed weight, its scales and zero points must be 16-byte aligned, ldx %% 8 == 0");
  w4::Params p{};
  p.weight = static_cast<const uint8_t*>(weight);
  p.scale = static_cast<const uint8_t*>(scale);
  p.zero = static_cast<const uint8_t*>(zero);
  p.bias = bias;
  p.ldx = ldx; p.ldo = ldo;
  p.N = (int)N; p.K = (int)K;
  const int units = (int)((N + w4::TILE_N - 1) / w4::TILE_N);
  const int tiles = (int)((K + w4::TILE_K - 1) / w4::TILE_K), step_tiles = w4::step_tiles(group);
  p.steps = tiles / step_tiles;
  p.groups = (int)(K / group);
  auto plan = [&](int rows, int split) {
    const int clusters = std::min(units, cluster_room(split)), sums = w4::TILE_N * (rows > 8 ? 16 : 8) * 4;
    p.x_at = w4::WARPS * w4::depth(rows > 8 ? 2 : 1) * w4::slot_bytes(group, zero != nullptr);
    p.split = split;
    p.units_each = units / clusters;
    p.units_over = units % clusters;
    p.pitch = ((p.steps + split - 1) / split) * step_tiles * 128 + 64;
    const int64_t kept = split > 1 ? (int64_t)(p.units_each + 1) * sums : 0;
    p.sums_at = p.x_at + rows * p.pitch;
    return p.sums_at + kept <= w4::SMEM_LIMIT - w4::fixed_bytes(rows > 8 ? 2 : 1) ? (int)(p.sums_at + kept) : 0;
  };
  // K is shared by a cluster where that fills the GPU, or makes room for the rows of x.
  int split = 1;
  auto fit = [&](int rows) {
    split = 1;
    while (split < 8 && 2 * split * units <= sm_count() && 2 * split <= p.steps) split *= 2;
    int smem;
    while ((smem = plan(rows, split)) == 0 && split < 8 && 2 * split <= p.steps) split *= 2;
    return smem;
  };
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  int launches = 0;
  for (int64_t m0 = 0; m0 < M; ++launches) {
    // As few passes over the weight as there is room for (x, and with a shared K the row tiles' sums), of equal sizes where those fit: nine to
    // sixteen rows may fit where eight do not, whose rings are deeper.  16 x 13824 -> 30720 takes 92 us in two passes; in three, as it was where
    // fewer rows were tried without clusters, 134.
    const int64_t left = M - m0;
    int rows = 0, smem = 0;
    for (int most = (int)std::min<int64_t>(16, left); smem == 0 && most > 0; --most) {
      const int64_t passes = (left + most - 1) / most;
      rows = (int)((left + passes - 1) / passes);
      smem = fit(rows);
      if (smem == 0 && rows < most) smem = fit(rows = most);
    }
    if (smem == 0) return fail(KSB_ERR_UNSUPPORTED, "no room for a row of %lld columns", (long long)K);
    p.M = rows;
    p.x = static_cast<const uint8_t*>(x) + m0 * ldx * 2;
    p.out = static_cast<uint8_t*>(out) + m0 * ldo * 2;
    const int grid = std::min(units, cluster_room(split)) * split;
    if (int rc = dtype == KSB_BF16 ? w4::dispatch<__nv_bfloat16>(p, group, grid, smem, st) : w4::dispatch<__half>(p, group, grid, smem, st)) return rc;
    m0 += rows;
  }
  return launches;
}
