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
// One CTA per SM, persistent over the row tiles: one thread copies the packed tiles of a row tile, up to CHUNK a stage, with their
// scales and zero points into a ring in shared memory (bulk copies: consecutive bytes all the way), sixteen warps take the tiles
// in turn, and their sums meet in shared memory in the order of the warps.  x waits in shared memory for all of it.
#include <algorithm>

#include "../../include/ksana_b200.h"
#include "common.cuh"
#include "host_utils.h"

namespace ksb {
namespace w4 {

constexpr int KERNEL_ID = 6;
constexpr int TILE_N = 16, TILE_K = 64, TILE_BYTES = 512;
constexpr int WARPS = 16, CHUNK = 32;  // tiles per stage
constexpr int THREADS = WARPS * 32 + 32;
constexpr int MAX_STAGES = 12;
constexpr int SMEM_LIMIT = 232448;
constexpr int BAR_BYTES = MAX_STAGES * 16;

struct Params {
  const void* x;
  const uint8_t* weight;
  const uint8_t* scale;  // halves
  const uint8_t* zero;   // or null
  const void* bias;      // or null
  void* out;
  int64_t ldx, ldo;
  int M, N, K;
  int units, tiles_k;    // row tiles, tiles of a row tile
  int group, groups;     // columns per group, groups of a row
  int pitch;             // bytes between rows of x in shared memory: 64 more than a multiple of 128, so that the eight 16-byte
                         // reads of a quarter warp (two rows, four neighbours each) are in different banks
  int stages, stage_bytes, zero_at;  // of the ring; where a stage's zero points are (its scales are behind CHUNK tiles)
  int* status;
};

template <typename T> struct Nibbles;
// 128 + q is the bf16 number 0x4300 | q, 1024 + q the fp16 number 0x6400 | q; 128 + z and 1024 + z are exact as well.
template <> struct Nibbles<__nv_bfloat16> {
  static __device__ __forceinline__ uint32_t offset(uint32_t z) { return (0x4300u | z) * 0x10001u; }
  static __device__ __forceinline__ uint32_t pair(uint32_t w, int i, uint32_t off) {
    const uint32_t v = ((w >> (4 * i)) & 0x000f000fu) | 0x43004300u;
    const __nv_bfloat162 d = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&v), *reinterpret_cast<const __nv_bfloat162*>(&off));
    return *reinterpret_cast<const uint32_t*>(&d);
  }
};
template <> struct Nibbles<__half> {
  static __device__ __forceinline__ uint32_t offset(uint32_t z) { return (0x6400u | z) * 0x10001u; }
  static __device__ __forceinline__ uint32_t pair(uint32_t w, int i, uint32_t off) {
    const uint32_t v = ((w >> (4 * i)) & 0x000f000fu) | 0x64006400u;
    const __half2 d = __hsub2(*reinterpret_cast<const __half2*>(&v), *reinterpret_cast<const __half2*>(&off));
    return *reinterpret_cast<const uint32_t*>(&d);
  }
};

template <typename T> __device__ __forceinline__ void mma16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <> __device__ __forceinline__ void mma16<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <> __device__ __forceinline__ void mma16<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar)
               : "memory");
}

// NT: blocks of eight rows of x.  FINE: groups of 32 columns, a scale per half tile.
template <typename T, int NT, bool ZEROS, bool FINE>
__global__ void __launch_bounds__(THREADS, 1) w4_kernel(const __grid_constant__ Params p) {
  extern __shared__ __align__(128) uint8_t smem[];
  constexpr int SUMS = TILE_N * 8 * NT;  // of a row tile
  __shared__ __align__(16) float red[2][WARPS][SUMS];
  __shared__ __align__(8) uint64_t bars[2 * MAX_STAGES];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t ring = smem_u32(smem), full0 = smem_u32(bars), empty0 = full0 + 8 * MAX_STAGES;
  uint8_t* xs = smem + p.stages * p.stage_bytes;
  if (threadIdx.x == 0) {
    for (int s = 0; s < p.stages; ++s) {
      mbar_init(full0 + 8 * s, 1);
      mbar_init(empty0 + 8 * s, WARPS);
    }
    fence_barrier_init();
  }
  __syncthreads();
  const int chunks = (p.tiles_k + CHUNK - 1) / CHUNK;
  const int chunk_groups = CHUNK * TILE_K / p.group;
  if (warp == WARPS) {
    if (lane == 0) {
      uint32_t it = 0;
      bool ok = true;
      for (int u = blockIdx.x; u < p.units && ok; u += gridDim.x) {
        for (int c = 0; c < chunks; ++c, ++it) {
          const uint32_t s = it % p.stages, ph = (it / p.stages) & 1;
          if (!mbar_wait(empty0 + 8 * s, ph ^ 1, p.status, (KERNEL_ID << 16) | 1)) { ok = false; break; }
          const int tiles = min(CHUNK, p.tiles_k - c * CHUNK), groups = min(chunk_groups, p.groups - c * chunk_groups);
          const int64_t g0 = static_cast<int64_t>(u) * p.groups + c * chunk_groups;
          const uint32_t dst = ring + s * p.stage_bytes, bar = full0 + 8 * s;
          mbar_arrive_expect_tx(bar, tiles * TILE_BYTES + groups * (ZEROS ? 48 : 32));
          bulk_load(dst, p.weight + (static_cast<int64_t>(u) * p.tiles_k + c * CHUNK) * TILE_BYTES, tiles * TILE_BYTES, bar);
          bulk_load(dst + CHUNK * TILE_BYTES, p.scale + g0 * 32, groups * 32, bar);
          if (ZEROS) bulk_load(dst + p.zero_at, p.zero + g0 * 16, groups * 16, bar);
        }
      }
      // what is on its way lands before the block leaves
      for (uint32_t i = it > (uint32_t)p.stages ? it - p.stages : 0; i < it; ++i)
        mbar_wait(full0 + 8 * (i % p.stages), (i / p.stages) & 1, p.status, (KERNEL_ID << 16) | 3);
    }
  } else {
    // x, zeros behind its last column
    const int units16 = p.tiles_k * 8, width = p.K / 8;  // 16-byte units of a row
    for (int i = threadIdx.x; i < p.M * units16; i += WARPS * 32) {
      const int m = i / units16, u = i - m * units16;
      const uint4 v = u < width ? reinterpret_cast<const uint4*>(static_cast<const T*>(p.x) + m * p.ldx)[u] : make_uint4(0, 0, 0, 0);
      *reinterpret_cast<uint4*>(xs + m * p.pitch + u * 16) = v;
    }
    asm volatile("bar.sync 1, %0;" ::"n"(WARPS * 32) : "memory");
    const int r = lane >> 2, t = lane & 3;
    const int group_shift = p.group == 128 ? 1 : 0;
    bool failed = false;
    uint32_t it = 0;
    int par = 0;
    for (int u = blockIdx.x; u < p.units; u += gridDim.x, par ^= 1) {
      float acc[NT][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[nt][i] = 0.f;
      for (int c = 0; c < chunks; ++c, ++it) {
        const uint32_t s = it % p.stages, ph = (it / p.stages) & 1;
        if (!failed && !mbar_wait_warp(full0 + 8 * s, ph, p.status, (KERNEL_ID << 16) | 2)) failed = true;
        if (failed) continue;
        const int tiles = min(CHUNK, p.tiles_k - c * CHUNK);
        const uint8_t* stage = smem + s * p.stage_bytes;
        const T* scales = reinterpret_cast<const T*>(stage + CHUNK * TILE_BYTES);
        const uint8_t* zeros = stage + p.zero_at;
        for (int j = warp; j < tiles; j += WARPS) {
          const uint4 a4 = *reinterpret_cast<const uint4*>(stage + j * TILE_BYTES + lane * 16);
          const uint32_t words[4] = {a4.x, a4.y, a4.z, a4.w};
          float part[NT][4], s0 = 0.f, s1 = 0.f;
          uint32_t z0 = Nibbles<T>::offset(8), z1 = z0;
#pragma unroll
          for (int kb = 0; kb < 2; ++kb) {
            if (FINE || kb == 0) {
              // a last half tile behind K has zeros in x: any group's scale will do
              const int g = FINE ? min(2 * j + kb, p.groups - 1 - c * chunk_groups) : j >> group_shift;
              s0 = HalfOps<T>::to_f(scales[g * 16 + r]);
              s1 = HalfOps<T>::to_f(scales[g * 16 + r + 8]);
              if (ZEROS) {
                z0 = Nibbles<T>::offset(zeros[g * 16 + r] & 15u);
                z1 = Nibbles<T>::offset(zeros[g * 16 + r + 8] & 15u);
              }
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int i = 0; i < 4; ++i) part[nt][i] = 0.f;
            }
            uint32_t a[2][4];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              a[h][0] = Nibbles<T>::pair(words[2 * kb], 2 * h, z0);
              a[h][1] = Nibbles<T>::pair(words[2 * kb + 1], 2 * h, z1);
              a[h][2] = Nibbles<T>::pair(words[2 * kb], 2 * h + 1, z0);
              a[h][3] = Nibbles<T>::pair(words[2 * kb + 1], 2 * h + 1, z1);
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              uint4 b = make_uint4(0, 0, 0, 0);
              const int m = nt * 8 + r;
              if (m < p.M) b = *reinterpret_cast<const uint4*>(xs + m * p.pitch + ((c * CHUNK + j) * 2 + kb) * 64 + t * 16);
              mma16<T>(part[nt], a[0], b.x, b.y);
              mma16<T>(part[nt], a[1], b.z, b.w);
            }
            if (FINE || kb == 1) {
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                acc[nt][0] = fmaf(s0, part[nt][0], acc[nt][0]);
                acc[nt][1] = fmaf(s0, part[nt][1], acc[nt][1]);
                acc[nt][2] = fmaf(s1, part[nt][2], acc[nt][2]);
                acc[nt][3] = fmaf(s1, part[nt][3], acc[nt][3]);
              }
            }
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(empty0 + 8 * s);
      }
      // [row of x][row of the weight]
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 4; ++i) red[par][warp][(nt * 8 + 2 * t + (i & 1)) * TILE_N + r + (i >> 1) * 8] = acc[nt][i];
      failed = named_bar_or(1, WARPS * 32, failed);
      if (failed) break;
      const int m = threadIdx.x >> 4, n = u * TILE_N + (threadIdx.x & 15);
      if (threadIdx.x < SUMS && m < p.M && n < p.N) {
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) v += red[par][w][threadIdx.x];
        if (p.bias) v += HalfOps<T>::to_f(static_cast<const T*>(p.bias)[n]);
        static_cast<T*>(p.out)[m * p.ldo + n] = HalfOps<T>::from_f(v);
      }
    }
  }
}

template <typename T, int NT, bool ZEROS, bool FINE> static int launch(const Params& p, int grid, size_t smem, cudaStream_t st) {
  auto kernel = w4_kernel<T, NT, ZEROS, FINE>;
  static DeviceOnce limit;
  const int fixed = 2 * WARPS * TILE_N * 8 * NT * 4 + 16 * MAX_STAGES + 64;
  if (int rc = limit.raise_smem(reinterpret_cast<const void*>(kernel), SMEM_LIMIT - fixed)) return rc;
  return launch_kernel("w4 linear", reinterpret_cast<const void*>(kernel), dim3((unsigned)grid), dim3(THREADS), smem, st, 1, false, p);
}
template <typename T> static int dispatch(const Params& p, int grid, size_t smem, cudaStream_t st) {
  const bool wide = p.M > 8, zeros = p.zero != nullptr, fine = p.group == 32;
  if (wide) {
    if (zeros) return fine ? launch<T, 2, true, true>(p, grid, smem, st) : launch<T, 2, true, false>(p, grid, smem, st);
    return fine ? launch<T, 2, false, true>(p, grid, smem, st) : launch<T, 2, false, false>(p, grid, smem, st);
  }
  if (zeros) return fine ? launch<T, 1, true, true>(p, grid, smem, st) : launch<T, 1, true, false>(p, grid, smem, st);
  return fine ? launch<T, 1, false, true>(p, grid, smem, st) : launch<T, 1, false, false>(p, grid, smem, st);
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
  p.status = status_words();
  if (!p.status) return fail(KSB_ERR_CUDA, "status words unavailable");
  p.weight = static_cast<const uint8_t*>(weight);
  p.scale = static_cast<const uint8_t*>(scale);
  p.zero = static_cast<const uint8_t*>(zero);
  p.bias = bias;
  p.ldx = ldx; p.ldo = ldo;
  p.N = (int)N; p.K = (int)K;
  p.units = (int)((N + w4::TILE_N - 1) / w4::TILE_N);
  p.tiles_k = (int)((K + w4::TILE_K - 1) / w4::TILE_K);
  p.group = group; p.groups = (int)(K / group);
  p.pitch = p.tiles_k * 128 + 64;
  const int chunk_groups = w4::CHUNK * w4::TILE_K / group;
  p.zero_at = w4::CHUNK * w4::TILE_BYTES + chunk_groups * 32;
  p.stage_bytes = p.zero_at + (zero ? chunk_groups * 16 : 0);
  const int grid = p.units < sm_count() ? p.units : sm_count();
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  int launches = 0;
  // Rows of one launch: what fits beside two stages and the sums.
  for (int64_t m0 = 0; m0 < M;) {
    const int room = w4::SMEM_LIMIT - 2 * w4::WARPS * w4::TILE_N * 16 * 4 - 16 * w4::MAX_STAGES - 64 - 2 * p.stage_bytes;
    const int64_t rows = std::min<int64_t>({M - m0, 16, room / p.pitch});
    p.M = (int)rows;
    p.x = static_cast<const uint8_t*>(x) + m0 * ldx * 2;
    p.out = static_cast<uint8_t*>(out) + m0 * ldo * 2;
    const int fixed = 2 * w4::WARPS * w4::TILE_N * (rows > 8 ? 16 : 8) * 4 + 16 * w4::MAX_STAGES + 64;
    p.stages = std::min(w4::MAX_STAGES, (w4::SMEM_LIMIT - fixed - (int)rows * p.pitch) / p.stage_bytes);
    const size_t smem = (size_t)p.stages * p.stage_bytes + (size_t)rows * p.pitch;
    if (int rc = dtype == KSB_BF16 ? w4::dispatch<__nv_bfloat16>(p, grid, smem, st) : w4::dispatch<__half>(p, grid, smem, st)) return rc;
    m0 += rows;
    ++launches;
  }
  return launches;
}
