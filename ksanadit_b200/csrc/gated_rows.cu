// The gated projections of a few rows of x: h = act(x Wg^T + bg) * (x Wu^T + bu), bound by the two weights' way from memory (4 F K bytes).
//
// A tile of mma.m16n8k16 holds eight rows of Wg and the same eight rows of Wu, so that the thread with an element of g has that of u.
// A lane's 16 bytes of a weight row are eight columns, and so are its 16 bytes of x: the order of the columns inside a product is the
// same for both, which is all it needs, and nothing is rearranged.  On the tensor cores' wide form (128 rows a product) a few rows of x take as
// long as 128: 1 x 5120 -> 13824 was 122 us with x as its A operand, bound by the products.
//
// One CTA of sixteen warps per SM takes an even share of the row tiles, each warp an even share of that share's steps of 64 columns.  A
// lane copies what it will read itself (cp.async, DEPTH - 1 steps ahead), so no warp waits for another until the end, when the
// sums of row tiles that several warps share are added up, in the order of the warps.  x waits in shared memory.  Where it leaves no room
// for that, or there are few row tiles, the CTAs of a cluster share K: each keeps its row tiles' sums, and in the end they are added
// up in the order of K through distributed shared memory.
//
// Measured: 1 x 1536 -> 8960 11.3 us (55 MB: 4.9 TB/s with launch and the last sums, 8.5 us at HBM's rate), 1 x 5120 -> 13824 46.7 us (6.1 TB/s; 48.1
// where the L2 does not ask for 256 bytes at once, 49.6 with a fourth slot, 49.2 with half of the products).
#include <algorithm>

#include "gated.h"
#include "host_utils.h"

namespace ksb {
namespace gated {

constexpr int TILE_F = 8, STEP = 64;                 // rows of each weight in a row tile, columns of a step
constexpr int WARPS = 16, ROWS_THREADS = WARPS * 32;
constexpr int DEPTH = 3, SLOT_BYTES = 2048;          // of a warp's ring: [block of 32 columns][weight][lane] 16 bytes
constexpr int SMEM_LIMIT = 232448;

struct RowsParams {
  RowsCall c;
  int split;                   // CTAs of a cluster, which share K
  int units_each, units_over;  // row tiles per cluster; the first clusters have one more
  int steps;                   // of a row tile
  int pitch;                   // bytes between rows of x in shared memory, 64 more than a multiple of 128: no two of a quarter warp's reads meet in a bank
  int x_at, sums_at;           // in shared memory, behind the rings
};

// A step takes 128 bytes of a weight's row: the L2 asks for the next 128 with them.
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool there) {
  const int bytes = there ? 16 : 0;  // the rest is filled with zeros
  asm volatile("cp.async.cg.shared.global.L2::256B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}

template <typename T> __device__ __forceinline__ void mma16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1);
template <> __device__ __forceinline__ void mma16<__nv_bfloat16>(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <> __device__ __forceinline__ void mma16<__half>(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float load_cluster(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}

// NT: blocks of eight rows of x
template <typename T, int NT> __global__ void __launch_bounds__(ROWS_THREADS, 1) rows_kernel(const __grid_constant__ RowsParams p) {
  extern __shared__ __align__(128) uint8_t smem[];
  constexpr int SUMS = 16 * 8 * NT;  // of a row tile: [row of x][8 of g, 8 of u]
  // [0]: of the row tile that a warp comes into midway.  [1]: of the one it leaves midway, and on its way to memory any other's
  __shared__ __align__(16) float parts[2][WARPS][SUMS];
  __shared__ __align__(16) uint8_t nothing[256];  // x of the rows there are not
  const RowsCall& c = p.c;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31, r = lane >> 2, t = lane & 3;
  const int split = p.split, rank = split > 1 ? (int)cluster_ctarank() : 0, cluster = blockIdx.x / split;
  const int k0 = p.steps * rank / split, steps = p.steps * (rank + 1) / split - k0;  // this CTA's steps of every row tile
  const int u0 = cluster * p.units_each + min(cluster, p.units_over), units = p.units_each + (cluster < p.units_over);
  const int64_t share = static_cast<int64_t>(units) * steps;
  const int begin = static_cast<int>(share * warp / WARPS), end = static_cast<int>(share * (warp + 1) / WARPS);
  uint8_t* xs = smem + p.x_at;
  float* sums = reinterpret_cast<float*>(smem + p.sums_at);  // split: [row tile][SUMS]
  const uint32_t ring = smem_u32(smem) + warp * (DEPTH * SLOT_BYTES) + lane * 16;
  const int x0 = k0 * STEP, width = min(c.K - x0, steps * STEP);  // this CTA's columns of x
  int u = begin / steps, k = begin - u * steps;
  // the lane's place in both weights for the next step to ask for
  int ahead = begin, ahead_k = k;
  const T* gate = static_cast<const T*>(c.w_gate) + static_cast<int64_t>((u0 + u) * TILE_F + r) * c.ldg + (k0 + k) * STEP + t * 8;
  const T* up = static_cast<const T*>(c.w_up) + static_cast<int64_t>((u0 + u) * TILE_F + r) * c.ldu + (k0 + k) * STEP + t * 8;
  const int64_t next_gate = TILE_F * c.ldg - steps * STEP, next_up = TILE_F * c.ldu - steps * STEP;
  auto fetch = [&](int slot) {
    if (ahead < end) {
      const int col = (k0 + ahead_k) * STEP + t * 8;
      const uint32_t dst = ring + slot * SLOT_BYTES;
      copy16(dst, gate, col < c.K);
      copy16(dst + 512, up, col < c.K);
      copy16(dst + 1024, gate + (col + 32 < c.K ? 32 : 0), col + 32 < c.K);
      copy16(dst + 1536, up + (col + 32 < c.K ? 32 : 0), col + 32 < c.K);
      ++ahead;
      gate += STEP;
      up += STEP;
      if (++ahead_k == steps) {
        ahead_k = 0;
        gate += next_gate;
        up += next_up;
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  pdl_wait();  // whatever ran ahead, the caller's kernels too
  pdl_release();
  {
    const int units16 = steps * (STEP / 8), full = width / 8;  // 16-byte units of a row
    const int each = WARPS / c.M, m = warp / each;  // warps per row (at most 16 rows); the last may have none
    if (m < c.M) {
      const T* row = static_cast<const T*>(c.x) + m * c.ldx + x0;
      for (int i = (warp - m * each) * 32 + lane; i < units16; i += each * 32) copy16(smem_u32(xs) + m * p.pitch + i * 16, row + (i < full ? i * 8 : 0), i < full);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    if (threadIdx.x < 16) reinterpret_cast<uint4*>(nothing)[threadIdx.x] = make_uint4(0, 0, 0, 0);
  }
#pragma unroll
  for (int d = 0; d < DEPTH - 1; ++d) fetch(d);
  asm volatile("cp.async.wait_group %0;" ::"n"(DEPTH - 1) : "memory");  // x, asked for first
  __syncthreads();

  float acc[NT][4];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[nt][i] = 0.f;
  auto put = [&](int which) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        parts[which][warp][(nt * 8 + 2 * t + (i & 1)) * 16 + r + (i >> 1) * 8] = acc[nt][i];
        acc[nt][i] = 0.f;
      }
    __syncwarp();
  };
  // element j = row of x * 8 + column of the row tile, of its two sums
  auto store = [&](int row_tile, int j, float g, float v) {
    const int f = (u0 + row_tile) * TILE_F + (j & 7);
    if (c.b_gate) g += HalfOps<T>::to_f(static_cast<const T*>(c.b_gate)[f]);
    if (c.b_up) v += HalfOps<T>::to_f(static_cast<const T*>(c.b_up)[f]);
    static_cast<T*>(c.h)[static_cast<int64_t>(j >> 3) * c.F + f] = HalfOps<T>::from_f(g * act_sigmoid(g, c.act) * v);
  };
  auto sum_at = [](int j) { return (j >> 3) * 16 + (j & 7); };
  auto keep = [&](int row_tile, int j, float g, float v) {
    if (split > 1) {
      sums[row_tile * SUMS + sum_at(j)] = g;
      sums[row_tile * SUMS + sum_at(j) + 8] = v;
    } else {
      store(row_tile, j, g, v);
    }
  };
  const int live = c.M * TILE_F;  // elements that there are
  const uint8_t* x_at[NT];
  int x_step[NT];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const bool there = nt * 8 + r < c.M;
    x_at[nt] = (there ? xs + (nt * 8 + r) * p.pitch : nothing) + t * 16;
    x_step[nt] = there ? STEP * 2 : 0;
  }
  bool entered = k != 0;  // the row tile was begun by an earlier warp
  int slot = 0;
  for (int at = begin; at < end; ++at) {
    asm volatile("cp.async.wait_group %0;" ::"n"(DEPTH - 2) : "memory");
    const uint32_t mine = ring + slot * SLOT_BYTES;
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const uint4 g4 = ld_shared_v4(mine + b * 1024), u4 = ld_shared_v4(mine + b * 1024 + 512);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const uint4 x4 = *reinterpret_cast<const uint4*>(x_at[nt] + k * x_step[nt] + b * 64);
        mma16<T>(acc[nt], g4.x, u4.x, g4.y, u4.y, x4.x, x4.y);
        mma16<T>(acc[nt], g4.z, u4.z, g4.w, u4.w, x4.z, x4.w);
      }
    }
    fetch(slot == 0 ? DEPTH - 1 : slot - 1);  // the slot that was read one step ago
    if (++slot == DEPTH) slot = 0;
    if (++k == steps) {  // the end of a row tile
      put(entered ? 0 : 1);
      if (!entered) {
#pragma unroll 1
        for (int j = lane; j < live; j += 32) keep(u, j, parts[1][warp][sum_at(j)], parts[1][warp][sum_at(j) + 8]);
        __syncwarp();
      }
      entered = false;
      k = 0;
      ++u;
    }
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  if (begin == end || k != 0) put(begin == end || entered ? 0 : 1);  // without a share: zeros
  __syncthreads();
  // Row tiles that several warps share, each known by the warp that has begun it and left it to others: 32 elements at a time, by all
  // warps in turn.
  const int batches = (live + 31) / 32;
#pragma unroll 1
  for (int i = warp; i < WARPS * batches; i += WARPS) {
    const int w0 = i / batches, j = (i - w0 * batches) * 32 + lane;
    const int first = static_cast<int>(share * w0 / WARPS), left = static_cast<int>(share * (w0 + 1) / WARPS), tail = left / steps, start = tail * steps;
    if (left == start || first == left || first > start || j >= live) continue;
    float g = parts[1][w0][sum_at(j)], v = parts[1][w0][sum_at(j) + 8];
#pragma unroll 4
    for (int w = w0 + 1; w < WARPS && static_cast<int>(share * w / WARPS) < start + steps; ++w) {
      g += parts[0][w][sum_at(j)];
      v += parts[0][w][sum_at(j) + 8];
    }
    keep(tail, j, g, v);
  }
  if (split > 1) {
    cluster_sync_all();  // every CTA's sums are there
    const uint32_t mine = smem_u32(sums);
    for (int i = rank * ROWS_THREADS + threadIdx.x; i < units * live; i += split * ROWS_THREADS) {
      const int row_tile = i / live, j = i - row_tile * live;
      float g = 0.f, v = 0.f;
      for (int s = 0; s < split; ++s) {
        const uint32_t from = mapa_shared(mine, s) + (row_tile * SUMS + sum_at(j)) * 4;
        g += load_cluster(from);
        v += load_cluster(from + 32);
      }
      store(row_tile, j, g, v);
    }
    cluster_sync_all();  // none leaves while another reads it
  }
}

constexpr int rows_fixed_bytes(int nt) { return 2 * WARPS * 16 * 8 * nt * 4 + 256 + 128; }
template <typename T, int NT> static int launch_rows(const RowsParams& p, int grid, size_t smem, cudaStream_t st) {
  auto kernel = rows_kernel<T, NT>;
  static DeviceOnce limit;
  if (int rc = limit.raise_smem(reinterpret_cast<const void*>(kernel), SMEM_LIMIT - rows_fixed_bytes(NT))) return rc;
  return launch_kernel("gated linear", reinterpret_cast<const void*>(kernel), dim3((unsigned)grid), dim3(ROWS_THREADS), smem, st, p.split, true, p);
}

int run_rows(const RowsCall& call, int dtype, cudaStream_t st) {
  RowsParams p{};
  p.c = call;
  const int units = call.F / TILE_F, nt = call.M > 8 ? 2 : 1;
  p.steps = (call.K + STEP - 1) / STEP;
  p.x_at = WARPS * DEPTH * SLOT_BYTES;
  int clusters = 1;
  auto plan = [&](int split) -> int64_t {
    clusters = std::min(units, cluster_room(split));
    p.split = split;
    p.units_each = units / clusters;
    p.units_over = units % clusters;
    const int64_t pitch = (int64_t)((p.steps + split - 1) / split) * (STEP * 2) + 64;
    const int64_t bytes = p.x_at + call.M * pitch + (split > 1 ? (int64_t)(p.units_each + 1) * (16 * 8 * nt * 4) : 0);
    if (bytes > SMEM_LIMIT - rows_fixed_bytes(nt)) return 0;
    p.pitch = (int)pitch;
    p.sums_at = (int)(p.x_at + call.M * pitch);
    return bytes;
  };
  int split = 1;
  while (split < 8 && 2 * split * units <= sm_count() && 2 * split <= p.steps) split *= 2;
  int64_t smem = 0;
  while ((smem = plan(split)) == 0 && split < 8 && 2 * split <= p.steps) split *= 2;
  if (smem == 0) return KSB_ERR_UNSUPPORTED;
  const int grid = clusters * split;
  if (dtype == KSB_BF16) return nt == 1 ? launch_rows<__nv_bfloat16, 1>(p, grid, smem, st) : launch_rows<__nv_bfloat16, 2>(p, grid, smem, st);
  return nt == 1 ? launch_rows<__half, 1>(p, grid, smem, st) : launch_rows<__half, 2>(p, grid, smem, st);
}

}  // namespace gated
}  // namespace ksb
