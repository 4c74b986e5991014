// The gated half of a feed-forward block, and its gradients, in 16-bit floating point on the Blackwell tensor cores:
//
//   g = x Wg^T + bg,  u = x Wu^T + bu,  h = act(g) u            act: SiLU or the tanh form of GELU, both v sigmoid(w(v))
//   dg = dh u act'(g),  du = dh act(g)
//   dx = dg Wg + du Wu,  dWg = dg^T x,  dWu = du^T x,  dbg = sum of dg over rows,  dbu = sum of du
//
// Tensor-bound (4 M F K flop forward, 8 M F K more for the gradients) except for few rows, which only stream the weights.
//
// One persistent kernel does all three kinds of products: a few threads, one per box of a stage, copy tiles of A and B by TMA into a ring
// of stages (with one thread for all boxes the weights' gradients, of up to 6 boxes a stage, took a seventh longer), one thread issues
// tcgen05.mma (kind::f16, fp32 accumulators in tensor memory, two of them so that one tile's output overlaps the next one's
// products), the other warps take the accumulator through registers and shared memory to TMA stores.
//   PROJECT  A = x, B = rows of Wg and, behind them, the same rows of Wu: a thread of the output holds g and u of the same element.
//            In a CTA pair (cta_group::2, 256 x 256 tiles) the even CTA brings the rows of Wg, the odd one those of Wu.
//   DX       two runs over F into one accumulator: A = dg, du as they lie, B = Wg, Wu read column by column (MN-major)
//   DW       two problems of one launch: A = dg, du and B = x, all read column by column
// The gradients of few output tiles with a long sum are split over it: each part leaves its fp32 accumulators in the workspace, and join_kernel
// adds them up in the order of the sum.
// A column-wise operand needs no transposed copy: a box of 64 columns x 64 rows lands in the layout that the tensor core reads as
// MN-major with 128-byte swizzle.
//
// Measured (bf16): 32760 x 1536 -> 8960 1155 us (1560 TFLOP/s, the library's product alone 1450; 1390 us once the card is at its power limit);
// forward and backward pass of 16380 x 5120 x 13824 11.4 - 12.1 ms (1150 - 1220 TFLOP/s, at the power limit).  8192 x 4096 x 4096 1432 (with what the
// backward pass is kept), dx 1494, weights' gradients 1492 TFLOP/s: operands that are read column by column cost nothing.  A pair's step of 64
// columns takes 0.36 - 0.37 us whether its tile is 256, 224 or 192 wide (512 x 4096 x 10240), so narrower tiles for even waves gained 3 % at best.
// 77 x 4096 x 10240 34 us, where the weights alone are 26: a product of 128 rows costs some 115 cycles however few its columns are, so
// tiles of as many columns as there are CTAs for are taken (FLEX).
#include <algorithm>

#include "gated.h"
#include "host_utils.h"

namespace ksb {
namespace gated {

constexpr int KERNEL_ID = 5;
constexpr int BM = 128, BK = 64, ROW_BYTES = BK * 2;  // a stage holds 64 columns of the sum: 128-byte rows
enum Kind : int { PROJECT = 0, DX = 1, DW = 2 };

// KIND: above.  CTAS: 1, or 2 = CTA pairs.  TN: columns of a tile's accumulator (PROJECT: half of them g, half u).  FLEX (PROJECT, single
// CTAs): at most TN columns, how many is the launch's choice.
template <int KIND, int CTAS, int TN, bool FLEX> struct Cfg {
  static constexpr int OUT_N = KIND == PROJECT ? TN / 2 : TN;  // columns of the output
  // PROJECT: pieces of 32 columns, since a warp's way through a piece (two accumulators, the activation, with `save` three stores one after the
  // other) is as long as a main loop of K = 1536; a half's piece, and a byte's
  static constexpr int PIECE_COLS = KIND == PROJECT ? 32 : 64, PIECE_BYTES = 32 * PIECE_COLS * (KIND == PROJECT ? 3 : 2);
  static constexpr int EW = FLEX ? 4 : 4 * (OUT_N / PIECE_COLS);  // output warps
  static constexpr int LOADS = KIND == PROJECT ? (CTAS == 2 ? 2 : 3) : KIND == DX ? 1 + TN / CTAS / 64 : 2 + TN / CTAS / 64;  // TMA boxes per stage
  static constexpr int THREADS = 32 * (LOADS + 1 + EW);
  static constexpr int A_BYTES = BM * ROW_BYTES, B_ROWS = TN / CTAS, B_BYTES = B_ROWS * ROW_BYTES, STAGE_BYTES = A_BYTES + B_BYTES;
  static constexpr int OUT_BYTES = FLEX ? 0 : EW * PIECE_BYTES;
  static constexpr int BIAS_COLS = FLEX ? TN / 2 : PIECE_COLS;                          // of an output warp
  static constexpr int BIAS_BYTES = KIND == PROJECT ? EW * 2 * BIAS_COLS * 4 : 0;
  static constexpr int MOST = FLEX ? 10 : 6;  // stages
  static constexpr int ROOM = 232448 - OUT_BYTES - BIAS_BYTES - (2 * MOST + 4) * 8 - 16;
  static constexpr int STAGES = ROOM / STAGE_BYTES > MOST ? MOST : ROOM / STAGE_BYTES;
  static constexpr int TMEM_COLS = 2 * TN;
  // [stages x (A | B)][output pieces][biases][barriers]
  static constexpr int SMEM_BYTES = FLEX ? 232448 : STAGES * STAGE_BYTES + OUT_BYTES + BIAS_BYTES + (2 * STAGES + 4) * 8 + 16;
  static_assert(SMEM_BYTES <= 232448 && STAGES >= 3, "shared memory");
};

struct Params {
  CUtensorMap a[2], b[2], out[5];  // PROJECT with `save`: h, upper and lower part of g, of u
  int M, N;                       // of the output
  int tiles_m, tiles_n, num_tiles, problem_tiles;
  int steps, num_k;               // stages per run over the sum, and over all of it
  int splits;                     // parts of the sum (gradients)
  float* parts;                   // with several: [problem][part][tile][CTA of a pair][four columns][128 rows] float4
  int group_m;                    // row tiles that go through all columns together
  const void* b_gate;             // PROJECT: halves or null
  const void* b_up;
  int act, save;                  // PROJECT: save g and u as well
  int flex_cols, stages;          // FLEX: columns of the output per tile, stages
  void* h;                        // FLEX
  int* status;
};

__device__ __forceinline__ uint64_t mn_major_desc(uint32_t smem_addr) {
  // blocks of 64 rows of the operand 8192 bytes apart (leading offset), groups of 8 columns of the sum 1024 bytes apart (stride offset)
  uint64_t d = static_cast<uint64_t>((smem_addr & 0x3ffff) >> 4);
  d |= static_cast<uint64_t>(8192 >> 4) << 16;
  d |= static_cast<uint64_t>(1024 >> 4) << 32;
  d |= static_cast<uint64_t>(1) << 46;
  d |= static_cast<uint64_t>(2) << 61;
  return d;
}
// both operands of one type (0 = fp16, 1 = bf16), fp32 accumulator; bits 15 and 16: A, B column by column
template <typename T> struct MmaType;
template <> struct MmaType<__half> { static constexpr uint32_t value = 0; };
template <> struct MmaType<__nv_bfloat16> { static constexpr uint32_t value = 1; };

__device__ __forceinline__ void mma_f16_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// 16 consecutive columns
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]),
        "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}

__device__ __forceinline__ void tmem_ld8(uint32_t taddr, uint32_t (&r)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]) : "r"(taddr) : "memory");
}

// g and u are kept for the backward pass as the upper 24 bits of their fp32 values, rounded (a plane of the upper 16, one of the next 8):
// kept in the half type they would put as much into the gradients' error as the rounding of dg and du that the tensor cores ask for.
__device__ __forceinline__ uint32_t round24(float v) { return v != v ? 0x7fc00000u : __float_as_uint(v) + 0x80u; }
__device__ __forceinline__ uint32_t high2(const uint32_t* r) { return __byte_perm(r[0], r[1], 0x7632); }
__device__ __forceinline__ uint32_t low4(const uint32_t* r) { return __byte_perm(__byte_perm(r[0], r[1], 0x0051), __byte_perm(r[2], r[3], 0x0051), 0x5410); }
// eight of them back
__device__ __forceinline__ void from24(const uint4& high, const uint2& low, float (&v)[8]) {
  const uint32_t h[4] = {high.x, high.y, high.z, high.w}, l[2] = {low.x, low.y};
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    v[i] = __uint_as_float(h[i / 2] << 16 | (l[i / 4] >> (i % 4 * 8) & 0xffu) << 8);
    v[i + 1] = __uint_as_float((h[i / 2] & 0xffff0000u) | (l[i / 4] >> (i % 4 * 8 + 8) & 0xffu) << 8);
  }
}
struct Saved {  // offsets of the planes, bytes
  int64_t low_ld, low, u, bytes;
};
static Saved saved_layout(int64_t M, int64_t F) {
  Saved s;
  s.low_ld = (F + 15) / 16 * 16;
  s.low = (M * F * 2 + 255) / 256 * 256;
  s.u = s.low + (M * s.low_ld + 255) / 256 * 256;
  s.bytes = 2 * s.u;
  return s;
}

// A piece of work: an output tile, and the part [k0, k1) of the sum.
struct Work {
  int problem, tm, tn, k0, k1;
};
__device__ __forceinline__ Work work_of(const Params& p, int tile) {
  Work w;
  const int part = tile / p.problem_tiles;
  w.problem = part / p.splits;
  const int split = part - w.problem * p.splits;
  w.k0 = static_cast<int>(static_cast<int64_t>(p.num_k) * split / p.splits);
  w.k1 = static_cast<int>(static_cast<int64_t>(p.num_k) * (split + 1) / p.splits);
  tile -= part * p.problem_tiles;
  const int per_group = p.group_m * p.tiles_n, rg = tile / per_group, first = rg * p.group_m;
  const int rows = min(p.group_m, p.tiles_m - first), r = tile - rg * per_group;
  w.tm = first + r % rows;
  w.tn = r / rows;
  return w;
}

template <typename T, int KIND, int CTAS, int TN, bool FLEX>
__global__ void __launch_bounds__(Cfg<KIND, CTAS, TN, FLEX>::THREADS, 1) gemm_kernel(const __grid_constant__ Params p) {
  using C = Cfg<KIND, CTAS, TN, FLEX>;
  const int OUT_N = FLEX ? p.flex_cols : C::OUT_N;
  const uint32_t STAGES = FLEX ? p.stages : C::STAGES, B_BYTES = FLEX ? p.flex_cols * 2 * ROW_BYTES : C::B_BYTES, STAGE_BYTES = C::A_BYTES + B_BYTES;
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t base = smem_u32(smem);
  const uint32_t pieces = base + STAGES * STAGE_BYTES, biases = pieces + C::OUT_BYTES, bars = biases + C::BIAS_BYTES;
  const uint32_t full0 = bars, empty0 = full0 + 8 * STAGES, tfull0 = empty0 + 8 * STAGES, tempty0 = tfull0 + 16, tmem_slot = tempty0 + 16;
  volatile uint32_t* tmem_slot_gen = reinterpret_cast<volatile uint32_t*>(smem + (tmem_slot - base));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t crank = CTAS == 2 ? cluster_ctarank() : 0u;
  const int worker = CTAS == 2 ? blockIdx.x >> 1 : blockIdx.x, workers = CTAS == 2 ? gridDim.x >> 1 : gridDim.x;
  if ((base & 1023u) != 0) {  // uniform over the grid
    if (threadIdx.x == 0) report_error(p.status, KSB_ERR_BAD_SMEM_ALIGNMENT, (KERNEL_ID << 16) | 99);
    return;
  }
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(full0 + 8 * s, C::LOADS);  // the loaders' expecting arrivals (of the even CTA in a pair) + the bytes
      mbar_init(empty0 + 8 * s, 1);         // one commit
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(tfull0 + 8 * a, 1);
      mbar_init(tempty0 + 8 * a, C::EW * CTAS);
    }
    fence_barrier_init();
  }
  if (warp == C::LOADS) {
    if (CTAS == 2) {
      tmem_alloc_pair(tmem_slot, C::TMEM_COLS);
      tmem_relinquish_pair();
    } else {
      tmem_alloc(tmem_slot, C::TMEM_COLS);
      tmem_relinquish();
    }
  }
  tc_fence_before();
  __syncthreads();
  if (CTAS == 2) cluster_sync_all();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot_gen;

  if (warp < C::LOADS) {
    // ------------------------------------------------------------------ loads: box `warp` of every stage
    if (lane == 0) {
      constexpr int A_BOXES = KIND == DW ? 2 : 1, B_BOXES = C::LOADS - A_BOXES;
      const uint32_t BOX_A = C::A_BYTES / A_BOXES, BOX_B = B_BYTES / B_BOXES;
      const bool of_a = warp < A_BOXES;
      const int box = of_a ? warp : warp - A_BOXES;
      const uint32_t bytes = of_a ? BOX_A : BOX_B, offset = of_a ? box * BOX_A : C::A_BYTES + box * BOX_B;
      pdl_wait();
      uint32_t it = 0, s = 0, ph = 1;
      bool ok = true;
      for (int tile = worker; tile < p.num_tiles && ok; tile += workers) {
        const Work w = work_of(p, tile);
        const int row = (w.tm * CTAS + (int)crank) * BM, col = w.tn * TN + (int)crank * C::B_ROWS;
        for (int k = w.k0; k < w.k1; ++k, ++it) {
          if (!mbar_wait(empty0 + 8 * s, ph, p.status, (KERNEL_ID << 16) | 1)) { ok = false; break; }
          if (CTAS == 1) mbar_arrive_expect_tx(full0 + 8 * s, bytes);
          else if (crank == 0) mbar_arrive_expect_tx(full0 + 8 * s, 2 * bytes);
          const int run = KIND == DX && k >= p.steps;
          const int kk = (run ? k - p.steps : k) * BK;
          const CUtensorMap* map;
          int x, y;
          if (of_a) {
            map = &p.a[KIND == DW ? w.problem : run];
            x = KIND == DW ? row + 64 * box : kk;
            y = KIND == DW ? kk : row;
          } else {
            map = &p.b[KIND == PROJECT ? (CTAS == 2 ? (int)crank : box) : run];
            x = KIND == PROJECT ? kk : col + 64 * box;
            y = KIND == PROJECT ? w.tn * OUT_N : kk;
          }
          const uint32_t dst = base + s * STAGE_BYTES + offset;
          if (CTAS == 2) tma_load_2d_pair(dst, map, mapa_shared(full0 + 8 * s, 0), x, y);
          else tma_load_2d(dst, map, full0 + 8 * s, x, y);
          if (++s == STAGES) {
            s = 0;
            ph ^= 1;
          }
        }
      }
      // what is on its way lands before the block leaves (of a pair, the even CTA hears of it)
      if (crank == 0)
        for (uint32_t i = it > STAGES ? it - STAGES : 0; i < it; ++i)
          if (!mbar_wait(full0 + 8 * (i % STAGES), (i / STAGES) & 1, p.status, (KERNEL_ID << 16) | 5)) break;
    }
  } else if (warp == C::LOADS) {
    // ------------------------------------------------------------------ products (in a pair: the even CTA's)
    if (lane == 0 && crank == 0) {
      constexpr bool a_mn = KIND == DW, b_mn = KIND != PROJECT;
      const uint32_t idesc = make_idesc(1, MmaType<T>::value, MmaType<T>::value, CTAS * BM, FLEX ? 2 * OUT_N : TN) | (a_mn ? 1u << 15 : 0u) | (b_mn ? 1u << 16 : 0u);
      uint32_t s = 0, ph = 0, count = 0;
      bool ok = true;
      for (int tile = worker; tile < p.num_tiles && ok; tile += workers, ++count) {
        const uint32_t acc = count & 1, aph = (count >> 1) & 1;
        if (!mbar_wait(tempty0 + 8 * acc, aph ^ 1, p.status, (KERNEL_ID << 16) | 2)) break;
        tc_fence_after();
        const uint32_t d = tmem_base + acc * TN;
        const Work w = work_of(p, tile);
        for (int k = w.k0; k < w.k1; ++k) {
          if (!mbar_wait(full0 + 8 * s, ph, p.status, (KERNEL_ID << 16) | 3)) { ok = false; break; }
          tc_fence_after();
          const uint32_t sa = base + s * STAGE_BYTES, sb = sa + C::A_BYTES;
          const uint64_t da = a_mn ? mn_major_desc(sa) : make_kmajor_sw128_desc(sa), db = b_mn ? mn_major_desc(sb) : make_kmajor_sw128_desc(sb);
#pragma unroll
          for (int kk = 0; kk < BK / 16; ++kk) {  // 16 columns of the sum: 32 bytes of a row, or 16 rows of 128 bytes
            const uint64_t ak = da + kk * (a_mn ? 128 : 2), bk = db + kk * (b_mn ? 128 : 2);
            if (CTAS == 2) mma_f16_pair(d, ak, bk, idesc, k != w.k0 || kk != 0);
            else mma_bf16_ss(d, ak, bk, idesc, k != w.k0 || kk != 0);
          }
          if (CTAS == 2) mma_commit_pair(empty0 + 8 * s); else mma_commit(empty0 + 8 * s);
          if (++s == STAGES) {
            s = 0;
            ph ^= 1;
          }
        }
        if (ok) {
          if (CTAS == 2) mma_commit_pair(tfull0 + 8 * acc); else mma_commit(tfull0 + 8 * acc);
        }
      }
    }
  } else {
    // ------------------------------------------------------------------ output
    pdl_wait();
    pdl_release();
    const int q = warp & 3, ew = warp - C::LOADS - 1, col0 = (ew >> 2) * C::PIECE_COLS;  // lanes of tensor memory; the warp's columns of a tile
    const uint32_t piece = pieces + ew * C::PIECE_BYTES;
    constexpr int UNITS = C::PIECE_COLS / 8;  // of 16 bytes in a row of a piece, swizzled as the tensor map has it
    const int swizzle = UNITS == 8 ? lane & 7 : (lane >> 1) & 3;
    const uint32_t piece_row = piece + lane * (C::PIECE_COLS * 2);
    const uint32_t tempty_even = CTAS == 2 ? mapa_shared(tempty0, 0) : 0u;
    uint32_t count = 0;
    for (int tile = worker; tile < p.num_tiles; tile += workers, ++count) {
      const Work w = work_of(p, tile);
      const uint32_t acc = count & 1, aph = (count >> 1) & 1;
      const int row0 = (w.tm * CTAS + (int)crank) * BM + q * 32, n0 = w.tn * OUT_N + col0;
      // The biases of the warp's columns, as fp32, ahead of the accumulator: read behind it, column by column, they took 5 us of
      // 77 x 4096 x 10240.
      const uint32_t bias_at = biases + ew * (2 * C::BIAS_COLS * 4);
      if (KIND == PROJECT) {
#pragma unroll
        for (int c = lane; c < 2 * C::BIAS_COLS; c += 32) {
          const int which = c / C::BIAS_COLS, col = n0 + c % C::BIAS_COLS;
          const void* bias = which ? p.b_up : p.b_gate;
          const float f = bias && col < p.N ? HalfOps<T>::to_f(static_cast<const T*>(bias)[col]) : 0.f;
          asm volatile("st.shared.f32 [%0], %1;" ::"r"(bias_at + c * 4), "f"(f) : "memory");
        }
        __syncwarp();
      }
      if (!mbar_wait_warp(tfull0 + 8 * acc, aph, p.status, (KERNEL_ID << 16) | 4)) break;
      tc_fence_after();
      if (row0 < p.M && n0 < p.N) {  // uniform over the warp
        const uint32_t t_row = tmem_base + acc * TN + (static_cast<uint32_t>(q * 32) << 16) + col0;
        auto take16 = [&](uint32_t at, float (&v)[16]) {
          uint32_t w[16];
          tmem_ld16(at, w);
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(w[i]);
        };
        auto put = [&](int c, const float (&y)[8]) {
          st_shared_v4(piece_row + (((c >> 3) ^ swizzle) << 4), make_uint4(HalfOps<T>::pack2(make_float2(y[0], y[1])), HalfOps<T>::pack2(make_float2(y[2], y[3])),
                                                                          HalfOps<T>::pack2(make_float2(y[4], y[5])), HalfOps<T>::pack2(make_float2(y[6], y[7]))));
        };
        auto open = [&]() {  // the piece's last store has read it
          if (lane == 0) bulk_wait_source_read<0>();
          __syncwarp();
        };
        auto close = [&](const CUtensorMap* map) {
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) tma_store_2d(map, piece, n0, row0);
        };
        if (KIND == PROJECT) {
          // eight columns with their bias
          auto with_bias = [&](const float* v, int up, int c, float (&y)[8]) {
            const uint4 a = ld_shared_v4(bias_at + (up * C::BIAS_COLS + c) * 4), b = ld_shared_v4(bias_at + (up * C::BIAS_COLS + c) * 4 + 16);
            y[0] = v[0] + __uint_as_float(a.x); y[1] = v[1] + __uint_as_float(a.y); y[2] = v[2] + __uint_as_float(a.z); y[3] = v[3] + __uint_as_float(a.w);
            y[4] = v[4] + __uint_as_float(b.x); y[5] = v[5] + __uint_as_float(b.y); y[6] = v[6] + __uint_as_float(b.z); y[7] = v[7] + __uint_as_float(b.w);
          };
          if constexpr (FLEX) {
            // few rows: straight to memory
            const int row = row0 + lane;
            for (int c = 0; c < OUT_N; c += 8) {
              uint32_t v[8], w[8];
              __syncwarp();  // lanes without a row come from the last turn by another way, and the loads are the whole warp's
              tmem_ld8(t_row + c, v);
              tmem_ld8(t_row + OUT_N + c, w);
              tmem_wait_ld();
              if (row >= p.M || n0 + c >= p.N) continue;
              float fv[8], fw[8], g[8], u[8];
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                fv[i] = __uint_as_float(v[i]);
                fw[i] = __uint_as_float(w[i]);
              }
              with_bias(fv, 0, c, g);
              with_bias(fw, 1, c, u);
#pragma unroll
              for (int i = 0; i < 8; ++i) g[i] = g[i] * act_sigmoid(g[i], p.act) * u[i];
              *reinterpret_cast<uint4*>(static_cast<T*>(p.h) + static_cast<int64_t>(row) * p.N + n0 + c) =
                  make_uint4(HalfOps<T>::pack2(make_float2(g[0], g[1])), HalfOps<T>::pack2(make_float2(g[2], g[3])), HalfOps<T>::pack2(make_float2(g[4], g[5])),
                             HalfOps<T>::pack2(make_float2(g[6], g[7])));
            }
          } else {
          if (p.save) {
            // the upper 24 bits of each fp32 value, as two planes
            const uint32_t low_row = piece + 32 * C::PIECE_COLS * 2 + lane * C::PIECE_COLS;
#pragma unroll 1
            for (int up = 0; up < 2; ++up) {
              open();
#pragma unroll
              for (int c = 0; c < C::PIECE_COLS; c += 16) {
                float v[16];
                take16(t_row + up * (TN / 2) + c, v);
                uint32_t r[16];
#pragma unroll
                for (int e = 0; e < 16; e += 8) {
                  float y[8];
                  with_bias(v + e, up, c + e, y);
#pragma unroll
                  for (int i = 0; i < 8; ++i) r[e + i] = round24(y[i]);
                  st_shared_v4(piece_row + ((((c + e) >> 3) ^ swizzle) << 4), make_uint4(high2(r + e), high2(r + e + 2), high2(r + e + 4), high2(r + e + 6)));
                }
                st_shared_v4(low_row + c, make_uint4(low4(r), low4(r + 4), low4(r + 8), low4(r + 12)));
              }
              close(&p.out[1 + 2 * up]);
              if (lane == 0) tma_store_2d(&p.out[2 + 2 * up], piece + 32 * C::PIECE_COLS * 2, n0, row0);
            }
          }
          open();
#pragma unroll
          for (int c = 0; c < C::PIECE_COLS; c += 16) {
            float v[16], w[16];
            take16(t_row + c, v);
            take16(t_row + TN / 2 + c, w);
#pragma unroll
            for (int e = 0; e < 16; e += 8) {
              float g[8], u[8];
              with_bias(v + e, 0, c + e, g);
              with_bias(w + e, 1, c + e, u);
#pragma unroll
              for (int i = 0; i < 8; ++i) g[i] = g[i] * act_sigmoid(g[i], p.act) * u[i];
              put(c + e, g);
            }
          }
          close(&p.out[0]);
          }
        } else if (p.splits > 1) {
          float4* to = reinterpret_cast<float4*>(p.parts) + (static_cast<int64_t>(tile) * CTAS + crank) * (BM * TN / 4) + q * 32 + lane;
#pragma unroll
          for (int c = 0; c < C::PIECE_COLS; c += 16) {
            float v[16];
            take16(t_row + c, v);
#pragma unroll
            for (int i = 0; i < 4; ++i) to[((col0 + c) / 4 + i) * BM] = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
          }
        } else {
          open();
#pragma unroll
          for (int c = 0; c < C::PIECE_COLS; c += 16) {
            float v[16];
            take16(t_row + c, v);
#pragma unroll
            for (int e = 0; e < 16; e += 8) {
              float y[8];
#pragma unroll
              for (int i = 0; i < 8; ++i) y[i] = v[e + i];
              put(c + e, y);
            }
          }
          close(&p.out[w.problem]);
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if (CTAS == 2) mbar_arrive_cluster_relaxed(tempty_even + 8 * acc); else mbar_arrive(tempty0 + 8 * acc);
      }
    }
    bulk_wait_all();  // no store of this thread may outlive the kernel's shared memory
  }

  // ------------------------------------------------------------------ common exit
  tc_fence_before();
  __syncthreads();
  if (CTAS == 2) cluster_sync_all();
  if (warp == C::LOADS) {
    tc_fence_after();
    if (CTAS == 2) tmem_dealloc_pair(tmem_base, C::TMEM_COLS); else tmem_dealloc(tmem_base, C::TMEM_COLS);
  }
}

// The outputs of a split launch: a warp adds up 32 rows x 16 columns of the parts, in their order, a row per lane.
struct JoinParams {
  Params p;
  void* out[2];
  int problems, ctas, tile_cols;  // as the products' launch had them
};
template <typename T> __global__ void __launch_bounds__(256) join_kernel(const __grid_constant__ JoinParams j) {
  const Params& p = j.p;
  pdl_wait();
  pdl_release();
  const int lane = threadIdx.x & 31, groups = j.tile_cols / 16, per_tile = j.ctas * 4 * groups;  // of 16 columns
  const int64_t total = static_cast<int64_t>(j.problems) * p.problem_tiles * per_tile, tile_floats = static_cast<int64_t>(j.ctas) * BM * j.tile_cols;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5); i < total; i += static_cast<int64_t>(gridDim.x) * 8) {
    const int64_t t = i / per_tile;
    const int r = static_cast<int>(i - t * per_tile), crank = r / (4 * groups), q = r / groups % 4, g = r % groups;
    const int problem = static_cast<int>(t / p.problem_tiles);
    const int64_t first = static_cast<int64_t>(problem) * p.splits * p.problem_tiles + (t - static_cast<int64_t>(problem) * p.problem_tiles);  // its first part
    const Work w = work_of(p, static_cast<int>(first));
    const int row = (w.tm * j.ctas + crank) * BM + q * 32 + lane, col = w.tn * j.tile_cols + g * 16;
    if (col >= p.N) continue;
    const float4* from = reinterpret_cast<const float4*>(p.parts + first * tile_floats) + crank * (BM * j.tile_cols / 4) + g * 4 * BM + q * 32 + lane;
    float4 v[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) v[c] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (row < p.M) {
#pragma unroll 2
      for (int s = 0; s < p.splits; ++s, from += static_cast<int64_t>(p.problem_tiles) * tile_floats / 4)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const float4 f = from[c * BM];
          v[c].x += f.x;
          v[c].y += f.y;
          v[c].z += f.z;
          v[c].w += f.w;
        }
      T* to = static_cast<T*>(j.out[problem]) + static_cast<int64_t>(row) * p.N + col;
#pragma unroll
      for (int h = 0; h < 2; ++h)
        if (col + 8 * h < p.N)
          *reinterpret_cast<uint4*>(to + 8 * h) = make_uint4(HalfOps<T>::pack2(make_float2(v[2 * h].x, v[2 * h].y)), HalfOps<T>::pack2(make_float2(v[2 * h].z, v[2 * h].w)),
                                                              HalfOps<T>::pack2(make_float2(v[2 * h + 1].x, v[2 * h + 1].y)), HalfOps<T>::pack2(make_float2(v[2 * h + 1].z, v[2 * h + 1].w)));
    }
  }
}

// dg and du, element by element, and a stretch of rows' sums of them: bound by HBM, 12 bytes per element.
struct ActParams {
  const void* dh;
  const uint8_t* saved;
  void* dg;
  void* du;
  float* parts;  // [row stretches][2][F], or null
  int64_t lddh, M, stretch;
  int64_t low_ld, low, u;  // planes of what is saved
  int F, act;
};
// A CTA's threads: chunks of eight columns, and takers of turns over the rows of its stretch.  One row at a time and 64 registers, for four CTAs per
// SM: 16380 x 13824 419 us (6.5 TB/s), with two rows at a time and two CTAs 597; 64 x 4 threads 423.
constexpr int ACT_COLS = 32, ACT_ROWS = 8;
template <typename T> __global__ void __launch_bounds__(ACT_COLS * ACT_ROWS, 4) act_grad_kernel(const __grid_constant__ ActParams p) {
  __shared__ __align__(16) float sums[2][ACT_ROWS][ACT_COLS * 8];
  const int c = blockIdx.x * ACT_COLS + threadIdx.x;
  const bool live = c * 8 < p.F;
  pdl_wait();
  pdl_release();
  const int64_t first = blockIdx.y * p.stretch, last = !live ? 0 : first + p.stretch < p.M ? first + p.stretch : p.M;
  float sg[8], su[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) sg[i] = su[i] = 0.f;
#pragma unroll 1
  for (int64_t row = first + threadIdx.y; row < last; row += ACT_ROWS) {
    const int64_t at = row * p.F + c * 8;
    const uint4 dv = *reinterpret_cast<const uint4*>(static_cast<const T*>(p.dh) + row * p.lddh + c * 8);
    const uint8_t *hp = p.saved + at * 2, *lp = p.saved + p.low + row * p.low_ld + c * 8;
    float gf[8], uf[8];
    from24(*reinterpret_cast<const uint4*>(hp), *reinterpret_cast<const uint2*>(lp), gf);
    from24(*reinterpret_cast<const uint4*>(hp + p.u), *reinterpret_cast<const uint2*>(lp + p.u), uf);
    const uint32_t dw[4] = {dv.x, dv.y, dv.z, dv.w};
    uint32_t og[4], ou[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 d = HalfOps<T>::unpack2(dw[i]), g = make_float2(gf[2 * i], gf[2 * i + 1]), u = make_float2(uf[2 * i], uf[2 * i + 1]);
      const float sx = act_sigmoid(g.x, p.act), sy = act_sigmoid(g.y, p.act);
      const float2 dg = make_float2(d.x * u.x * act_slope(g.x, sx, p.act), d.y * u.y * act_slope(g.y, sy, p.act));
      const float2 du = make_float2(d.x * g.x * sx, d.y * g.y * sy);
      og[i] = HalfOps<T>::pack2(dg);
      ou[i] = HalfOps<T>::pack2(du);
      sg[2 * i] += dg.x;
      sg[2 * i + 1] += dg.y;
      su[2 * i] += du.x;
      su[2 * i + 1] += du.y;
    }
    *reinterpret_cast<uint4*>(static_cast<T*>(p.dg) + at) = make_uint4(og[0], og[1], og[2], og[3]);
    *reinterpret_cast<uint4*>(static_cast<T*>(p.du) + at) = make_uint4(ou[0], ou[1], ou[2], ou[3]);
  }
  if (p.parts) {  // the CTA's sums of its stretch, in the order of the turns
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float* v = h ? su : sg;
      float4* at = reinterpret_cast<float4*>(&sums[h][threadIdx.y][threadIdx.x * 8]);
      at[0] = make_float4(v[0], v[1], v[2], v[3]);
      at[1] = make_float4(v[4], v[5], v[6], v[7]);
    }
    __syncthreads();
    float* to = p.parts + static_cast<int64_t>(blockIdx.y) * 2 * p.F;
    for (int i = threadIdx.y * ACT_COLS + threadIdx.x; i < 2 * ACT_COLS * 8; i += ACT_COLS * ACT_ROWS) {
      const int h = i / (ACT_COLS * 8), j = i - h * (ACT_COLS * 8), col = blockIdx.x * (ACT_COLS * 8) + j;
      float v = 0.f;
#pragma unroll
      for (int y = 0; y < ACT_ROWS; ++y) v += sums[h][y][j];
      if (col < p.F) to[static_cast<int64_t>(h) * p.F + col] = v;
    }
  }
}
// The bias gradients from the stretches' sums, in their order: 32 columns and 32 takers of turns per CTA.
constexpr int TAKERS = 32;
template <typename T> __global__ void __launch_bounds__(32 * TAKERS) bias_grad_kernel(const float* parts, int stretches, int F, void* dbg, void* dbu) {
  __shared__ float sums[TAKERS][33];
  const int lane = threadIdx.x & 31, j = threadIdx.x >> 5;
  const int64_t cols = 2 * static_cast<int64_t>(F), col = static_cast<int64_t>(blockIdx.x) * 32 + lane;
  pdl_wait();
  pdl_release();
  float s = 0.f;
  if (col < cols)
#pragma unroll 4
    for (int i = j; i < stretches; i += TAKERS) s += parts[i * cols + col];
  sums[j][lane] = s;
  __syncthreads();
  if (j != 0 || col >= cols) return;
  s = 0.f;
#pragma unroll
  for (int i = 0; i < TAKERS; ++i) s += sums[i][lane];
  void* to = col < F ? dbg : dbu;
  if (to) static_cast<T*>(to)[col < F ? col : col - F] = HalfOps<T>::from_f(s);
}

// ---------------------------------------------------------------------------------------------------------------- host side

struct Operand {
  const void* ptr;
  int64_t rows, cols, ld;
};
static int map_of(CUtensorMap* m, const Operand& o, int box_cols, int box_rows, int elem = 2) {
  return encode_tmap_2d(m, elem == 2 ? CU_TENSOR_MAP_DATA_TYPE_UINT16 : CU_TENSOR_MAP_DATA_TYPE_UINT8, elem, o.ptr, (uint64_t)o.cols, (uint64_t)o.rows, (uint64_t)o.ld * elem,
                        (uint32_t)box_cols, (uint32_t)box_rows);
}

template <typename T, int KIND, int CTAS, int TN, bool FLEX> static int launch_as(const Params& p, bool chained, cudaStream_t st) {
  using C = Cfg<KIND, CTAS, TN, FLEX>;
  auto kernel = gemm_kernel<T, KIND, CTAS, TN, FLEX>;
  static DeviceOnce smem_limit;
  if (int rc = smem_limit.raise_smem(reinterpret_cast<const void*>(kernel), C::SMEM_BYTES)) return rc;
  const int workers = std::max(1, sm_count() / CTAS), grid = CTAS * std::min(p.num_tiles, workers);
  return launch_kernel("gated linear", reinterpret_cast<const void*>(kernel), dim3((unsigned)grid), dim3(C::THREADS), C::SMEM_BYTES, st, CTAS, chained, p);
}

// A launch: operands as the kernel's kind wants them, outputs, and the columns that are summed over.
struct Job {
  Operand a[2], b[2], out[5];
  int outs;
  int64_t M, N, sum;
  int problems;
  Params p;
};

template <int KIND, int CTAS, int TN, bool FLEX = false> static int launch_form(Job& j, int dtype, bool chained, cudaStream_t st, int flex_cols = 0, int splits = 1) {
  using C = Cfg<KIND, CTAS, TN, FLEX>;
  Params& p = j.p;
  p.status = status_words();
  if (!p.status) return fail(KSB_ERR_CUDA, "status words unavailable");
  const bool a_mn = KIND == DW, b_mn = KIND != PROJECT;
  const int out_n = FLEX ? flex_cols : C::OUT_N;
  for (int i = 0; i < (KIND == PROJECT ? 1 : 2); ++i)
    if (int rc = map_of(&p.a[i], j.a[i], BK, a_mn ? BK : BM)) return rc;
  for (int i = 0; i < (KIND == DW ? 1 : 2); ++i)
    if (int rc = map_of(&p.b[i], j.b[i], BK, b_mn ? BK : out_n)) return rc;
  for (int i = 0; i < j.outs && !FLEX; ++i)
    if (int rc = map_of(&p.out[i], j.out[i], C::PIECE_COLS, 32, KIND == PROJECT && i > 0 && i % 2 == 0 ? 1 : 2)) return rc;
  p.M = (int)j.M;
  p.N = (int)j.N;
  p.tiles_m = (int)((j.M + CTAS * BM - 1) / (CTAS * BM));
  p.tiles_n = (int)((j.N + out_n - 1) / out_n);
  const int64_t tiles = (int64_t)p.tiles_m * p.tiles_n * j.problems * splits;
  if (tiles > INT32_MAX) return fail(KSB_ERR_UNSUPPORTED, "too many tiles");
  p.problem_tiles = p.tiles_m * p.tiles_n;
  p.num_tiles = (int)tiles;
  p.steps = (int)((j.sum + BK - 1) / BK);
  p.num_k = p.steps * (KIND == DX ? 2 : 1);
  p.splits = splits;
  p.flex_cols = out_n;
  p.stages = std::min<int>(C::MOST, C::ROOM / (C::A_BYTES + 2 * out_n * ROW_BYTES));  // FLEX
  // Row tiles that share each column tile's operand while it is in L2; their own operand's rows are to take about 32 MB of it.
  const int64_t row_bytes = (int64_t)CTAS * BM * p.num_k * ROW_BYTES;
  p.group_m = (int)std::max<int64_t>(KIND == DW ? 8 : 4, std::min<int64_t>(64, (32ll << 20) / row_bytes));
  return dtype == KSB_BF16 ? launch_as<__nv_bfloat16, KIND, CTAS, TN, FLEX>(p, chained, st) : launch_as<__half, KIND, CTAS, TN, FLEX>(p, chained, st);
}

static double waves(int64_t M, int64_t N, int tm, int tn, int workers, int problems) {
  return (double)((((M + tm - 1) / tm) * ((N + tn - 1) / tn) * problems + workers - 1) / workers);
}

// The form of a projection: by estimated time, waves x stages of a tile x time of a stage (us).  Pairs / 128 x 256 / free columns, us: 77 x 4096 x
// 10240 (80 tiles of pairs for 74) 51 / 39 / 33, 128 x 5120 x 13824 63 / 51 / 48, 64 x 1536 x 4096 12.8 / 15.4 / 12.4, 17 x 1536 x 8960 (one
// wave of each) 17.3 / 17.8 / 19.5; 1101 x 1536 x 4616 30 / 37, 300 x 1536 x 8960 23 / 28.
static int project(Job& j, int dtype, cudaStream_t st) {
  const int sms = sm_count();
  const double pair = sms < 2 ? 1e30 : waves(j.M, j.N, 256, 128, sms / 2, 1) * 0.285, wide = waves(j.M, j.N, 128, 128, sms, 1) * 0.40;
  double flex = 1e30;
  int cols = 0;
  if (!j.p.save && j.M <= BM)
    for (int c = 8; c <= 128; c += 8) {
      const double t = waves(j.M, j.N, 128, c, sms, 1) * std::max(0.25, 0.285 * c / 128);
      if (t <= flex) flex = t, cols = c;
    }
  if (flex < wide && flex < pair) return launch_form<PROJECT, 1, 256, true>(j, dtype, true, st, cols);
  return wide < pair ? launch_form<PROJECT, 1, 256>(j, dtype, true, st) : launch_form<PROJECT, 2, 256>(j, dtype, true, st);
}

// The form of a gradient's products, and into how many parts the sum is split.
struct GradPlan {
  int form, splits;  // 0: CTA pairs, 256 x 256; 1: 128 x 256; 2: 128 x 128
  double us;
  int64_t floats;    // of the parts
};
static GradPlan plan_gradient(int64_t M, int64_t N, int64_t num_k, int problems) {
  const int sms = sm_count();
  const struct { int tm, tn, workers; double step; } forms[3] = {{256, 256, sms / 2, 0.285}, {128, 256, sms, 0.40}, {128, 128, sms, 0.25}};
  GradPlan best{0, 1, 1e30, 0};
  for (int f = 0; f < 3; ++f) {
    if (forms[f].workers < 1) continue;
    const int64_t tiles = ((M + forms[f].tm - 1) / forms[f].tm) * ((N + forms[f].tn - 1) / forms[f].tn) * problems, tile_floats = (int64_t)forms[f].tm * forms[f].tn;
    for (int s = 1; s <= 64 && (s == 1 || num_k / s >= 8); ++s) {
      // Pairs in 1, 2, 4 parts / 128 x 256 / 128 x 128, us: dx of 300 x 1536 x 8960 95, 62, 45 / 131, 82, 54 / 79, 52, 38; of 1101 x 1536 x 4616
      // 64, 54, 60 / 84, 64, 70 / 60, 69, 65; weights' of 8192 x 256 x 512 53, 38, 31 / 61, 42, 34 / 47, 35, 29 (of more parts 28), of
      // 1101 x 1536 x 4616 48 / 48 / 54.
      // Estimated: waves x (stages of a part x time of a stage + output), and for a split the parts written and read at some 3.5 TB/s and
      // the second launch.  With one part and with this rule, the elements' gradients included: dx of 300 x 1536 x 8960 83 and 45 us, of
      // 1101 x 1536 x 4616 63 and 55.5; the weights' of 75600 x 256 x 512 396 and 147 us, of 32760 x 64 x 128 162 and 44.
      const double waves = (double)((tiles * s + forms[f].workers - 1) / forms[f].workers);
      const double us = waves * ((double)((num_k + s - 1) / s) * forms[f].step + 1.5) + (s > 1 ? 3.0 + (double)(tiles * s * tile_floats) * 8 / 3.5e6 : 0.0);
      if (us < 0.97 * best.us) best = {f, s, us, s > 1 ? tiles * s * tile_floats : 0};
      if (tiles * (s + 1) > 4 * (int64_t)forms[f].workers) break;
    }
  }
  return best;
}
static int64_t num_k_of(int64_t sum, int runs) { return (sum + BK - 1) / BK * runs; }

template <int KIND> static int gradient(Job& j, int dtype, float* parts, cudaStream_t st) {
  // One weight gradient alone is planned as both are: the same bits whatever is asked for.
  const GradPlan plan = plan_gradient(j.M, j.N, num_k_of(j.sum, KIND == DX ? 2 : 1), KIND == DX ? 1 : 2);
  j.p.parts = parts;
  int rc;
  if (plan.form == 0) rc = launch_form<KIND, 2, 256>(j, dtype, true, st, 0, plan.splits);
  else if (plan.form == 1) rc = launch_form<KIND, 1, 256>(j, dtype, true, st, 0, plan.splits);
  else rc = launch_form<KIND, 1, 128>(j, dtype, true, st, 0, plan.splits);
  if (rc || plan.splits == 1) return rc;
  JoinParams join{};
  join.p = j.p;
  for (int i = 0; i < j.problems; ++i) join.out[i] = const_cast<void*>(j.out[i].ptr);
  join.problems = j.problems;
  join.ctas = plan.form == 0 ? 2 : 1;
  join.tile_cols = plan.form == 2 ? 128 : 256;
  const int64_t items = (int64_t)j.problems * j.p.problem_tiles * join.ctas * 4 * (join.tile_cols / 16);
  const unsigned grid = (unsigned)std::min<int64_t>((items + 7) / 8, (int64_t)sm_count() * 8);
  return launch_kernel("gated linear", dtype == KSB_BF16 ? reinterpret_cast<const void*>(join_kernel<__nv_bfloat16>) : reinterpret_cast<const void*>(join_kernel<__half>), dim3(grid),
                       dim3(256), 0, st, 1, true, join);
}

static int64_t row_stretch(int64_t M, int64_t F) {
  // Rows per CTA: enough CTAs for two waves of four per SM, at least two rows a thread.  Shorter ones keep the bias sums busy: 32760 x 128 of two
  // and eight rows a thread 29 and 20 us; longer ones the GPU idle: 1101 x 4616 12.9 and 15.0.
  const int64_t columns = (F / 8 + ACT_COLS - 1) / ACT_COLS, want = std::max<int64_t>(1, (int64_t)sm_count() * 8 / columns);
  return std::max<int64_t>(2, ((M + want - 1) / want + ACT_ROWS - 1) / ACT_ROWS) * ACT_ROWS;
}

}  // namespace gated
}  // namespace ksb

using namespace ksb;

static int check_gated(int dtype, int64_t M, int64_t F, int64_t K, int act) {
  if (dtype != KSB_BF16 && dtype != KSB_FP16) return fail(KSB_ERR_INVALID, "dtype must be KSB_BF16 or KSB_FP16");
  if (act != KSB_ACT_SILU && act != KSB_ACT_GELU_TANH) return fail(KSB_ERR_INVALID, "unknown activation %d", act);
  if (M < 0 || F <= 0 || K <= 0 || M > (1 << 30) || F > (1 << 30) || K > (1 << 30)) return fail(KSB_ERR_INVALID, "bad shape M=%lld F=%lld K=%lld", (long long)M, (long long)F, (long long)K);
  if (F % 8 != 0 || K % 8 != 0) return fail(KSB_ERR_INVALID, "F and K must be multiples of 8 (F=%lld K=%lld)", (long long)F, (long long)K);
  return 0;
}
static bool rows_ok(const void* p, int64_t ld, int64_t cols, int64_t rows) { return p && aligned16(p) && (rows <= 1 || (ld >= cols && ld % 8 == 0)); }

extern "C" int ksb_gated_linear(const void* x, int64_t ldx, const void* w_gate, int64_t ldg, const void* w_up, int64_t ldu, const void* b_gate, const void* b_up,
                                int dtype, int64_t M, int64_t F, int64_t K, int act, void* h, void* saved, ksb_stream_t stream) {
  if (int rc = check_gated(dtype, M, F, K, act)) return rc;
  if (M == 0) return 0;
  if (!rows_ok(x, ldx, K, M) || !rows_ok(w_gate, ldg, K, F) || !rows_ok(w_up, ldu, K, F) || !h || !aligned16(h) || !aligned16(b_gate) || !aligned16(b_up) ||
      !aligned16(saved))
    return fail(KSB_ERR_INVALID, "null or unaligned pointer, or rows not a multiple of 8 elements apart");
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  // Few rows: 1 x 1536 x 8960 11.3 us, on the wide tensor-core form 18 - 20; 16 rows 14.3 and 17.5; 16 x 5120 x 1536 10.7 and 27.5.
  if (M <= gated::MAX_ROWS && !saved) {
    const gated::RowsCall call{x, w_gate, w_up, b_gate, b_up, h, ldx, ldg, ldu, (int)M, (int)F, (int)K, act};
    const int rc = gated::run_rows(call, dtype, st);
    if (rc != KSB_ERR_UNSUPPORTED) return rc ? rc : 1;  // else: no room for so many columns
  }
  gated::Job j{};
  j.a[0] = {x, M, K, M > 1 ? ldx : K};
  j.b[0] = {w_gate, F, K, ldg};
  j.b[1] = {w_up, F, K, ldu};
  j.out[0] = {h, M, F, F};
  const gated::Saved lay = gated::saved_layout(M, F);
  uint8_t* planes = static_cast<uint8_t*>(saved);
  for (int i = 0; i < 2; ++i) {
    j.out[1 + 2 * i] = {planes + i * lay.u, M, F, F};
    j.out[2 + 2 * i] = {planes + i * lay.u + lay.low, M, F, lay.low_ld};
  }
  j.outs = saved ? 5 : 1;
  j.M = M; j.N = F; j.sum = K; j.problems = 1;
  j.p.b_gate = b_gate; j.p.b_up = b_up; j.p.act = act; j.p.save = saved != nullptr; j.p.h = h;
  if (int rc = gated::project(j, dtype, st)) return rc;
  return 1;
}

extern "C" int64_t ksb_gated_linear_saved(int64_t M, int64_t F) { return M <= 0 || F <= 0 || F % 8 != 0 ? 0 : gated::saved_layout(M, F).bytes; }

// [dg][du][sums of the bias gradients][parts of the products' sums: of dx, then of the weights']
static int64_t gated_bytes(int64_t M, int64_t F) { return (M * F * 2 + 255) / 256 * 256; }
static int64_t bias_bytes(int64_t M, int64_t F) {
  const int64_t stretch = gated::row_stretch(M, F);
  return ((M + stretch - 1) / stretch * 2 * F * 4 + 255) / 256 * 256;
}
extern "C" int64_t ksb_gated_linear_workspace(int64_t M, int64_t F, int64_t K) {
  if (M <= 0 || F <= 0 || F % 8 != 0 || K <= 0 || K % 8 != 0) return 0;
  const int64_t floats = std::max(gated::plan_gradient(M, K, gated::num_k_of(F, 2), 1).floats, gated::plan_gradient(F, K, gated::num_k_of(M, 1), 2).floats);
  return 2 * gated_bytes(M, F) + bias_bytes(M, F) + floats * 4;
}

extern "C" int ksb_gated_linear_backward(const ksb_gated_linear_grads* a, void* workspace, ksb_stream_t stream) {
  if (!a) return fail(KSB_ERR_INVALID, "null pointer");
  const int64_t M = a->M, F = a->F, K = a->K;
  if (int rc = check_gated(a->dtype, M, F, K, a->act)) return rc;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (M == 0) {  // sums over no rows
    for (void* w : {a->dw_gate, a->dw_up})
      if (w && cudaMemsetAsync(w, 0, (size_t)F * K * 2, st) != cudaSuccess) return fail(KSB_ERR_CUDA, "cannot clear the gradients");
    for (void* b : {a->db_gate, a->db_up})
      if (b && cudaMemsetAsync(b, 0, (size_t)F * 2, st) != cudaSuccess) return fail(KSB_ERR_CUDA, "cannot clear the gradients");
    return 0;
  }
  const bool weights = a->dw_gate || a->dw_up;
  if (!rows_ok(a->dh, a->lddh, F, M) || !a->saved || !aligned16(a->saved) || !workspace || !aligned16(workspace) ||
      (weights && !rows_ok(a->x, a->ldx, K, M)) || (a->dx && (!rows_ok(a->w_gate, a->ldg, K, F) || !rows_ok(a->w_up, a->ldu, K, F))))
    return fail(KSB_ERR_INVALID, "null or unaligned pointer, or rows not a multiple of 8 elements apart");
  for (const void* t : {a->dx, a->dw_gate, a->dw_up})
    if (!aligned16(t)) return fail(KSB_ERR_INVALID, "unaligned pointer");
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  void *dg = ws, *du = ws + gated_bytes(M, F);
  float* parts = reinterpret_cast<float*>(ws + 2 * gated_bytes(M, F) + bias_bytes(M, F));
  const bool biases = a->db_gate || a->db_up;
  const int before = launch_count();
  gated::ActParams e{};
  e.dh = a->dh; e.lddh = M > 1 ? a->lddh : F; e.dg = dg; e.du = du;
  const gated::Saved lay = gated::saved_layout(M, F);
  e.saved = static_cast<const uint8_t*>(a->saved); e.low_ld = lay.low_ld; e.low = lay.low; e.u = lay.u;
  e.parts = biases ? reinterpret_cast<float*>(ws + 2 * gated_bytes(M, F)) : nullptr;
  e.M = M; e.F = (int)F; e.act = a->act;
  e.stretch = gated::row_stretch(M, F);
  const int stretches = (int)((M + e.stretch - 1) / e.stretch);
  const bool bf16 = a->dtype == KSB_BF16;
  const dim3 grid((unsigned)((F / 8 + gated::ACT_COLS - 1) / gated::ACT_COLS), (unsigned)stretches);
  if (int rc = launch_kernel("gated linear", bf16 ? reinterpret_cast<const void*>(gated::act_grad_kernel<__nv_bfloat16>) : reinterpret_cast<const void*>(gated::act_grad_kernel<__half>),
                             grid, dim3(gated::ACT_COLS, gated::ACT_ROWS), 0, st, 1, true, e))
    return rc;
  if (biases) {
    const float* parts = e.parts;
    const int cols = (int)F;
    void *dbg = a->db_gate, *dbu = a->db_up;
    if (int rc = launch_kernel("gated linear", bf16 ? reinterpret_cast<const void*>(gated::bias_grad_kernel<__nv_bfloat16>) : reinterpret_cast<const void*>(gated::bias_grad_kernel<__half>),
                               dim3((unsigned)((2 * F + 31) / 32)), dim3(32 * gated::TAKERS), 0, st, 1, true, parts, stretches, cols, dbg, dbu))
      return rc;
  }
  if (a->dx) {
    gated::Job j{};
    j.a[0] = {dg, M, F, F};
    j.a[1] = {du, M, F, F};
    j.b[0] = {a->w_gate, F, K, a->ldg};
    j.b[1] = {a->w_up, F, K, a->ldu};
    j.out[0] = {a->dx, M, K, K};
    j.outs = 1;
    j.M = M; j.N = K; j.sum = F; j.problems = 1;
    if (int rc = gated::gradient<gated::DX>(j, a->dtype, parts, st)) return rc;
  }
  if (weights) {
    gated::Job j{};
    j.problems = 0;
    for (int i = 0; i < 2; ++i) {
      void* to = i ? a->dw_up : a->dw_gate;
      if (!to) continue;
      j.a[j.problems] = {i ? du : dg, M, F, F};
      j.out[j.problems] = {to, F, K, K};
      ++j.problems;
    }
    j.a[1] = j.problems == 2 ? j.a[1] : j.a[0];
    j.outs = j.problems;
    j.b[0] = {a->x, M, K, M > 1 ? a->ldx : K};
    j.M = F; j.N = K; j.sum = M;
    if (int rc = gated::gradient<gated::DW>(j, a->dtype, parts, st)) return rc;
  }
  return launch_count() - before;
}
