// attn_window: attention of a packed batch of sequences with a sliding window and first tokens that stay visible.
//
//   s_ij = scale * q_i . k_j over the keys j that row i sees,  m_i = max_j s_ij,
//   out_i = sum_j exp(s_ij - m_i) v_j / sum_j exp(s_ij - m_i),   lse_i = m_i + ln sum_j exp(s_ij - m_i)
//
// Row i of a sequence of Lq rows and Lk keys stands at p = i + Lk - Lq and sees j <= p + right (right >= 0) that are
// j >= p - left (left >= 0) or j < sinks.
//
// Two matrix products of 4 D flops per pair with one exponential between: the tensor cores bound it, the exponentials
// (16 per clock and SM) nearly as much.  One CTA of 384 threads holds 256 rows of one head as two halves of 128:
//   warps 0-3, 4-7: the softmax of one half each, a thread per row.  A score tile (128 rows x 128 keys, fp32) comes from
//                   tensor memory into registers, its row maximum, exponentials and their sum are taken there, and the
//                   probabilities go back as bf16 (the type of V, which the product needs);
//   warps 8, 10:    issue tcgen05.mma: S = Q K^T from shared memory (8), O += P V with P from tensor memory (10);
//   warp 9:         TMA: Q once, then the tiles of K and V through a ring of shared-memory stages (128-byte swizzle);
//   warp 11:        finds the tiles: the CTA's own, then those of CTAs that have not started (cluster launch control).
// A tile's loads, first products and its search run while the tile before it is finished.
// Tensor memory: one score tile (128 columns), which the halves use in turn, the probabilities P of each half (64) and the
// output O of each half (128), 512 in all.  A score tile is free as soon as its half has it in registers, so the tensor pipe
// makes the next one, and the products with V, while the softmax runs: S0 | S1 | S0' P0 V | S1' P1 V | ...  Nothing goes
// round in a chain but the softmax of a half, which has a whole turn of the tensor pipe for itself.  (With the
// probabilities written over their scores, two score tiles fit, but then a half's next scores have to wait for its product
// with V: measured 3900 clocks per turn of four products of 128 x 128 x 128, 2820 this way, and 2050 is the pipe's own rate.)
// The running maximum that the exponentials use moves only when it would grow by more than 2^8 (results are the same:
// every sum is relative to it), so O is rescaled rarely, by the half's own warps, once its products so far have retired.
// Blocks of 128 keys outside of every row's view are not visited; only blocks at the edge of some row's view pay for the
// mask.  There, what a row does not see still takes part in the product as 0 * v, which is not 0 where v is not finite: an
// output that is not finite has its rows' edge blocks looked through, and if it can have come from there the row is taken
// again by a plain loop (row_attention) that never touches what the row does not see.
//
// Measured (D = 128): 2 x 4352 rows x 24 heads, everything visible, 361 us = 1290 TFLOP/s from a cold start, 420 us = 1108
// TFLOP/s in a run of seconds, where the power limit holds the clock near 1530 MHz (a library product: 1651 and 1393);
// 33272 rows x 5 heads with a window of 6240 each way and 1560 first keys 800 us; nine packed causal prompts of 14 to 3414 rows,
// 32 heads on 8, window 1024: 114 us; one prompt of 77 rows: 6.8 us.  Heads of 72 or 80 take products of 128: 336 us for the first case.  What bounds it: the tensor pipe, busy 69 % of the time
// (the scores' operands both come from shared memory, 98 clocks instead of 64 per product), and the last round of tiles.
#include <cuda.h>

#include <atomic>

#include "bulk_copy.cuh"
#include "common.cuh"
#include "kv_cache.cuh"
#include "tuning.h"

namespace mxk {
namespace {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct AttnLaunch {
  MxkAttnArgs a;
  int left, right, sinks;  // a's, no bound as kFar
  int group;               // query heads per key head
  float scale2;            // scale * log2(e)
  int* err;
};
constexpr int kFar = 1 << 30;  // rows and keys are fewer, so that positions and bounds add up in 32 bits

// Keys that a row at position p of a sequence of nk keys sees: [0, first) and [lo, hi).
struct Seen {
  int first, lo, hi;
};
__device__ __forceinline__ Seen seen_by(const AttnLaunch& L, int p, int nk) {
  Seen s;
  s.hi = max(0, min(nk, p + L.right + 1));
  s.lo = max(0, min(s.hi, p - L.left));
  s.first = min(L.sinks, s.lo);
  return s;
}

// One row and head by one warp, 32 keys at a time: a lane takes a key's product with q, then the warp adds the keys'
// values, each lane holding channels 2 lane, 2 lane + 1, + 64.  `qs`: the warp's 128 floats of shared memory.
__device__ __forceinline__ void row_attention(const AttnLaunch& L, int64_t row, int h, int64_t k0, int p, int nk, float* qs) {
  const MxkAttnArgs& a = L.a;
  const int lane = threadIdx.x & 31, D = a.D, g = h / L.group;
  const Seen seen = seen_by(L, p, nk);
  const mxk_bf16* q = a.q + row * a.q_stride + int64_t(h) * D;
  __syncwarp();
  for (int d = lane; d < D; d += 32) qs[d] = __uint_as_float(unsigned(q[d]) << 16);
  __syncwarp();
  const mxk_bf16* kb = a.k + k0 * a.k_stride + int64_t(g) * D;
  const mxk_bf16* vb = a.v + k0 * a.v_stride + int64_t(g) * D;
  float m = -INFINITY, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
  const int n = seen.first + seen.hi - seen.lo;
  for (int i0 = 0; i0 < n; i0 += 32) {
    const int i = i0 + lane;
    const int j = i < seen.first ? i : i - seen.first + seen.lo;
    float s = -INFINITY;
    if (i < n) {
      s = 0.f;
      const uint4* kr = reinterpret_cast<const uint4*>(kb + int64_t(j) * a.k_stride);
      for (int c = 0; c < D / 8; c++) {
        float f[8];
        unpack8(kr[c], f);
#pragma unroll
        for (int e = 0; e < 8; e++) s = fmaf(f[e], qs[8 * c + e], s);
      }
      s *= L.scale2;
    }
    float mx = s;
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
    const float mn = fmaxf(m, mx), base = mn == -INFINITY ? 0.f : mn, f = ex2_approx(m - base);
    m = mn;
    const float w = ex2_approx(s - base);
    l = l * f + warp_sum(w);
#pragma unroll
    for (int e = 0; e < 4; e++) o[e] *= f;
    const int cnt = min(32, n - i0);
    for (int t = 0; t < cnt; t++) {
      const float pt = __shfl_sync(0xffffffffu, w, t);
      const int jt = __shfl_sync(0xffffffffu, j, t);
      const mxk_bf16* vr = vb + int64_t(jt) * a.v_stride;
#pragma unroll
      for (int half = 0; half < 2; half++) {
        const int d = 2 * lane + 64 * half;
        if (d < D) {
          const unsigned x = *reinterpret_cast<const unsigned*>(vr + d);
          o[2 * half] = fmaf(pt, bf16_lo(x), o[2 * half]);
          o[2 * half + 1] = fmaf(pt, bf16_hi(x), o[2 * half + 1]);
        }
      }
    }
  }
  const float f = l > 0.f || l != l ? 1.f / l : 0.f;
  mxk_bf16* dst = a.out + row * a.out_stride + int64_t(h) * D;
#pragma unroll
  for (int half = 0; half < 2; half++) {
    const int d = 2 * lane + 64 * half;
    if (d < D) *reinterpret_cast<unsigned*>(dst + d) = n > 0 ? pack_bf16(o[2 * half] * f, o[2 * half + 1] * f) : 0u;
  }
  if (lane == 0 && a.lse) a.lse[row * a.H + h] = l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2;
}

// ---- tensor-core kernel ----------------------------------------------------------------------------------------

constexpr int kM = 128, kN = 128;              // rows of a half, keys of a block
constexpr int kScoreWarp = 8, kTmaWarp = 9, kValueWarp = 10, kScheduleWarp = 11, kThreadsW = 384;
constexpr int kReaders = kThreadsW / 32 - 1;    // warps that are told the tiles
constexpr int kSub = 128 * 128;                // bytes of a 128-row x 64-channel tile
// Registers a thread: 384 x 168 at launch; a softmax thread holds 128 scores, the others need fewer.
constexpr int kRegsSoft = 216, kRegsOther = 72;
static_assert(256 * kRegsSoft + 128 * kRegsOther <= kThreadsW * 168, "the groups' registers are those of the launch");
constexpr int kAskAhead = 6;                   // loads of a tile that are still to come when the next tile is asked for
constexpr unsigned kTmemS = 0, kTmemP = 128, kTmemO = 256, kTmemCols = 512;  // S, 2 x 64 of P, 2 x 128 of O
constexpr float kSlack = 8.f;                  // log2 of how far a score may lie above the maximum in use

template <int DP>
struct WindowCfg {
  static constexpr int kSubs = DP / 64;               // 64-channel tiles of a row
  static constexpr int kTileBytes = kSubs * kSub;     // Q half, K block, V block
  static constexpr int kStages = DP == 128 ? 4 : 8;
};

__device__ __forceinline__ void tma_load_3d(unsigned dst, const CUtensorMap* map, int c0, int c1, int c2, unsigned bar) {
  asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst),
               "l"(map), "r"(bar), "r"(c0), "r"(c1), "r"(c2)
               : "memory");
}
__device__ __forceinline__ void mbar_arrive1(unsigned bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// The matrix instructions are issued by one lane of a converged warp: the whole warp computes the operands (which then are
// uniform registers, as the instruction wants them) and the instruction itself is predicated.  Issued from a branch of one
// lane, every operand is moved between register files first, and the issue takes longer than the product.
__device__ __forceinline__ unsigned elect_lane() {
  unsigned r;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
  return r;
}
__device__ __forceinline__ void commit_to(unsigned bar, unsigned leader) {
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar),
      "r"(leader)
      : "memory");
}
// D (+)= A B, A and B from shared memory
__device__ __forceinline__ void mma_ss(unsigned d, uint64_t a, uint64_t b, unsigned idesc, unsigned acc, unsigned leader) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(acc), "r"(leader)
      : "memory");
}
// D (+)= A B, A from tensor memory
__device__ __forceinline__ void mma_ts(unsigned d, unsigned a, uint64_t b, unsigned idesc, unsigned acc, unsigned leader) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(acc), "r"(leader)
      : "memory");
}
// Shared-memory matrix descriptors under the 128-byte swizzle (1024-byte aligned tiles of 128-byte rows): start address,
// leading and stride offsets in 16-byte units, version 1, layout type 2.
//   Q, K: K-major (a row's channels are adjacent): eight rows every 1024 bytes (stride offset).
//   V: MN-major (the keys are the contraction, the channels adjacent): eight keys every 1024 bytes (stride offset), the next
//      64 channels one 16 KB tile further (leading offset).
__device__ __forceinline__ uint64_t desc_sw128(unsigned addr, unsigned leading) {
  return uint64_t((addr & 0x3ffffu) >> 4) | (uint64_t(leading >> 4) << 16) | (uint64_t(1024 >> 4) << 32) | (uint64_t(1) << 46) | (uint64_t(2) << 61);
}
// kind::f16, fp32 accumulator, bf16 operands; b_mn: B is MN-major
template <int M, int N, bool B_MN>
constexpr unsigned kInstr = (1u << 4) | (1u << 7) | (1u << 10) | (unsigned(B_MN) << 16) | (unsigned(N >> 3) << 17) | (unsigned(M >> 4) << 24);
#define MXK_R4(a, i) "=r"(a[i]), "=r"(a[i + 1]), "=r"(a[i + 2]), "=r"(a[i + 3])
#define MXK_R32(a, i) \
  MXK_R4(a, i), MXK_R4(a, i + 4), MXK_R4(a, i + 8), MXK_R4(a, i + 12), MXK_R4(a, i + 16), MXK_R4(a, i + 20), MXK_R4(a, i + 24), MXK_R4(a, i + 28)
// 32 columns of this thread's lane; tmem_wait_ld() before the first use
__device__ __forceinline__ void tmem_ld32(unsigned addr, unsigned (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, "
      "%20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : MXK_R32(r, 0)
      : "r"(addr)
      : "memory");
}
// The loads have landed; the empty statements tie the registers to this point.
__device__ __forceinline__ void tmem_wait_ld(unsigned (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < 32; i++) asm volatile("" : "+r"(r[i]));
}
__device__ __forceinline__ void tmem_touch(unsigned (&r)[32]) {
#pragma unroll
  for (int i = 0; i < 32; i++) asm volatile("" : "+r"(r[i]));
}
__device__ __forceinline__ void tmem_ld16(unsigned addr, unsigned (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : MXK_R4(r, 0), MXK_R4(r, 4), MXK_R4(r, 8), MXK_R4(r, 12)
      : "r"(addr)
      : "memory");
}
__device__ __forceinline__ void tmem_st16(unsigned addr, const unsigned (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(addr), "r"(r[0]),
      "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]),
      "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
// This warp's stores to tensor memory so far are for the tensor pipe to read.
__device__ __forceinline__ void hand_over(unsigned long long* bar, int lane) {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
  fence_before();
  __syncwarp();
  if (lane == 0) mbar_arrive1(smem_u32(bar));
}

__device__ __forceinline__ float max_nan(float a, float b, float c) {  // NaN if one of them is
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// Pairs of fp32 operations in one instruction.
__device__ __forceinline__ uint64_t pair(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void split(uint64_t v, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// Probabilities of 32 scores: p = 2^(s * scale2 - base), their sum into l (four partial sums), rounded to bf16 in pairs.
// Pairs of fp32 operations where there are any: single ones take 367 instead of 363 us on 2 x 4352 rows x 24 heads and 129
// instead of 121 us on the packed prompts.  (Some of the 2^x as polynomials beside the special-function unit, which is busy
// two thirds of the time, made the kernel slower in proportion to their number, in every form tried: its warps and, in long
// runs, its power have less to spare than that unit.)
__device__ __forceinline__ void exp_chunk(const unsigned (&s)[32], uint64_t scale2, uint64_t neg_base, uint64_t (&l)[2], unsigned (&p)[16]) {
#pragma unroll
  for (int i = 0; i < 16; i++) {
    float x, y;
    split(fma2(pair(__uint_as_float(s[2 * i]), __uint_as_float(s[2 * i + 1])), scale2, neg_base), x, y);
    x = ex2_approx(x), y = ex2_approx(y);
    l[i & 1] = add2(l[i & 1], pair(x, y));
    p[i] = pack_bf16(x, y);
  }
}

struct WindowLaunch {
  AttnLaunch L;
  int halves;     // 128-row halves of a tile: 2, or 1 where that leaves SMs idle
  int max_tiles;  // the grid has max_tiles * H CTAs
  int reversed;   // 1: the numbers of tiles fall with those of the CTAs
  unsigned tries;  // of a wait
};

// What a tile is: rows [r0, r0 + rows) and head `head` of a sequence that starts at row q0 / key k0 and has nq rows, nk keys.
// rows = 0: there is no further one.
struct WindowTile {
  int q0, nq, k0, nk, r0, rows, head;
};

// Where a warp's search for tiles has got to: `seqs` sequences from the back with `tiles` tiles.
struct TileSearch {
  int seqs = 0, tiles = 0;
};

// Tile number `cta` of the launch, by one warp; rows = 0 if there is no such tile.  Counted from the back: the tiles at the end
// of a causal sequence, which have the most keys, come first, all heads of a tile one behind the other (the other way round,
// head by head, the CTAs at work crowd on the same few lines of the keys: packed prompts 195 against 145 us).  A search goes on
// where the CTA's last one ended; where the hardware hands out a number from in front of that (nothing promises an order), it
// starts again.
__device__ __forceinline__ WindowTile find_tile(const WindowLaunch& W, int cta, TileSearch& from) {
  const MxkAttnArgs& a = W.L.a;
  const int lane = threadIdx.x & 31, tile_rows = kM * W.halves, place = cta / a.H;
  WindowTile t{0, int(a.q_rows), 0, int(a.k_rows), 0, 0, cta - place * a.H};
  if (!a.cu_q) {
    t.r0 = (W.max_tiles - 1 - place) * tile_rows;
    t.rows = min(tile_rows, t.nq - t.r0);
    return t;
  }
  if (place < from.tiles) from = TileSearch{};
  constexpr int kAhead = 4;  // groups of 32 sequences whose ends are asked for at once
  for (; from.seqs < a.n_seqs; from.seqs += 32 * kAhead) {
    int x[kAhead][4];
#pragma unroll
    for (int u = 0; u < kAhead; u++) {
      const int b = a.n_seqs - 1 - (from.seqs + 32 * u + lane);
      x[u][0] = x[u][1] = x[u][2] = x[u][3] = 0;
      if (b >= 0) x[u][0] = a.cu_q[b], x[u][1] = a.cu_q[b + 1], x[u][2] = a.cu_k[b], x[u][3] = a.cu_k[b + 1];
    }
    int at = from.tiles;
#pragma unroll
    for (int u = 0; u < kAhead; u++) {
      if (from.seqs + 32 * u >= a.n_seqs) break;
      // held inside the arrays and in order whatever they hold
      const int q0 = max(0, min(x[u][0], int(a.q_rows))), q1 = max(q0, min(x[u][1], int(a.q_rows)));
      const int k0 = max(0, min(x[u][2], int(a.k_rows))), k1 = max(k0, min(x[u][3], int(a.k_rows)));
      if ((q0 != x[u][0] || q1 != x[u][1] || k0 != x[u][2] || k1 != x[u][3]) && W.L.err) atomicExch(W.L.err, kErrBadIndex);
      const int mine = (q1 - q0 + tile_rows - 1) / tile_rows;
      int incl = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += y;
      }
      const int first = at + incl - mine;
      const unsigned hit = __ballot_sync(0xffffffffu, place >= first && place < first + mine);
      if (hit) {
        const int src = __ffs(hit) - 1;
        t.q0 = __shfl_sync(0xffffffffu, q0, src), t.nq = __shfl_sync(0xffffffffu, q1 - q0, src);
        t.k0 = __shfl_sync(0xffffffffu, k0, src), t.nk = __shfl_sync(0xffffffffu, k1 - k0, src);
        t.r0 = __shfl_sync(0xffffffffu, mine - 1 - (place - first), src) * tile_rows;
        t.rows = min(tile_rows, t.nq - t.r0);
        return t;
      }
      at += __shfl_sync(0xffffffffu, incl, 31);
    }
    from.tiles = at;
  }
  return t;
}

template <int DP>
struct __align__(1024) WindowSmem {
  unsigned char q[2][WindowCfg<DP>::kTileBytes];
  unsigned char kv[WindowCfg<DP>::kStages][WindowCfg<DP>::kTileBytes];
  unsigned char stage[2][kSub];  // the halves' output on its way to memory, 64 channels at a time
  unsigned long long q_full[2], q_empty[2], full[WindowCfg<DP>::kStages], empty[WindowCfg<DP>::kStages], s_full[2], s_free, p_full[2], pv_done[2], o_empty[2],
      tile_full[2], tile_empty[2], wanted, asked;
  uint4 answer[1];
  WindowTile tile[2];
  unsigned tmem_base;
};

// The blocks of 128 keys that a tile's rows see.
struct TileView {
  int halves, shift;     // a row's position is its number + shift
  Seen first[2], end[2];  // of the first and the last row of each half: the nearest end, the farthest window start
  int wb0, n_sink, n_blocks;
  __device__ __forceinline__ TileView(const AttnLaunch& L, const WindowTile& t) {
    halves = t.rows > kM ? 2 : 1;
    shift = t.nk - t.nq;
#pragma unroll
    for (int h = 0; h < 2; h++) {
      first[h] = seen_by(L, t.r0 + h * kM + shift, t.nk);
      end[h] = seen_by(L, t.r0 + min((h + 1) * kM, t.rows) - 1 + shift, t.nk);
    }
    const Seen s = first[0], e = halves == 2 ? end[1] : end[0];
    wb0 = s.lo / kN;  // the tile's blocks: n_sink from the front, the others from wb0 on
    n_sink = min((e.first + kN - 1) / kN, wb0);
    n_blocks = n_sink + (e.hi > s.lo ? (e.hi + kN - 1) / kN - wb0 : 0);
  }
  __device__ __forceinline__ int block(int j) const { return j < n_sink ? j : wb0 + j - n_sink; }
  // whether some row of half h sees keys of the block; the last such block, -1 if there is none
  __device__ __forceinline__ int last(int h) const { return h >= halves ? -1 : end[h].hi > first[h].lo ? (end[h].hi - 1) / kN : (end[h].first + kN - 1) / kN - 1; }
  __device__ __forceinline__ bool has(int h, int b) const { return b <= last(h) && (b * kN < end[h].first || b >= first[h].lo / kN); }
};

// Whether a block of keys that some row of half h of the tile sees only a part of holds a value that is not finite, in any of
// its 128 rows (those behind the sequence too: they have been loaded with it).  By one warp, and rarely.
__device__ __forceinline__ bool hidden_value_odd(const AttnLaunch& L, const WindowTile& t, int h) {
  const MxkAttnArgs& a = L.a;
  const TileView v(L, t);
  const Seen f = h == 0 ? v.first[0] : v.first[1], e = h == 0 ? v.end[0] : v.end[1];
  const int lane = threadIdx.x & 31, chunks = a.D / 8;
  const mxk_bf16* vb = a.v + int64_t(t.head / L.group) * a.D;
  bool odd = false;
  for (int j = 0; j < v.n_blocks; j++) {
    const int block = v.block(j), key0 = block * kN;
    if (!(h == 0 ? v.has(0, block) : v.has(1, block)) || (key0 + kN <= f.hi && (key0 >= e.lo || key0 + kN <= f.first))) continue;
    const int rows = int(min(int64_t(kN), a.k_rows - t.k0 - key0));
    for (int i = lane; i < rows * chunks; i += 32) {
      const int r = i / chunks;
      const uint4 x = *reinterpret_cast<const uint4*>(vb + (int64_t(t.k0) + key0 + r) * a.v_stride + (i - r * chunks) * 8);
      constexpr unsigned m = 0x7f807f80u, one = 0x00800080u;  // an exponent of all ones carries into the sign bit
      odd |= ((((x.x & m) + one) | ((x.y & m) + one) | ((x.z & m) + one) | ((x.w & m) + one)) & 0x80008000u) != 0;
    }
  }
  return __any_sync(0xffffffffu, odd);
}

// Asks the hardware for a CTA of this launch that has not started; its number, or -1 when there is none left.  The answer lands
// in shared memory (16 bytes) and completes `bar`.
__device__ __forceinline__ void ask_for_tile(unsigned answer, unsigned bar) {
  mbar_expect_tx(bar, 16);
  asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(answer), "r"(bar) : "memory");
}
__device__ __forceinline__ int tile_answer(unsigned answer) {
  int x = -1;
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b128 r;\n\tld.shared.b128 r, [%1];\n\tclusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, r;\n\t"
      "@p clusterlaunchcontrol.query_cancel.get_first_ctaid.v4.b32.b128 {%0, _, _, _}, r;\n\t}"
      : "+r"(x)
      : "r"(answer)
      : "memory");
  return x;
}

template <int DP>
__global__ void __launch_bounds__(kThreadsW, 1)
    window_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                  const __grid_constant__ WindowLaunch W) {
  using Cfg = WindowCfg<DP>;
  constexpr int kSt = Cfg::kStages;
  // There is no room to align the tiles by hand; without static shared memory the dynamic part starts on a 1 KB boundary.
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  WindowSmem<DP>& sm = *reinterpret_cast<WindowSmem<DP>*>(smem_raw);
  const AttnLaunch& L = W.L;
  const MxkAttnArgs& a = L.a;
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  if (smem_u32(smem_raw) & 1023u) {  // never seen; nothing is computed on tiles that the swizzle would not fit
    if (tid == 0 && L.err) atomicExch(L.err, kErrBulkTimeout);
    return;
  }

  if (tid == 0) {
    for (int i = 0; i < 2; i++) {
      mbar_init(smem_u32(&sm.q_full[i]), 1), mbar_init(smem_u32(&sm.q_empty[i]), 1), mbar_init(smem_u32(&sm.s_full[i]), 1);
      mbar_init(smem_u32(&sm.pv_done[i]), 1), mbar_init(smem_u32(&sm.p_full[i]), 4), mbar_init(smem_u32(&sm.o_empty[i]), 4);
      mbar_init(smem_u32(&sm.tile_full[i]), 1), mbar_init(smem_u32(&sm.tile_empty[i]), kReaders);
    }
    mbar_init(smem_u32(&sm.s_free), 4), mbar_init(smem_u32(&sm.asked), 1), mbar_init(smem_u32(&sm.wanted), 1);
    for (int i = 0; i < kSt; i++) mbar_init(smem_u32(&sm.full[i]), 1), mbar_init(smem_u32(&sm.empty[i]), 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == kScoreWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sm.tmem_base)), "r"(kTmemCols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (warp == kTmaWarp && lane < 3) {
    const CUtensorMap* map = lane == 0 ? &map_q : lane == 1 ? &map_k : &map_v;
    asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
  }
  pdl_launch_dependents();
  fence_before();
  __syncthreads();
  fence_after();
  const unsigned tmem = __shfl_sync(0xffffffffu, sm.tmem_base, 0);
  pdl_wait();  // nothing above touches global memory

  // Every wait is bounded; a role whose wait runs out leaves its loop, the others' waits then run out too.
  bool ok = true;
  auto lane_wait = [&](unsigned long long* bar, int phase) { return mbar_wait_spin(smem_u32(bar), unsigned(phase) & 1u, W.tries); };
  auto wait = [&](unsigned long long* bar, int phase) {
    const bool r = __all_sync(0xffffffffu, lane_wait(bar, phase));
    fence_after();
    return r;
  };
  // The n-th tile of this CTA, from the ring of two that the scheduling warp fills; false: there is none (or the wait ran out).
  auto next_tile = [&](int n, WindowTile& t) {
    ok = wait(&sm.tile_full[n & 1], n >> 1);
    if (!ok) return false;
    t = sm.tile[n & 1];
    __syncwarp();
    if (lane == 0) mbar_arrive1(smem_u32(&sm.tile_empty[n & 1]));
    return t.rows > 0;
  };
  int issued = 0, q_issued[2] = {0, 0};  // TMA: stage and Q fills so far

  if (warp >= kScoreWarp) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsOther));
    const unsigned leader = elect_lane();
    WindowTile t;
    if (warp == kScheduleWarp) {
      // ---- which tiles: this CTA's own, then those of CTAs that have not started yet.  One is asked for when the loads of
      // the tile at hand come to their end, no earlier: what a CTA has asked for no other can take at the end of the launch.
      int cta = int(blockIdx.x), n = 0;
      TileSearch search;
      for (int asks = 0; ok; asks++) {
        t = find_tile(W, W.reversed ? int(gridDim.x) - 1 - cta : cta, search);
        if (t.rows > 0) {
          if (n >= 2) ok = wait(&sm.tile_empty[n & 1], (n >> 1) - 1);
          if (ok && leader) {
            sm.tile[n & 1] = t;
            mbar_arrive1(smem_u32(&sm.tile_full[n & 1]));
          }
          __syncwarp();
          if (ok) ok = wait(&sm.wanted, n);
          n++;
        }
        if (!ok) break;
        if (leader) ask_for_tile(smem_u32(sm.answer), smem_u32(&sm.asked));
        ok = wait(&sm.asked, asks);
        cta = ok ? tile_answer(smem_u32(sm.answer)) : -1;
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // read before it is written over
        __syncwarp();
        if (cta < 0) break;
      }
      if (ok && n >= 2) ok = wait(&sm.tile_empty[n & 1], (n >> 1) - 1);
      if (ok && leader) {
        sm.tile[n & 1].rows = 0;
        mbar_arrive1(smem_u32(&sm.tile_full[n & 1]));
      }
    } else if (warp == kTmaWarp) {
      for (int n = 0; next_tile(n, t); n++) {
        const TileView v(L, t);
        const int kv_head = t.head / L.group;
        auto load_q = [&](int h) {
          if (v.last(h) < 0) return;
          if (q_issued[h] > 0 && ok) ok = wait(&sm.q_empty[h], q_issued[h] - 1);
          if (!ok) return;
          const unsigned bar = smem_u32(&sm.q_full[h]);
          if (leader) {
            mbar_expect_tx(bar, Cfg::kTileBytes);
            for (int c = 0; c < Cfg::kSubs; c++) tma_load_3d(smem_u32(sm.q[h]) + c * kSub, &map_q, c * 64, t.head, t.q0 + t.r0 + h * kM, bar);
          }
          q_issued[h]++;
        };
        // in the order in which they are needed: Q of the first half, K, Q of the second half, V, ...
        const int n_fills = 2 * v.n_blocks, want_at = max(0, n_fills - kAskAhead);
        if (n_fills == 0 && leader) mbar_arrive1(smem_u32(&sm.wanted));
        for (int i = 0; i < n_fills && ok; i++) {  // 2 j: K of block j; 2 j + 1: its V
          if (i == want_at && leader) mbar_arrive1(smem_u32(&sm.wanted));
          if (i < 2) load_q(i);
          const int st = issued % kSt;
          if (ok && issued >= kSt) ok = wait(&sm.empty[st], issued / kSt - 1);
          if (!ok) break;
          const unsigned bar = smem_u32(&sm.full[st]);
          const int key = t.k0 + v.block(i >> 1) * kN;
          if (leader) {
            mbar_expect_tx(bar, Cfg::kTileBytes);
            const CUtensorMap* map = (i & 1) ? &map_v : &map_k;
            for (int c = 0; c < Cfg::kSubs; c++) tma_load_3d(smem_u32(sm.kv[st]) + c * kSub, map, c * 64, kv_head, key, bar);
          }
          issued++;
        }
        if (!ok) break;
      }
    } else if (warp == kScoreWarp) {
      int fill0 = 0, made = 0, q_used[2] = {0, 0};  // fills in front of this tile, score tiles, Q tiles so far
      for (int n = 0; next_tile(n, t); n++) {
        const TileView v(L, t);
        bool fresh[2] = {true, true};
        for (int j = 0; j < v.n_blocks && ok; j++) {
          const int block = v.block(j), fill = fill0 + 2 * j;
          ok = wait(&sm.full[fill % kSt], fill / kSt);
          const unsigned ka = smem_u32(sm.kv[fill % kSt]);
#pragma unroll
          for (int h = 0; h < 2; h++) {
            if (!ok || !v.has(h, block)) continue;
            if (fresh[h]) ok = wait(&sm.q_full[h], q_used[h]), fresh[h] = false;
            if (ok && made > 0) ok = wait(&sm.s_free, made - 1);  // the tile before this one is in its half's registers
            if (!ok) continue;
            const unsigned qa = smem_u32(sm.q[h]);
#pragma unroll
            for (int c = 0; c < Cfg::kSubs; c++)
#pragma unroll
              for (int k = 0; k < 4; k++)
                mma_ss(tmem + kTmemS, desc_sw128(qa + c * kSub, 16) + uint64_t(2 * k), desc_sw128(ka + c * kSub, 16) + uint64_t(2 * k),
                       kInstr<kM, kN, false>, (c | k) != 0 ? 1u : 0u, leader);
            commit_to(smem_u32(&sm.s_full[h]), leader);
            made++;
            if (block == v.last(h)) commit_to(smem_u32(&sm.q_empty[h]), leader), q_used[h]++;
          }
          if (ok) commit_to(smem_u32(&sm.empty[fill % kSt]), leader);
        }
        if (!ok) break;
        fill0 += 2 * v.n_blocks;
      }
    } else if (warp == kValueWarp) {
      int fill0 = 0, done[2] = {0, 0}, used[2] = {0, 0};  // fills in front of this tile; blocks and outputs a half has had
      for (int n = 0; next_tile(n, t); n++) {
        const TileView v(L, t);
        bool fresh[2] = {true, true};
        for (int j = 0; j < v.n_blocks && ok; j++) {
          const int block = v.block(j), fill = fill0 + 2 * j + 1;
          ok = wait(&sm.full[fill % kSt], fill / kSt);
          const unsigned va = smem_u32(sm.kv[fill % kSt]);
#pragma unroll
          for (int h = 0; h < 2; h++) {
            if (!ok || !v.has(h, block)) continue;
            if (fresh[h] && used[h] > 0) ok = wait(&sm.o_empty[h], used[h] - 1);  // the output of the tile before is in registers
            if (ok) ok = wait(&sm.p_full[h], done[h]);
            if (!ok) continue;
#pragma unroll
            for (int k = 0; k < kN / 16; k++)  // 16 keys: 8 columns of P, 2048 bytes of V
              mma_ts(tmem + kTmemO + unsigned(h) * 128, tmem + kTmemP + unsigned(h) * 64 + unsigned(k) * 8, desc_sw128(va, kSub) + uint64_t(k * 128),
                     kInstr<kM, DP, true>, k > 0 || !fresh[h] ? 1u : 0u, leader);
            commit_to(smem_u32(&sm.pv_done[h]), leader);
            done[h]++, fresh[h] = false;
          }
          if (ok) commit_to(smem_u32(&sm.empty[fill % kSt]), leader);
        }
        if (!ok) break;
        fill0 += 2 * v.n_blocks;
#pragma unroll
        for (int h = 0; h < 2; h++)
          if (!fresh[h]) used[h]++;
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSoft));
    // ---- softmax of half h: thread (warp & 3) * 32 + lane owns that row ----
    const int h = warp >> 2, row_h = (warp & 3) * 32 + lane;
    const unsigned lanes = unsigned((warp & 3) * 32) << 16;
    const unsigned ts = tmem + lanes + kTmemS, tp = tmem + lanes + kTmemP + unsigned(h) * 64, to = tmem + lanes + kTmemO + unsigned(h) * 128;
    unsigned char* stage = sm.stage[h] + (warp & 3) * (32 * 128);  // 32 rows of 64 channels on their way out
    int all = 0;  // blocks that the half has had
    for (int n = 0;; n++) {
      // The tile stays this warp's until its output is done; what the loop over the blocks does not need is read again behind it
      // (a row of scores leaves few registers).
      ok = wait(&sm.tile_full[n & 1], n >> 1);
      if (!ok) break;
      const WindowTile& tile = sm.tile[n & 1];
      if (tile.rows <= 0) break;
      int blocks, wb0, n_sink, last, from, sinks, full_from, full_sinks, full_to;
      {
        const WindowTile t = tile;
        const TileView v(L, t);
        const Seen f = h == 0 ? v.first[0] : v.first[1], e = h == 0 ? v.end[0] : v.end[1];
        blocks = v.n_blocks, wb0 = v.wb0, n_sink = v.n_sink;
        last = h == 0 ? v.last(0) : v.last(1);                         // blocks that some row of the half sees: as TileView::has
        from = f.lo / kN, sinks = (e.first + kN - 1) / kN;
        full_from = (e.lo + kN - 1) / kN, full_sinks = f.first / kN, full_to = f.hi / kN;  // blocks that all its rows see all of
      }
      float m = -INFINITY, l = 0.f;  // maximum in use (of the raw scores), sum
      int done = 0;                  // blocks of this tile that some row of the half sees, so far
      for (int j = 0; j < blocks; j++) {
        const int block = j < n_sink ? j : wb0 + j - n_sink;
        if (!(block <= last && (block < sinks || block >= from))) continue;
        const bool edge = !(block < full_to && (block >= full_from || block < full_sinks));
        // A wait that runs out: the warp goes on without waiting for anything else.  Its lanes agree on the outcome.
        ok = ok && __all_sync(0xffffffffu, lane_wait(&sm.s_full[h], all));
        fence_after();
        unsigned s[4][32];
#pragma unroll
        for (int c = 0; c < 4; c++) tmem_ld32(ts + 32 * c, s[c]);
        tmem_wait_ld(s[0]);
        tmem_touch(s[1]), tmem_touch(s[2]), tmem_touch(s[3]);
        fence_before();
        __syncwarp();
        if (ok && lane == 0) mbar_arrive1(smem_u32(&sm.s_free));  // the other half's scores may come
        if (edge) {
          // bit i of below(n): i < n
          auto below = [](int n) { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u; };
          const Seen mine = seen_by(L, min(tile.r0 + h * kM + row_h, tile.nq - 1) + tile.nk - tile.nq, tile.nk);
#pragma unroll
          for (int c = 0; c < 4; c++) {
            const int k0 = block * kN + 32 * c;
            const unsigned see = below(mine.first - k0) | (below(mine.hi - k0) & ~below(mine.lo - k0));
#pragma unroll
            for (int i = 0; i < 32; i++) s[c][i] = (see >> i) & 1u ? s[c][i] : 0xff800000u;
          }
        }
        float mx;
        {
          float part[4];
#pragma unroll
          for (int c = 0; c < 4; c++) {
            part[c] = max_nan(__uint_as_float(s[c][0]), __uint_as_float(s[c][1]), __uint_as_float(s[c][2]));
#pragma unroll
            for (int i = 3; i < 31; i += 2) part[c] = max_nan(part[c], __uint_as_float(s[c][i]), __uint_as_float(s[c][i + 1]));
          }
          mx = max_nan(max_nan(part[0], __uint_as_float(s[0][31]), part[1]), __uint_as_float(s[1][31]), max_nan(part[2], __uint_as_float(s[2][31]), part[3]));
          mx = max_nan(mx, __uint_as_float(s[3][31]), mx);
        }
        if (!(mx < INFINITY)) l = __uint_as_float(0x7fc00000u);  // a NaN or an infinity among the scores: the whole row is NaN
        const bool grow = (mx - m) * L.scale2 > kSlack;          // also the first finite score (m = -inf); false for NaN
        if (__any_sync(0xffffffffu, grow)) {
          float f = 1.f;
          if (grow) {
            f = ex2_approx((m - mx) * L.scale2);
            m = mx, l *= f;
          }
          if (done > 0 && ok) {
            ok = __all_sync(0xffffffffu, lane_wait(&sm.pv_done[h], all - 1));
            fence_after();
#pragma unroll 1
            for (int c = 0; c < DP / 16; c++) {
              unsigned o[16];
              tmem_ld16(to + 16 * c, o);
#pragma unroll
              for (int i = 0; i < 16; i++) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
              tmem_st16(to + 16 * c, o);
            }
          }
        }
        const float base = m == -INFINITY ? 0.f : m * L.scale2;
        const uint64_t scale2 = pair(L.scale2, L.scale2), neg_base = pair(-base, -base);
        uint64_t l2[2] = {0, 0};
#pragma unroll
        for (int c = 0; c < 4; c++) {
          unsigned p[16];
          exp_chunk(s[c], scale2, neg_base, l2, p);
          if (c == 0 && done > 0 && ok) {  // P is the product's until it has retired
            ok = __all_sync(0xffffffffu, lane_wait(&sm.pv_done[h], all - 1));
            fence_after();
          }
          tmem_st16(tp + 16 * c, p);
        }
        if (ok) hand_over(&sm.p_full[h], lane);
        float l0, l1;
        split(add2(l2[0], l2[1]), l0, l1);
        l += l0 + l1;
        done++, all++;
      }
      // ---- output ----
      if (ok && done > 0) ok = lane_wait(&sm.pv_done[h], all - 1);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      fence_after();
      const WindowTile t = tile;
      const int rh0 = t.r0 + h * kM + (warp & 3) * 32, rows_w = min(32, t.rows - (rh0 - t.r0));  // of this warp, none if negative
      const int64_t row0 = int64_t(t.q0) + rh0;
      const bool some = l > 0.f || l != l;
      const float f = some ? 1.f / l : 0.f;
      const uint64_t f2 = pair(f, f);
      uint64_t odd2 = 0;  // becomes NaN with an output that is not finite
      mxk_bf16* dst = a.out + (row0 + (lane >> 3)) * a.out_stride + int64_t(t.head) * a.D + 8 * (lane & 7);
      unsigned o[DP / 32][32];
      if (done == 0) {
#pragma unroll
        for (int c = 0; c < DP / 32; c++)
#pragma unroll
          for (int i = 0; i < 32; i++) o[c][i] = 0u;
      } else {
#pragma unroll
        for (int c = 0; c < DP / 32; c++) tmem_ld32(to + 32 * c, o[c]);
        tmem_wait_ld(o[0]);
#pragma unroll
        for (int c = 1; c < DP / 32; c++) tmem_touch(o[c]);
        fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive1(smem_u32(&sm.o_empty[h]));  // the next tile's output may come
      }
#pragma unroll
      for (int c = 0; c < DP / 64; c++) {
        // A row per lane from tensor memory, 128 bytes of four rows per store to memory: through shared memory, the 16-byte
        // chunks of a row exchanged by the row's number.
#pragma unroll
        for (int i = 0; i < 8; i++) {
          unsigned w[4];
#pragma unroll
          for (int e = 0; e < 4; e++) {
            const int k = 8 * (i & 3) + 2 * e;
            const unsigned(&r)[32] = o[2 * c + (i >> 2)];
            const uint64_t x = fma2(pair(__uint_as_float(r[k]), __uint_as_float(r[k + 1])), f2, 0);  // 0 * 0 in a row that sees nothing
            odd2 = fma2(x, 0, odd2);
            float lo, hi;
            split(x, lo, hi);
            w[e] = pack_bf16(lo, hi);
          }
          *reinterpret_cast<uint4*>(stage + lane * 128 + ((i ^ (lane & 7)) * 16)) = make_uint4(w[0], w[1], w[2], w[3]);
        }
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 8; i++) {
          const int r = 4 * i + (lane >> 3);
          const uint4 x = *reinterpret_cast<const uint4*>(stage + r * 128 + (((lane & 7) ^ (r & 7)) * 16));
          if (r < rows_w && 64 * c + 8 * (lane & 7) < a.D) *reinterpret_cast<uint4*>(dst + 4 * i * a.out_stride + 64 * c) = x;
        }
        __syncwarp();
      }
      if (a.lse && lane < rows_w)
        a.lse[(row0 + lane) * a.H + t.head] = some ? (m == -INFINITY ? 0.f : m * L.scale2 * kLn2) + log2f(l) * kLn2 : -INFINITY;
      // An output that is not finite although the row's scores are: a value that the row sees, or one of a block that it does
      // not see all of, which has come in as 0 * v.  Where there is such a value, the row is taken again without it.
      float odd, odd_hi;
      split(odd2, odd, odd_hi);
      odd += odd_hi;
      unsigned again = __ballot_sync(0xffffffffu, odd != odd && l == l && lane < rows_w);
      if (again && hidden_value_odd(L, t, h)) {
        for (; again; again &= again - 1) {
          const int r = __ffs(again) - 1;
          row_attention(L, row0 + r, t.head, t.k0, rh0 + r + t.nk - t.nq, t.nk, reinterpret_cast<float*>(stage));
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive1(smem_u32(&sm.tile_empty[n & 1]));
    }
  }

  if (!ok && L.err) atomicExch(L.err, kErrBulkTimeout);
  fence_before();
  // Every role's waits are bounded, so all threads arrive here.  After a failure the copies under way get a bounded chance
  // to land before the shared memory goes.
  if (__syncthreads_or(!ok) != 0) {
    if (warp == kTmaWarp) {
      for (int h = 0; h < 2; h++)
        if (q_issued[h] > 0) mbar_wait(smem_u32(&sm.q_full[h]), unsigned(q_issued[h] - 1) & 1u);
      for (int i = issued > kSt ? issued - kSt : 0; i < issued; i++) mbar_wait(smem_u32(&sm.full[i % kSt]), unsigned(i / kSt) & 1u);
    }
    __syncthreads();
  }
  if (warp == kScoreWarp) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
  }
}

// cuTensorMapEncodeTiled through the runtime's driver entry point (no link against libcuda).
using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                              const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeFn encode_fn() {
  static std::atomic<EncodeFn> cached{nullptr};
  EncodeFn f = cached.load(std::memory_order_acquire);
  if (f) return f;
  void* p = nullptr;
  cudaDriverEntryPointQueryResult q;
  if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess || !p) {
    cudaGetLastError();
    return nullptr;
  }
  f = reinterpret_cast<EncodeFn>(p);
  cached.store(f, std::memory_order_release);
  return f;
}

// bf16 [rows, heads, D]: boxes of 64 channels of one head of 128 rows, 128-byte swizzle; what lies outside reads as 0.
int make_map(const char* name, CUtensorMap* map, const void* base, int64_t rows, int heads, int D, int64_t stride) {
  EncodeFn enc = encode_fn();
  if (!enc) return fail(MXK_ERR_CUDA, "%s: cuTensorMapEncodeTiled is not available from this driver", name);
  if (rows == 1) stride = int64_t(heads) * D;  // never used
  const cuuint64_t dims[3] = {cuuint64_t(D), cuuint64_t(heads), cuuint64_t(rows)};
  const cuuint64_t strides[2] = {cuuint64_t(D) * 2, cuuint64_t(stride) * 2};
  const cuuint32_t box[3] = {64, 1, 128};
  const cuuint32_t elem[3] = {1, 1, 1};
  const CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(MXK_ERR_CUDA, "%s: cuTensorMapEncodeTiled failed with code %d", name, int(r));
  return MXK_OK;
}

template <int DP>
int launch_window(const char* name, WindowLaunch& W, cudaStream_t s) {
  const MxkAttnArgs& a = W.L.a;
  CUtensorMap mq, mk, mv;
  if (int rc = make_map(name, &mq, a.q, a.q_rows, a.H, a.D, a.q_stride)) return rc;
  // without a key nothing is loaded; the maps then only have to be valid
  if (int rc = make_map(name, &mk, a.k_rows > 0 ? a.k : a.q, a.k_rows > 0 ? a.k_rows : 1, a.k_rows > 0 ? a.Hkv : 1, a.D, a.k_stride)) return rc;
  if (int rc = make_map(name, &mv, a.k_rows > 0 ? a.v : a.q, a.k_rows > 0 ? a.k_rows : 1, a.k_rows > 0 ? a.Hkv : 1, a.D, a.v_stride)) return rc;
  auto k = window_kernel<DP>;
  const size_t smem = sizeof(WindowSmem<DP>);
  const cudaError_t e = allow_smem(k, smem);
  if (e != cudaSuccess) return fail(MXK_ERR_CUDA, "%s: cudaFuncSetAttribute: %s", name, cudaGetErrorString(e));
  const int64_t ctas = int64_t(W.max_tiles) * a.H;
  if (ctas >= (int64_t(1) << 31)) return fail(MXK_ERR_TOO_LARGE, "%s: %lld tiles", name, (long long)ctas);
  launch_pdl(k, dim3(unsigned(ctas)), dim3(kThreadsW), smem, s, mq, mk, mv, W);
  return after_launch(name);
}

}  // namespace
}  // namespace mxk

using namespace mxk;

extern "C" int mxk_attn_window(const MxkAttnArgs* args, mxk_stream_t stream) {
  const char* name = "attn_window";
  if (!args) return fail(MXK_ERR_INVALID_ARG, "%s: null args", name);
  AttnLaunch L{};
  L.a = *args;
  const MxkAttnArgs& a = L.a;
  if (a.q_rows <= 0 || a.n_seqs <= 0) return MXK_OK;
  if (!a.q || !a.out) return fail(MXK_ERR_INVALID_ARG, "%s: null q or out", name);
  if (a.k_rows < 0 || (a.k_rows > 0 && (!a.k || !a.v))) return fail(MXK_ERR_INVALID_ARG, "%s: k_rows=%lld, null k or v", name, (long long)a.k_rows);
  if (a.H <= 0 || a.Hkv <= 0 || a.H % a.Hkv != 0)
    return fail(MXK_ERR_INVALID_ARG, "%s: H=%d must be a positive multiple of Hkv=%d", name, a.H, a.Hkv);
  if (a.D < 8 || a.D > MXK_ATTN_MAX_HEAD_DIM || a.D % 8 != 0)
    return fail(MXK_ERR_INVALID_ARG, "%s: head dimension %d must be a multiple of 8 and at most %d", name, a.D, MXK_ATTN_MAX_HEAD_DIM);
  if ((a.cu_q == nullptr) != (a.cu_k == nullptr) || (!a.cu_q && a.n_seqs != 1))
    return fail(MXK_ERR_INVALID_ARG, "%s: cu_q and cu_k come together, and several sequences need them (n_seqs=%d)", name, a.n_seqs);
  if (a.q_rows >= kFar || a.k_rows >= kFar)
    return fail(MXK_ERR_TOO_LARGE, "%s: q_rows=%lld k_rows=%lld", name, (long long)a.q_rows, (long long)a.k_rows);
  if (a.q_stride % 8 != 0 || a.k_stride % 8 != 0 || a.v_stride % 8 != 0 || a.out_stride % 8 != 0)
    return fail(MXK_ERR_INVALID_ARG, "%s: strides must be multiples of 8", name);
  if ((a.q_rows > 1 && (a.q_stride < int64_t(a.H) * a.D || a.out_stride < int64_t(a.H) * a.D)) ||
      (a.k_rows > 1 && (a.k_stride < int64_t(a.Hkv) * a.D || a.v_stride < int64_t(a.Hkv) * a.D)))
    return fail(MXK_ERR_INVALID_ARG, "%s: row strides smaller than a row's heads", name);
  if (!aligned(a.q, 16) || !aligned(a.k, 16) || !aligned(a.v, 16) || !aligned(a.out, 16))
    return fail(MXK_ERR_INVALID_ARG, "%s: q, k, v and out must be 16-byte aligned", name);
  if (a.sinks < 0) return fail(MXK_ERR_INVALID_ARG, "%s: sinks=%lld", name, (long long)a.sinks);
  if (!(a.scale > 0.f) || a.scale > 1e30f) return fail(MXK_ERR_INVALID_ARG, "%s: scale must be positive and at most 1e30", name);
  L.group = a.H / a.Hkv;
  L.scale2 = a.scale * kLog2e;
  L.err = device_error_word();
  L.left = a.left < 0 || a.left > kFar ? kFar : int(a.left);
  L.right = a.right < 0 || a.right > kFar ? kFar : int(a.right);
  L.sinks = a.sinks > kFar ? kFar : int(a.sinks);
  WindowLaunch W{L, 2, 0, tune(TUNE_WINDOW_ORDER, 1) == 2, 0u};
  // What a warp may have to wait for grows with the keys: up to 32 rows taken again by one warp, each 32 keys at a time, are as many
  // steps as there are keys, 4.6 us each measured, 15.6 us with all warps of the GPU at it (30000 keys of 128 channels: 139 and
  // 469 ms a tile); and with the sequences that a search passes, 128 at a time.  128 tries are twelve times such a step.
  const int64_t tries = tune(TUNE_WINDOW_WAIT_TRIES, int(kSpinTries)) + 128 * a.k_rows + a.n_seqs;
  W.tries = unsigned(tries < 0xffffffffll ? tries : 0xffffffffll);
  // at most one tile per sequence is not full
  auto tiles = [&](int rows) { return a.n_seqs == 1 ? ceil_div(a.q_rows, rows) : a.q_rows / rows + (a.n_seqs < a.q_rows ? a.n_seqs : a.q_rows); };
  if (tiles(2 * kM) * a.H <= sm_count() / 2) W.halves = 1;  // twice the CTAs still fit the GPU at once
  const int64_t most = tiles(W.halves * kM);
  if (most >= (int64_t(1) << 31)) return fail(MXK_ERR_TOO_LARGE, "%s: %lld tiles", name, (long long)most);
  W.max_tiles = int(most);
  return a.D <= 64 ? launch_window<64>(name, W, as_stream(stream)) : launch_window<128>(name, W, as_stream(stream));
}
