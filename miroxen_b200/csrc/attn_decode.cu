// attn_decode_paged: attention of one new token of each sequence over a paged key/value cache, the work split evenly
// over the GPU along the cached tokens and joined.
//
//   s_j = scale * q . k_j,   m = max_j s_j,   out = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m)
//
// Every cached key and value in view is read once: 2 * Hkv * D elements per token against 4 * H * D flops, so memory
// bounds it as long as the heads that share a key head are computed together.  They are the rows of the matrix
// instructions here (mma.sync m16n8k16, up to 16 query heads of one key head; unused rows are zero): the tensor pipe is
// far from busy at this ratio, and the operands come from shared memory tiles that change with every use, which is
// what the warp-level instruction takes without a detour.
//
// Split: a tile is 64 or 128 tokens of one (sequence, key head, block of 16 query heads).  All tiles of the call in order
// (sequence, head, token) are cut into equal runs, one per resident CTA, whatever the lengths are - a CTA's run may
// end inside a sequence's tokens and cover several short sequences.  Each CTA finds the run's start itself by summing the
// lengths.  A run that covers a (sequence, head) alone writes its output; otherwise the CTA leaves its running maximum,
// sum and unnormalised output in its slots of the workspace (one for the segment its run starts in, one for the segment
// it ends in) and join_kernel, launched behind it, adds them up in order.  Results do not depend on timing.
//
// Within a CTA a fifth warp brings the tiles of K and V into a ring of shared-memory stages (16-byte cp.async, rows found
// through the page table one tile ahead, completion counted on mbarriers) and four warps do the arithmetic.  For the scores
// each takes a quarter of the tile's tokens; for the product with V each takes a quarter of the channels of all tokens, so
// that the output stays in a few registers and only the probabilities pass through shared memory.  They are taken relative
// to a maximum that all four share and that moves only when a score lies more than 2^8 above it (every sum is relative to
// it, so the result is the same): one barrier per tile, which also carries that vote.
// Scores, maxima, sums and output are fp32; probabilities are rounded to bf16 (f16 for an e4m3 cache) for the product, as
// the tensor instruction needs the type of V.
#include <cuda_fp16.h>

#include "bulk_copy.cuh"
#include "common.cuh"
#include "kv_cache.cuh"

namespace mxk {
namespace {

constexpr int kRows = 16;       // query heads per work item
constexpr int kWarps = 4;       // that compute; one more copies
constexpr int kConsumers = 32 * kWarps, kThreadsD = kConsumers + 32;
constexpr float kSlack = 8.f;   // log2 of how far a score may lie above the maximum in use
#ifndef MXK_TOKW
#define MXK_TOKW(E, DP) 16
#define MXK_STAGES(E, DP) ((E) || (DP) == 64 ? 4 : 3)
#endif
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct DecodeLaunch {
  MxkDecodeArgs a;
  MxkKvCache c;
  int group;       // query heads per key head
  int blocks;      // blocks of 16 of those
  int heads;       // Hkv * blocks: work items per sequence
  int ctas;        // runs
  float scale2;    // scale * log2(e)
  unsigned page_recip;  // floor((2^32 - 1) / page_size)
  float* part_o;   // [2 ctas][16][DP]
  float* part_ml;  // [2 ctas][16][2]
  int* err;
};

// Tokens in view of a sequence of length n are [0, first) and [skip, n); view_len of them.
struct View {
  int len, first, skip;
};
__device__ __forceinline__ View view_of(const DecodeLaunch& p, int b) {
  int n = p.a.seq_lens[b];
  const int cap = p.c.max_pages * p.c.page_size;
  if (n < 0 || n > cap) {  // never followed past the table
    if (p.err) atomicExch(p.err, kErrBadIndex);
    n = n < 0 ? 0 : cap;
  }
  View v{n, 0, 0};
  if (p.a.left >= 0 && int64_t(n) - 1 > p.a.left) {
    const int lo = int(int64_t(n) - 1 - p.a.left);
    v.first = p.a.sinks < lo ? int(p.a.sinks) : lo;
    v.skip = lo;
    v.len = v.first + n - lo;
  }
  return v;
}

// Tiles of sequence b, all its work items.
template <int TILE>
__device__ __forceinline__ int tiles_of(const DecodeLaunch& p, int b) {
  return (view_of(p, b).len + TILE - 1) / TILE * p.heads;
}

// Finds, with the whole CTA: the number of tiles of the call, and for tile `want` of the caller's choosing (a function of
// the total) the sequence it lies in and the number of tiles in front of that sequence.
template <int TILE, class Want>
__device__ __forceinline__ void locate(const DecodeLaunch& p, int* red, Want want, int& total, int& seq, int& before) {
  constexpr int W = kThreadsD / 32;
  const int n = p.c.n_seqs, t = threadIdx.x, lane = t & 31, warp = t >> 5;
  int mine = 0, first = 0;  // thread t sums a contiguous share of the sequences
  const int share = (n + kThreadsD - 1) / kThreadsD, b0 = min(n, t * share), b1 = min(n, b0 + share);
  for (int b = b0; b < b1; b++) {
    const int k = tiles_of<TILE>(p, b);
    if (b == b0) first = k;
    mine += k;
  }
  int incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += x;
  }
  if (lane == 31) red[warp] = incl;
  if (t == 0) red[W] = -1;
  __syncthreads();
  int base = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < W; w++) {
    if (w < warp) base += red[w];
    total += red[w];
  }
  int at = base + incl - mine;
  const int target = want(total);
  if (target >= at && target < at + mine) {
    int b = b0;
    for (int k = first; target >= at + k; k = tiles_of<TILE>(p, b)) at += k, b++;
    red[W] = b, red[W + 1] = at;
  }
  __syncthreads();
  seq = red[W], before = red[W + 1];
}

// A place in the order of tiles.
struct Cursor {
  int b, head, tile, n_tiles;  // tile of n_tiles of work item `head` (key head * blocks + block) of sequence b
  View v;
};
template <int TILE>
__device__ __forceinline__ void cursor_sequence(const DecodeLaunch& p, Cursor& c) {  // sequences without a token are passed over
  while (c.b < p.c.n_seqs) {
    c.v = view_of(p, c.b);
    c.n_tiles = (c.v.len + TILE - 1) / TILE;
    if (c.n_tiles > 0) return;
    c.b++;
  }
}
template <int TILE>
__device__ __forceinline__ void cursor_next(const DecodeLaunch& p, Cursor& c) {
  if (++c.tile < c.n_tiles) return;
  c.tile = 0;
  if (++c.head < p.heads) return;
  c.head = 0, c.b++;
  cursor_sequence<TILE>(p, c);
}

// 16 bytes, or 16 zeros
__device__ __forceinline__ void cp_async16(unsigned dst, const void* src, unsigned bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
// One arrival on `bar` once this thread's copies so far have landed.
__device__ __forceinline__ void cp_async_arrive(unsigned bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void arrive(unsigned bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }
// Barrier of the computing warps; `vote`: whether any of them has v set.
__device__ __forceinline__ void meet() { asm volatile("bar.sync 1, %0;" ::"n"(kConsumers) : "memory"); }
__device__ __forceinline__ bool vote(bool v) {
  unsigned r;
  asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 q, %1, 0;\n\tbarrier.cta.red.or.pred p, 1, %2, q;\n\tselp.u32 %0, 1, 0, p;\n\t}"
               : "=r"(r)
               : "r"(unsigned(v)), "n"(kConsumers)
               : "memory");
  return r != 0;
}
__device__ __forceinline__ void ldsm4(unsigned addr, unsigned (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void ldsm4_t(unsigned addr, unsigned (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
template <bool F16>
__device__ __forceinline__ void mma16816(float (&d)[4], const unsigned (&a)[4], unsigned b0, unsigned b1) {
  if (F16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// two e4m3 values (exact in f16)
__device__ __forceinline__ unsigned e4m3x2_to_f16x2(unsigned pair) {
  unsigned r;
  asm("{\n\t.reg .b16 t;\n\tcvt.u16.u32 t, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, t;\n\t}" : "=r"(r) : "r"(pair));
  return r;
}
__device__ __forceinline__ unsigned pack_f16(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const unsigned*>(&h);
}

// A stage holds a tile of K and one of V, a row per token, rows 16 bytes longer than their DP elements: the eight rows that
// an ldmatrix phase reads then start four banks apart.  Tokens per tile and stages: about 32 KB a stage where a token's row
// is long, twice the tokens where it is short, so that what a tile costs beside its bytes (a barrier, the vote, the
// exchange of probabilities) is spread over as many.
template <bool E4M3, int DP>
struct DecodeCfg {
  static constexpr int kTokW = MXK_TOKW(E4M3, DP);  // tokens per warp
  static constexpr int kTile = kTokW * kWarps;
  static constexpr int kRowBytes = DP * (E4M3 ? 1 : 2), kPitch = kRowBytes + 16;
  static constexpr int kChunks = kRowBytes / 16;
  static constexpr int kTileBytes = kTile * kPitch;
  static constexpr int kStages = MXK_STAGES(E4M3, DP);
  static constexpr int kSmem = kStages * 2 * kTileBytes;
};

template <bool E4M3, int DP>
__global__ void __launch_bounds__(kThreadsD) decode_kernel(const __grid_constant__ DecodeLaunch p) {
  using Cfg = DecodeCfg<E4M3, DP>;
  using elem = typename KvElem<E4M3>::type;
  constexpr int kSt = Cfg::kStages, kTile = Cfg::kTile, kTokW = Cfg::kTokW, kPitch = Cfg::kPitch;
  constexpr int kKSteps = DP / 16, kNW = DP / kWarps / 8, kNT = kTokW / 8;  // k-steps of the scores; 8-channel tiles, 8-token tiles per warp
  extern __shared__ __align__(128) unsigned char ring[];
  __shared__ __align__(16) unsigned short prob[2][kRows][kTile + 8];
  __shared__ float wmax[kWarps][kRows], wsum[kWarps][kRows];
  __shared__ unsigned there[kSt][kTile / 32];  // which tokens of a tile exist
  __shared__ unsigned long long full[kSt], empty[kSt];
  __shared__ int red[kThreadsD / 32 + 2];
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  const int D = p.c.D;
  const unsigned ring_u = smem_u32(ring);
  pdl_launch_dependents();
  if (tid == 0) {
    // a stage is full when the copies of the copying warp's 32 threads have landed and its word on the tokens is written
    for (int i = 0; i < kSt; i++) mbar_init(smem_u32(&full[i]), 33), mbar_init(smem_u32(&empty[i]), kWarps);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (D < DP) {  // channels [D, DP) of every row stay zero (the copies never touch them)
    for (int i = tid; i < Cfg::kSmem / 16; i += kThreadsD) reinterpret_cast<uint4*>(ring)[i] = make_uint4(0u, 0u, 0u, 0u);
  }
  pdl_wait();

  int total, seq0, before;
  int per = 0;
  locate<kTile>(p, red, [&](int t) { return int(blockIdx.x) * (per = (t + p.ctas - 1) / p.ctas); }, total, seq0, before);
  const int t0 = min(total, int(blockIdx.x) * per), n_my = min(total, t0 + per) - t0;
  // sequences that have no token in view: out 0, lse -inf
  for (int b = blockIdx.x; b < p.c.n_seqs; b += gridDim.x) {
    if (view_of(p, b).len > 0) continue;
    for (int i = tid; i < p.a.H * D; i += kThreadsD) p.a.out[int64_t(b) * p.a.H * D + i] = 0;
    if (p.a.lse)
      for (int i = tid; i < p.a.H; i += kThreadsD) p.a.lse[int64_t(b) * p.a.H + i] = -INFINITY;
  }
  if (n_my <= 0) return;

  Cursor cur;
  cur.b = seq0;
  cursor_sequence<kTile>(p, cur);
  cur.head = (t0 - before) / cur.n_tiles, cur.tile = (t0 - before) % cur.n_tiles;
  bool ok = true;

  if (warp == kWarps) {
    // ---- the copying warp ----
    constexpr int kPerInstr = 32 / Cfg::kChunks, kWords = kTile / 32;  // rows per instruction; tokens a lane looks up
    const int ch = lane % Cfg::kChunks, sub = lane / Cfg::kChunks;
    const bool copies = ch * 16 < D * int(sizeof(elem));
    const unsigned char *kb = static_cast<const unsigned char*>(p.c.k) + ch * 16, *vb = static_cast<const unsigned char*>(p.c.v) + ch * 16;
    // Pages and slots of tokens lane, lane + 32, ... of the tile that is copied next (slot -1: no token), asked for before the
    // tile in front of it is copied and not looked at until then, so that the page table's latency passes meanwhile.
    int page[kWords], slot[kWords];
    int64_t head_off;
    auto look_up = [&]() {
      head_off = int64_t(cur.head / p.blocks) * p.c.head_stride;
#pragma unroll
      for (int u = 0; u < kWords; u++) {
        const int i = cur.tile * kTile + u * 32 + lane;
        page[u] = 0, slot[u] = -1;
        if (i < cur.v.len) {  // inside the table: the length is held to it
          const int tok = i < cur.v.first ? i : i - cur.v.first + cur.v.skip;
          // tok / page_size by the reciprocal rounded down, at most one too small for tok < 2^31
          int n = int(__umulhi(unsigned(tok), p.page_recip)), r = tok - n * p.c.page_size;
          if (r >= p.c.page_size) n++, r -= p.c.page_size;
          slot[u] = r;
          page[u] = p.c.page_table[int64_t(cur.b) * p.c.table_stride + n];
        }
      }
      cursor_next<kTile>(p, cur);
    };
    look_up();
    int st = 0;
    for (int i = 0; i < n_my; i++) {
      int64_t off[kWords];  // byte offsets, -1: not there
#pragma unroll
      for (int u = 0; u < kWords; u++) {
        off[u] = -1;
        if (slot[u] >= 0) {
          if (page[u] >= 0 && page[u] < p.c.num_pages) off[u] = (int64_t(page[u]) * p.c.page_stride + int64_t(slot[u]) * p.c.token_stride + head_off) * int(sizeof(elem));
          else if (p.err) atomicExch(p.err, kErrBadIndex);
        }
      }
      if (i + 1 < n_my) look_up();
      if (i >= kSt) {
        ok = __all_sync(0xffffffffu, mbar_wait_spin(smem_u32(&empty[st]), unsigned(i / kSt - 1) & 1u));
        if (!ok) break;
      }
      const unsigned dk = ring_u + unsigned(st) * 2 * Cfg::kTileBytes + unsigned(sub * kPitch + ch * 16);
#pragma unroll
      for (int u = 0; u < kWords; u++) {
        const unsigned word = __ballot_sync(0xffffffffu, off[u] >= 0);
        if (lane == 0) there[st][u] = word;
#pragma unroll
        for (int r = 0; r < 32 / kPerInstr; r++) {
          const int row = u * 32 + r * kPerInstr;  // + sub
          const int64_t o = __shfl_sync(0xffffffffu, off[u], r * kPerInstr + sub);
          if (copies) {  // a token that is not there reads as zeros: its value must not carry anything into 0 * v
            const unsigned n = o >= 0 ? 16u : 0u;
            const int64_t x = o >= 0 ? o : 0;
            cp_async16(dk + unsigned(row * kPitch), kb + x, n);
            cp_async16(dk + unsigned(Cfg::kTileBytes + row * kPitch), vb + x, n);
          }
        }
      }
      cp_async_arrive(smem_u32(&full[st]));
      if (lane == 0) arrive(smem_u32(&full[st]));
      if (++st == kSt) st = 0;
    }
    // nothing of this CTA's may be under way when its shared memory goes
    asm volatile("cp.async.wait_all;" ::: "memory");
    if (!ok && p.err) atomicExch(p.err, kErrBulkTimeout);
    return;
  }

  // ---- the computing warps ----
  // this warp's state: rows r0 = lane / 4 and r0 + 8; channel tiles of the warp's quarter of the output
  float o[kNW][4];
  float base[2], l[2];  // maximum in use (in units of log2), this thread's part of the sum
  unsigned qf[kKSteps][4];
  float qs[2] = {1.f, 1.f}, ks2 = 0.f;
  const int r0 = lane >> 2, c2 = (lane & 3) * 2;
  bool fresh = true;
  int first_tile = 0, st = 0, g = 0, rows = 0, h0 = 0;
  unsigned ph = 0;

  for (int i = 0; i < n_my; i++) {
    if (fresh) {  // a new (sequence, head): its queries into registers
      fresh = false, first_tile = cur.tile;
      g = cur.head / p.blocks;
      const int blk = cur.head - g * p.blocks;
      rows = min(kRows, p.group - blk * kRows), h0 = g * p.group + blk * kRows;
      ks2 = p.scale2 * (E4M3 && p.c.k_scale ? p.c.k_scale[g] : 1.f);
#pragma unroll
      for (int n = 0; n < kNW; n++) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
      base[0] = base[1] = -INFINITY, l[0] = l[1] = 0.f;
      const mxk_bf16* q = p.a.q + int64_t(cur.b) * p.a.q_stride + int64_t(h0) * D;
#pragma unroll
      for (int half = 0; half < 2; half++) {
        const int r = r0 + 8 * half;
        const bool on = r < rows;
        if (!E4M3) {
#pragma unroll
          for (int s = 0; s < kKSteps; s++)
#pragma unroll
            for (int hi = 0; hi < 2; hi++) {
              const int d = 16 * s + 8 * hi + c2;
              qf[s][half + 2 * hi] = on && d < D ? *reinterpret_cast<const unsigned*>(q + int64_t(r) * D + d) : 0u;
            }
        } else {
          // e4m3 keys are taken as f16, which holds them exactly; so are the queries, scaled by a power of two (per head)
          // that brings their largest into [2^13, 2^14): what f16 then loses lies 2^-38 below it.  The order of channels in
          // a 16-channel step is the one the keys are read in: lane c: channels 4 c + {0, 1 | 2, 3}.
          unsigned raw[kKSteps][2];
          float big = 0.f;
#pragma unroll
          for (int s = 0; s < kKSteps; s++)
#pragma unroll
            for (int hi = 0; hi < 2; hi++) {
              const int d = 16 * s + 2 * c2 + 2 * hi;
              raw[s][hi] = on && d < D ? *reinterpret_cast<const unsigned*>(q + int64_t(r) * D + d) : 0u;
              big = fmaxf(big, fmaxf(fabsf(bf16_lo(raw[s][hi])), fabsf(bf16_hi(raw[s][hi]))));
            }
          big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
          big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
          // exponent of `big` by its bits; zero, subnormal and infinite rows keep a factor that changes nothing that matters
          int e = int((__float_as_uint(big) >> 23) & 255) - 127;
          e = e < -110 ? -110 : e > 127 ? 127 : e;
          const float up = __uint_as_float(unsigned(127 + 13 - e) << 23);
          qs[half] = __uint_as_float(unsigned(127 - 13 + e) << 23);
#pragma unroll
          for (int s = 0; s < kKSteps; s++)
#pragma unroll
            for (int hi = 0; hi < 2; hi++) qf[s][half + 2 * hi] = pack_f16(bf16_lo(raw[s][hi]) * up, bf16_hi(raw[s][hi]) * up);
        }
      }
    }
    // A wait that runs out does not leave the loop: the four warps go on meeting, without waiting for anything else.
    ok = ok && __all_sync(0xffffffffu, mbar_wait_spin(smem_u32(&full[st]), ph));
    const unsigned k_u = ring_u + unsigned(st) * 2 * Cfg::kTileBytes, v_u = k_u + Cfg::kTileBytes;

    // ---- scores of this warp's tokens ----
    float s[kNT][4];
#pragma unroll
    for (int n = 0; n < kNT; n++) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
    if (!E4M3) {
      const unsigned a = k_u + unsigned((warp * kTokW + (lane & 7) + ((lane >> 4) << 3)) * kPitch + ((lane >> 3) & 1) * 16);
#pragma unroll
      for (int ks = 0; ks < kKSteps; ks++)
#pragma unroll
        for (int n = 0; n < kNT; n += 2) {
          unsigned b[4];
          ldsm4(a + unsigned(n * 8 * kPitch + ks * 32), b);
          mma16816<false>(s[n], qf[ks], b[0], b[1]);
          mma16816<false>(s[n + 1], qf[ks], b[2], b[3]);
        }
    } else {
      // four 16-byte chunks of 8 tokens: a register holds four channels of one token, two pairs of one 16-channel step
      const unsigned a = k_u + unsigned((warp * kTokW + (lane & 7)) * kPitch + (lane >> 3) * 16);
#pragma unroll
      for (int grp = 0; grp < DP / 64; grp++)
#pragma unroll
        for (int n = 0; n < kNT; n++) {
          unsigned w[4];
          ldsm4(a + unsigned(n * 8 * kPitch + grp * 64), w);
#pragma unroll
          for (int ks = 0; ks < 4; ks++) mma16816<true>(s[n], qf[4 * grp + ks], e4m3x2_to_f16x2(w[ks] & 0xffffu), e4m3x2_to_f16x2(w[ks] >> 16));
        }
    }
    // the warp's bits of the tile's tokens
    const unsigned word = there[st][warp * kTokW / 32] >> (warp * kTokW % 32);
    const bool all_there = kTokW == 32 ? word == 0xffffffffu : (word & 0xffffu) == 0xffffu;
    const float f0 = E4M3 ? ks2 * qs[0] : ks2, f1 = E4M3 ? ks2 * qs[1] : ks2;
#pragma unroll
    for (int n = 0; n < kNT; n++) s[n][0] *= f0, s[n][1] *= f0, s[n][2] *= f1, s[n][3] *= f1;
    if (!all_there) {
#pragma unroll
      for (int n = 0; n < kNT; n++)
#pragma unroll
        for (int e = 0; e < 4; e++)
          if (!(word >> (8 * n + c2 + (e & 1)) & 1u)) s[n][e] = -INFINITY;
    }
    float mx[2] = {fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])};
#pragma unroll
    for (int n = 1; n < kNT; n++) mx[0] = fmaxf(mx[0], fmaxf(s[n][0], s[n][1])), mx[1] = fmaxf(mx[1], fmaxf(s[n][2], s[n][3]));
    unsigned short(*pr)[kTile + 8] = prob[i & 1];
    float add[2];
    auto probabilities = [&]() {
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const float b = base[h] == -INFINITY ? 0.f : base[h];  // nothing seen yet: exp2(-inf - 0) = 0 everywhere
        add[h] = 0.f;
#pragma unroll
        for (int n = 0; n < kNT; n++) {
          const float p0 = ex2_approx(s[n][2 * h] - b), p1 = ex2_approx(s[n][2 * h + 1] - b);
          add[h] += p0 + p1;
          *reinterpret_cast<unsigned*>(&pr[r0 + 8 * h][warp * kTokW + 8 * n + c2]) = E4M3 ? pack_f16(p0, p1) : pack_bf16(p0, p1);
        }
      }
    };
    probabilities();
    if (vote(mx[0] > base[0] + kSlack || mx[1] > base[1] + kSlack)) {  // always in a segment's first tile
#pragma unroll
      for (int h = 0; h < 2; h++) {
        mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 1));
        mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 2));
        if ((lane & 3) == 0) wmax[warp][r0 + 8 * h] = mx[h];
      }
      meet();
#pragma unroll
      for (int h = 0; h < 2; h++) {
        float mn = base[h];
#pragma unroll
        for (int w = 0; w < kWarps; w++) mn = fmaxf(mn, wmax[w][r0 + 8 * h]);
        if (mn != base[h]) {
          const float f = ex2_approx(base[h] - mn);  // 0 for the first maximum
          l[h] *= f;
#pragma unroll
          for (int n = 0; n < kNW; n++) o[n][2 * h] *= f, o[n][2 * h + 1] *= f;
          base[h] = mn;
        }
      }
      probabilities();
      meet();
    }
    l[0] += add[0], l[1] += add[1];
    // ---- this warp's channels of the product with V ----
    const unsigned pa_u = smem_u32(&pr[(lane & 7) + (((lane >> 3) & 1) << 3)][(lane >> 4) << 3]);
    const unsigned va_u = v_u + unsigned(((lane & 7) + (((lane >> 3) & 1) << 3)) * kPitch) +
                          unsigned((E4M3 ? (kNW / 2 == 2 ? warp * 2 + (lane >> 4) : warp) : warp * kNW + (lane >> 4)) * 16);
#pragma unroll
    for (int ks = 0; ks < kTile / 16; ks++) {
      unsigned pa[4];
      ldsm4(pa_u + unsigned(ks * 32), pa);
      if (!E4M3) {
#pragma unroll
        for (int n = 0; n < kNW; n += 2) {
          unsigned b[4];
          ldsm4_t(va_u + unsigned(ks * 16 * kPitch + n * 16), b);
          mma16816<false>(o[n], pa, b[0], b[1]);
          mma16816<false>(o[n + 1], pa, b[2], b[3]);
        }
      } else {
        // a 16-bit transposed load of 8-bit pairs: register: (token 2c: channels 2n, 2n + 1), (token 2c + 1: the same);
        // the pairs of one channel are then its bytes 0, 2 and 1, 3, so two channel tiles hold the even and the odd ones
        constexpr int kPairs = kNW / 2;  // 16-byte chunks of the warp (16 channels each)
        unsigned b[4];
        ldsm4_t(va_u + unsigned(ks * 16 * kPitch), b);
#pragma unroll
        for (int n = 0; n < kPairs; n++) {
          const unsigned lo = b[2 * n], hi = b[2 * n + 1];  // tokens 0-7 and 8-15 of the step
          mma16816<true>(o[2 * n], pa, e4m3x2_to_f16x2(__byte_perm(lo, 0, 0x4420)), e4m3x2_to_f16x2(__byte_perm(hi, 0, 0x4420)));
          mma16816<true>(o[2 * n + 1], pa, e4m3x2_to_f16x2(__byte_perm(lo, 0, 0x4431)), e4m3x2_to_f16x2(__byte_perm(hi, 0, 0x4431)));
        }
      }
    }
    __syncwarp();
    if (lane == 0) arrive(smem_u32(&empty[st]));
    if (++st == kSt) st = 0, ph ^= 1u;

    const bool last = cur.tile + 1 == cur.n_tiles;
    if (last || i + 1 == n_my) {  // the (sequence, head) or the run ends: store
      const bool whole = last && first_tile == 0;
#pragma unroll
      for (int h = 0; h < 2; h++) {
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
        if ((lane & 3) == 0) wsum[warp][r0 + 8 * h] = l[h];
      }
      meet();
      const float vs = E4M3 && p.c.v_scale ? p.c.v_scale[g] : 1.f;
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const int r = r0 + 8 * h;
        if (r >= rows) continue;
        float sum = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; w++) sum += wsum[w][r];
        const int64_t slot = 2 * int64_t(blockIdx.x) + (first_tile == 0 ? 1 : 0);
        const float f = whole ? (sum > 0.f || sum != sum ? vs / sum : 0.f) : vs;
#pragma unroll
        for (int n = 0; n < kNW; n++) {
          // channels of o[n][2h], o[n][2h + 1]
          const int d0 = E4M3 ? (warp * (kNW / 2) + n / 2) * 16 + 2 * c2 + (n & 1) : (warp * kNW + n) * 8 + c2, d1 = E4M3 ? d0 + 2 : d0 + 1;
          if (whole) {
            mxk_bf16* dst = p.a.out + (int64_t(cur.b) * p.a.H + h0 + r) * D;
            const unsigned w = pack_bf16(o[n][2 * h] * f, o[n][2 * h + 1] * f);
            if (d0 < D) dst[d0] = mxk_bf16(w & 0xffffu);
            if (d1 < D) dst[d1] = mxk_bf16(w >> 16);
          } else {
            float* dst = p.part_o + (slot * kRows + r) * DP;
            dst[d0] = o[n][2 * h] * f, dst[d1] = o[n][2 * h + 1] * f;
          }
        }
        if (warp == 0 && (lane & 3) == 0) {
          if (!whole) {
            p.part_ml[(slot * kRows + r) * 2] = base[h], p.part_ml[(slot * kRows + r) * 2 + 1] = sum;
          } else if (p.a.lse) {
            p.a.lse[int64_t(cur.b) * p.a.H + h0 + r] = sum == 0.f ? -INFINITY : (base[h] + log2f(sum)) * kLn2;
          }
        }
      }
      fresh = true;
    }
    cursor_next<kTile>(p, cur);
  }
  if (!ok && p.err) atomicExch(p.err, kErrBulkTimeout);
}

// Adds up, for each (sequence, head) that several runs share, the parts in the order of the runs: one CTA per work item and
// row, warp w taking parts w, w + 4, ... (all channels of a part per access, several parts in flight), the warps' sums in
// order at the end.
template <int DP, int TILE>
__global__ void __launch_bounds__(kConsumers) join_kernel(const __grid_constant__ DecodeLaunch p) {
  constexpr int kCh = DP / 32;  // channels of a lane
  __shared__ int sums[2][kWarps];
  __shared__ float top[kWarps], part_l[kWarps], part[kWarps][DP];
  pdl_launch_dependents();
  pdl_wait();
  const int b = int(blockIdx.x) / p.heads, head = int(blockIdx.x) - b * p.heads, r = int(blockIdx.y);
  const int g = head / p.blocks, blk = head - g * p.blocks, h = g * p.group + blk * kRows + r;
  if (r >= min(kRows, p.group - blk * kRows)) return;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  // tiles in total and in front of sequence b
  int total = 0, before = 0;
  for (int x = tid; x < p.c.n_seqs; x += kConsumers) {
    const int k = tiles_of<TILE>(p, x);
    total += k;
    if (x < b) before += k;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o), before += __shfl_xor_sync(0xffffffffu, before, o);
  if (lane == 0) sums[0][warp] = total, sums[1][warp] = before;
  __syncthreads();
  total = sums[0][0] + sums[0][1] + sums[0][2] + sums[0][3], before = sums[1][0] + sums[1][1] + sums[1][2] + sums[1][3];
  const int n_tiles = (view_of(p, b).len + TILE - 1) / TILE;
  if (n_tiles == 0) return;
  const int per = (total + p.ctas - 1) / p.ctas;
  const int s0 = before + head * n_tiles, c0 = s0 / per, c1 = (s0 + n_tiles - 1) / per;
  if (c0 == c1) return;  // one run had all of it and has written the output
  // a part's slot: the one of the segment its run starts in, unless the work item starts inside the run (or with it)
  auto slot = [&](int c) { return (2 * int64_t(c) + (c == c0 ? 1 : 0)) * kRows + r; };
  float mx = -INFINITY;
  for (int c = c0 + tid; c <= c1; c += kConsumers) mx = fmaxf(mx, p.part_ml[slot(c) * 2]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  if (lane == 0) top[warp] = mx;
  __syncthreads();
  mx = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
  const float base = mx == -INFINITY ? 0.f : mx;
  float sum = 0.f, o[kCh];
#pragma unroll
  for (int i = 0; i < kCh; i++) o[i] = 0.f;
#pragma unroll 4
  for (int c = c0 + warp; c <= c1; c += kWarps) {
    const int64_t at = slot(c);
    const float2 ml = *reinterpret_cast<const float2*>(p.part_ml + at * 2);
    float v[kCh];
    if (kCh == 4) {
      const float4 x = *reinterpret_cast<const float4*>(p.part_o + at * DP + 4 * lane);
      v[0] = x.x, v[1] = x.y, v[kCh - 2] = x.z, v[kCh - 1] = x.w;
    } else {
      const float2 x = *reinterpret_cast<const float2*>(p.part_o + at * DP + 2 * lane);
      v[0] = x.x, v[1] = x.y;
    }
    const float f = ex2_approx(ml.x - base);
    sum = fmaf(ml.y, f, sum);
#pragma unroll
    for (int i = 0; i < kCh; i++) o[i] = fmaf(v[i], f, o[i]);
  }
#pragma unroll
  for (int i = 0; i < kCh; i++) part[warp][lane * kCh + i] = o[i];
  if (lane == 0) part_l[warp] = sum;
  __syncthreads();
  sum = part_l[0] + part_l[1] + part_l[2] + part_l[3];
  const float f = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
  if (tid < p.c.D)
    p.a.out[(int64_t(b) * p.a.H + h) * p.c.D + tid] = mxk_bf16(pack_bf16((part[0][tid] + part[1][tid] + part[2][tid] + part[3][tid]) * f, 0.f) & 0xffffu);
  if (tid == 0 && p.a.lse) p.a.lse[int64_t(b) * p.a.H + h] = sum == 0.f ? -INFINITY : (mx + log2f(sum)) * kLn2;
}

template <bool E4M3, int DP>
int decode_ctas() {
  auto k = decode_kernel<E4M3, DP>;
  cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, DecodeCfg<E4M3, DP>::kSmem);
  return sm_count() * resident_ctas(k, kThreadsD, DecodeCfg<E4M3, DP>::kSmem);
}

template <bool E4M3, int DP>
int launch_decode(const char* name, DecodeLaunch& p, cudaStream_t s) {
  p.ctas = decode_ctas<E4M3, DP>();
  // no more runs than there can be tiles
  const int64_t most = int64_t(p.c.n_seqs) * p.heads * ceil_div(int64_t(p.c.max_pages) * p.c.page_size, DecodeCfg<E4M3, DP>::kTile);
  if (p.ctas > most) p.ctas = int(most < 1 ? 1 : most);
  p.part_o = static_cast<float*>(p.a.workspace);
  p.part_ml = p.part_o + int64_t(2) * p.ctas * kRows * DP;
  launch_pdl(decode_kernel<E4M3, DP>, dim3(unsigned(p.ctas)), dim3(kThreadsD), DecodeCfg<E4M3, DP>::kSmem, s, p);
  if (int rc = after_launch(name)) return rc;
  launch_pdl(join_kernel<DP, DecodeCfg<E4M3, DP>::kTile>, dim3(unsigned(p.c.n_seqs * p.heads), unsigned(p.group < kRows ? p.group : kRows)), dim3(kConsumers), 0, s, p);
  return after_launch(name);
}

int check_heads(const char* name, const MxkKvCache* c, int H) {
  if (H <= 0 || H % c->Hkv != 0) return fail(MXK_ERR_INVALID_ARG, "%s: H=%d must be a positive multiple of Hkv=%d", name, H, c->Hkv);
  return MXK_OK;
}

}  // namespace
}  // namespace mxk

using namespace mxk;

extern "C" {

int64_t mxk_attn_decode_workspace_bytes(const MxkKvCache* cache, int H) {
  const char* name = "attn_decode_workspace_bytes";
  if (int rc = check_cache(name, cache)) return rc;
  if (int rc = check_heads(name, cache, H)) return rc;
  const bool e = cache->type == MXK_KV_E4M3;
  const int dp = cache->D <= 64 ? 64 : 128;
  const int ctas = dp == 64 ? (e ? decode_ctas<true, 64>() : decode_ctas<false, 64>()) : (e ? decode_ctas<true, 128>() : decode_ctas<false, 128>());
  cudaGetLastError();
  return int64_t(2) * ctas * kRows * (dp + 2) * int64_t(sizeof(float));
}

int mxk_attn_decode_paged(const MxkDecodeArgs* args, const MxkKvCache* cache, mxk_stream_t stream) {
  const char* name = "attn_decode_paged";
  if (!args) return fail(MXK_ERR_INVALID_ARG, "%s: null args", name);
  if (int rc = check_cache(name, cache)) return rc;
  if (cache->n_seqs <= 0) return MXK_OK;
  if (int rc = check_heads(name, cache, args->H)) return rc;
  if (cache->max_pages > 0 && cache->num_pages > 0)
    if (int rc = check_cache_pointers(name, cache)) return rc;
  DecodeLaunch p{};
  p.a = *args, p.c = *cache;
  const MxkDecodeArgs& a = p.a;
  if (!a.q || !a.seq_lens || !a.out || !a.workspace) return fail(MXK_ERR_INVALID_ARG, "%s: null q, seq_lens, out or workspace", name);
  if (a.q_stride % 8 != 0 || a.q_stride < 0) return fail(MXK_ERR_INVALID_ARG, "%s: q_stride must be a multiple of 8", name);
  if (!aligned(a.q, 16) || !aligned(a.out, 16) || !aligned(static_cast<const char*>(a.workspace), 16))
    return fail(MXK_ERR_INVALID_ARG, "%s: q, out and workspace must be 16-byte aligned", name);
  if (a.sinks < 0) return fail(MXK_ERR_INVALID_ARG, "%s: sinks=%lld", name, (long long)a.sinks);
  if (!(a.scale > 0.f) || a.scale > 3.0e38f) return fail(MXK_ERR_INVALID_ARG, "%s: scale must be positive and finite", name);
  p.group = a.H / cache->Hkv;
  p.blocks = int(ceil_div(p.group, kRows));
  p.heads = cache->Hkv * p.blocks;
  const int64_t tiles = int64_t(cache->n_seqs) * p.heads * (ceil_div(int64_t(cache->max_pages) * cache->page_size, 64) + 1);
  if (tiles >= (int64_t(1) << 30)) return fail(MXK_ERR_TOO_LARGE, "%s: n_seqs * heads * tokens too large (%lld tiles)", name, (long long)tiles);
  p.scale2 = a.scale * kLog2e;
  p.page_recip = 0xffffffffu / unsigned(cache->page_size);
  p.err = device_error_word();
  const cudaStream_t s = as_stream(stream);
  if (cache->D <= 64) return cache->type == MXK_KV_E4M3 ? launch_decode<true, 64>(name, p, s) : launch_decode<false, 64>(name, p, s);
  return cache->type == MXK_KV_E4M3 ? launch_decode<true, 128>(name, p, s) : launch_decode<false, 128>(name, p, s);
}

}  // extern "C"
