// attn_decode_paged: attention of one new token of each sequence over a paged key/value cache, the work split evenly
// over the GPU along the cached tokens and joined.
//
//   s_j = scale * q . k_j,   m = max_j s_j,   out = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m)
//
// Every cached key and value in view is read once: 2 * Hkv * D elements per token against 4 * H * D flops, so memory
// bounds it as long as the heads that share a key head are computed together.  They are the columns of the matrix
// instructions here (mma.sync m16n8k16, 8 or 16 query heads of one key head; unused columns are zero): S^T = K Q^T, O^T =
// V^T P^T.  The tensor pipe is far from busy at this ratio, and the operands come from shared memory tiles that change with
// every use, which is what the warp-level instruction takes without a detour.
//
// Split: a tile is 64 or 128 tokens of one (sequence, key head, block of query heads).  All tiles of the call in order
// (sequence, head, token) are cut into equal runs, one per resident CTA, whatever the lengths are - a CTA's run may
// end inside a sequence's tokens and cover several short sequences.  Each CTA finds the run's start itself by summing the
// lengths.  A run that covers a (sequence, head) alone writes its output; otherwise the CTA leaves its running maximum,
// sum and unnormalised output in its slots of the workspace (one for the segment its run starts in, one for the segment
// it ends in) and join_kernel, launched behind it, adds them up in order.  Where the whole call is short, that second launch is
// most of it: if up to 8 CTAs for each (sequence, head), as many as the GPU holds, leave at most kShort tiles for each, they are a
// cluster and add up through each other's shared memory (1 sequence of 500 tokens, 8 key heads of 128: 5.5 against 8.0 us;
// 32 of 300: 8.6 against 12.8).  And where there are more (sequence, head)s than CTAs by half, each of kMedium tiles at
// most, a CTA takes one as a whole: the heads of the same tokens, which lie side by side in a page, are then read at the
// same time (200 sequences of 2000 tokens: 252 against 278 us).  Results do not depend on timing.
//
// Within a CTA two warps bring the tiles of K and V into a ring of shared-memory stages (16-byte cp.async, rows found
// through the page table one tile ahead, completion counted on mbarriers) and four warps do the arithmetic.  For the scores
// each takes a quarter of the tile's tokens; for the product with V each takes a quarter of the channels of all tokens, so
// that the output stays in a few registers and only the probabilities pass through shared memory.  They are taken relative
// to a maximum that all four share and that moves only when a score lies more than 2^8 above it (every sum is relative to
// it, so the result is the same): one barrier per tile, which also carries that vote.
// Scores, maxima, sums and output are fp32; probabilities are rounded to bf16 (f16 for an e4m3 cache) for the product, as
// the tensor instruction needs the type of V.
//
// Measured in replays on the same inputs (floor at 6560 GB/s in brackets): 64 sequences of 4100 to 16384 bf16 tokens, 32 heads on 8
// of 128, pages of 16: 407 us (382; 420 in a run with changing inputs); 8 sequences with 32833 e4m3 tokens in view, 40 heads on 8:
// 95 us (82; 108); 48 of 2250 to 9000 e4m3 tokens, 28 heads on 4 of 64: 38 us (22; 40) - rows of 64 bytes take as many instructions per
// token as longer ones: issue slots 50 % used, ALU 43 %; with the heads outermost in a page the same.
// Blocks of 16 heads, 64 sequences of 4100 to 16384 tokens, 2 key heads of 128 (bf16: 106, e4m3: 53): 8 heads on each 120 and 84 us, 12
// heads 122 and 78, 16 heads 124 and 80, 32 heads, two blocks, which read the cache one after the other, 214 and 146.
#include <cuda_fp16.h>

#include <type_traits>

#include "bulk_copy.cuh"
#include "common.cuh"
#include "kv_cache.cuh"
#include "tuning.h"

namespace mxk {
namespace {

constexpr int kWarps = 4;       // that compute
constexpr int kCopyWarps = 2;   // that copy, 32 tokens of a tile each
constexpr int kConsumers = 32 * kWarps, kThreadsD = kConsumers + 32 * kCopyWarps;
constexpr int kShort = 8, kMedium = 32;  // tiles of a CTA up to which a call takes the forms without a second launch
constexpr int kSingle = 4;               // tiles of a work item up to which it is one CTA's
constexpr float kSlack = 8.f;   // log2 of how far a score may lie above the maximum in use
// Probabilities in f16 (of an e4m3 cache) are taken relative to a maximum 2^7 lower than the scores': they reach 2^15 then, which
// f16 holds, and what it rounds them to at the small end is 2^-32 of the largest instead of 2^-25 (a million tokens that are
// each that small are 3 % of the sum).
constexpr float kLift = 7.f;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct DecodeLaunch {
  MxkDecodeArgs a;
  MxkKvCache c;
  int group;       // query heads per key head
  int blocks;      // blocks of 8 or 16 of those
  int heads;       // Hkv * blocks: work items per sequence
  int ctas;        // runs
  int cluster;     // 0: runs over all tiles; n > 0: the tiles of a work item cut among n CTAs (a cluster where n > 1)
  float scale2;    // scale * log2(e)
  unsigned tries;       // of a wait for a tile
  unsigned page_recip;  // floor((2^32 - 1) / page_size)
  float* part_o;   // [2 ctas][rows][DP], rows: query heads per block
  float* part_ml;  // [2 ctas][rows][2]
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

// Tiles of `len` tokens; 31 bits hold the tokens, but not their number rounded up.
template <int TILE>
__device__ __forceinline__ int tiles_in(int len) {
  return int((unsigned(len) + TILE - 1) / TILE);
}
// Tiles of sequence b, all its work items.
template <int TILE>
__device__ __forceinline__ int tiles_of(const DecodeLaunch& p, int b) {
  return tiles_in<TILE>(view_of(p, b).len) * p.heads;
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

// A place in a CTA's tiles: tile of [lo, hi), the CTA's part of the n_tiles of work item `head` (key head * blocks + block) of
// sequence b, with `left` of that part and `rest` of the CTA's tiles behind that part to come.
struct Cursor {
  int b, head, tile, n_tiles, lo, hi, left, rest;
  View v;
};
template <int TILE>
__device__ __forceinline__ void cursor_sequence(const DecodeLaunch& p, Cursor& c) {  // sequences without a token are passed over
  while (c.b < p.c.n_seqs) {
    c.v = view_of(p, c.b);
    c.n_tiles = tiles_in<TILE>(c.v.len);
    if (c.n_tiles > 0) return;
    c.b++;
  }
}
// The part that starts at tile lo, of a CTA with n tiles from there on.
__device__ __forceinline__ void cursor_part(Cursor& c, int lo, int n) {
  c.tile = c.lo = lo, c.hi = min(c.n_tiles, lo + n);
  c.left = c.hi - lo, c.rest = n - c.left;
}
template <int TILE>
__device__ __forceinline__ void cursor_next(const DecodeLaunch& p, Cursor& c) {
  if (--c.left > 0) {
    if (++c.tile == c.hi) c.tile = c.lo;
    return;
  }
  if (c.rest <= 0) return;
  if (++c.head == p.heads) {
    c.head = 0, c.b++;
    cursor_sequence<TILE>(p, c);
  }
  cursor_part(c, 0, c.rest);
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
// The cluster's threads that are still there; what they wrote to shared memory is visible to the others.
__device__ __forceinline__ void cluster_meet() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// What stands at this shared-memory address in CTA `rank` of the cluster.
__device__ __forceinline__ float ld_cluster(unsigned addr, unsigned rank) {
  float v;
  asm volatile("{\n\t.reg .u32 a;\n\tmapa.shared::cluster.u32 a, %1, %2;\n\tld.shared::cluster.f32 %0, [a];\n\t}" : "=f"(v) : "r"(addr), "r"(rank) : "memory");
  return v;
}
__device__ __forceinline__ void ld_cluster2(unsigned addr, unsigned rank, float& x, float& y) {
  asm volatile("{\n\t.reg .u32 a;\n\tmapa.shared::cluster.u32 a, %2, %3;\n\tld.shared::cluster.v2.f32 {%0, %1}, [a];\n\t}"
               : "=f"(x), "=f"(y)
               : "r"(addr), "r"(rank)
               : "memory");
}
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
// Four e4m3 values as f16, which holds them exactly: bytes 0, 1 and bytes 2, 3.
__device__ __forceinline__ void e4m3x4_to_f16(unsigned x, unsigned& lo, unsigned& hi) {
  asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}" : "=r"(lo), "=r"(hi) : "r"(x));
}
__device__ __forceinline__ unsigned pack_f16(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const unsigned*>(&h);
}

// A stage holds a tile of K and one of V, a row per token, rows 16 bytes longer than their DP elements: the eight rows that
// an ldmatrix phase reads then start four banks apart.  A tile has 16 tokens for each computing warp; 32 (LONG) where rows are
// short, D <= 64, and the call is cut into runs.  Stages: as many as leave
//   two CTAs per SM to bf16 rows of D > 64 (64 long sequences: 421 us with three stages, 455 with two and three CTAs, 804 with four
//   and one) and to LONG tiles (48 sequences of up to 9000 tokens, 4 heads of 64: e4m3 38 us against 42 with tiles of 64 and four
//   CTAs, 46 with one CTA; bf16 56 against 75 with three CTAs and 58 with tiles of 64 and two) - fewer rows of the memory are then
//   open at a time;
//   as many CTAs as there are registers for to the other e4m3 rows (8 sequences with 32832 tokens in view, D = 128: 95 us with two
//   stages, 102.5 with three or four, 112 with LONG tiles), which take more arithmetic per byte, and to short calls, where a CTA has
//   few tiles (300 sequences of 600 tokens, 4 heads of 64: e4m3 22 us against 28, bf16 30 against 34 with LONG tiles).
// Chosen with blocks of 8 heads.  Blocks of 16 take the same for want of a case where it counts for more: D = 128, 32 heads on 2, 64
// sequences of up to 16384 tokens, bf16 124 us with three stages, 123 with two or four; e4m3 80 with two, 77.5 with three or four.
template <bool E4M3, int DP, bool LONG>
struct DecodeCfg {
  static_assert(!LONG || DP == 64, "LONG tiles belong to short rows");
  static constexpr int kTokW = LONG ? 32 : 16;  // tokens per warp
  static constexpr int kTile = kTokW * kWarps;
  static constexpr int kPerLane = kTile / (32 * kCopyWarps);  // tokens that a lane of a copying warp looks up
  static constexpr int kRowBytes = DP * (E4M3 ? 1 : 2), kPitch = kRowBytes + 16;
  static constexpr int kChunks = kRowBytes / 16;
  static constexpr int kTileBytes = kTile * kPitch;
  static constexpr int kStages = LONG ? (E4M3 ? 5 : 2) : DP == 64 ? 4 : E4M3 ? 2 : 3;
  static constexpr int kSmem = kStages * 2 * kTileBytes;
};

// NH: blocks of 8 query heads.
template <bool E4M3, int DP, int NH, bool LONG>
__global__ void __launch_bounds__(kThreadsD) decode_kernel(const __grid_constant__ DecodeLaunch p) {
  using Cfg = DecodeCfg<E4M3, DP, LONG>;
  using elem = typename KvElem<E4M3>::type;
  constexpr int kSt = Cfg::kStages, kTile = Cfg::kTile, kTokW = Cfg::kTokW, kPitch = Cfg::kPitch, kRows = 8 * NH;
  constexpr int kKSteps = DP / 16, kMT = DP / kWarps / 16, kTT = kTokW / 16;  // 16-channel steps, 16-channel tiles, 16-token tiles of a warp
  extern __shared__ __align__(128) unsigned char ring[];
  __shared__ __align__(16) unsigned short prob[2][NH][kTile][8];  // [head block][token][head]
  __shared__ float wmax[kWarps][kRows], wsum[kWarps][kRows];
  __shared__ unsigned there[kSt][kTile / 32];  // which tokens of a tile exist
  __shared__ unsigned long long full[kSt], empty[kSt];
  __shared__ int red[kThreadsD / 32 + 2];
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  const int D = p.c.D;
  const unsigned ring_u = smem_u32(ring);
  pdl_launch_dependents();
  if (tid == 0) {
    // a stage is full when the copies of the copying warps' threads have landed and their words on the tokens are written
    for (int i = 0; i < kSt; i++) mbar_init(smem_u32(&full[i]), 33 * kCopyWarps), mbar_init(smem_u32(&empty[i]), kWarps);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (D < DP) {  // channels [D, DP) of every row stay zero (the copies never touch them)
    for (int i = tid; i < Cfg::kSmem / 16; i += kThreadsD) reinterpret_cast<uint4*>(ring)[i] = make_uint4(0u, 0u, 0u, 0u);
  }
  pdl_wait();

  Cursor cur;
  int n_my;  // tiles of this CTA's run, which starts at the cursor
  if (p.cluster == 0) {
    int total, before, per = 0;
    locate<kTile>(p, red, [&](int t) { return int(blockIdx.x) * (per = (t + p.ctas - 1) / p.ctas); }, total, cur.b, before);
    const int t0 = min(total, int(blockIdx.x) * per);
    n_my = min(total, t0 + per) - t0;
    if (n_my > 0) {
      cursor_sequence<kTile>(p, cur);
      cur.head = (t0 - before) / cur.n_tiles;
      cursor_part(cur, (t0 - before) % cur.n_tiles, n_my);
      // The part is gone through from its first multiple of the run's length on and then from its start: the CTAs with other heads
      // of the same tokens, whose parts start elsewhere, are then at the same tokens at the same time, and those lie side by
      // side in a page (8 sequences of 60000 e4m3 tokens, 4 heads of 64: 44 against 53 us; 8 heads of 128: 134 against 139; bf16 rows,
      // which fill whole lines, the same as before).
      const int from = (cur.lo + per - 1) / per * per;
      if (from < cur.hi) cur.tile = from;
    }
  } else {
    const int item = int(blockIdx.x) / p.cluster, rank = int(blockIdx.x) - item * p.cluster;
    cur.b = item / p.heads, cur.head = item - cur.b * p.heads;
    cur.v = view_of(p, cur.b);
    cur.n_tiles = tiles_in<kTile>(cur.v.len);
    const int lo = rank * cur.n_tiles / p.cluster;
    n_my = (rank + 1) * cur.n_tiles / p.cluster - lo;
    cur.tile = cur.lo = lo, cur.hi = lo + n_my, cur.left = n_my, cur.rest = 0;
    __syncthreads();  // barriers and zeroed channels are there
  }
  // sequences that have no token in view: out 0, lse -inf
  for (int b = blockIdx.x; b < p.c.n_seqs; b += gridDim.x) {
    if (view_of(p, b).len > 0) continue;
    for (int64_t i = tid; i < int64_t(p.a.H) * D; i += kThreadsD) p.a.out[int64_t(b) * p.a.H * D + i] = 0;
    if (p.a.lse)
      for (int64_t i = tid; i < p.a.H; i += kThreadsD) p.a.lse[int64_t(b) * p.a.H + i] = -INFINITY;
  }
  const bool joins = p.cluster > 1 && cur.n_tiles > 0;  // the same for the whole cluster
  if (n_my <= 0 && (!joins || warp >= kWarps)) return;

  bool ok = true;

  if (warp >= kWarps) {
    // ---- the copying warps ----
    constexpr int kPerInstr = 32 / Cfg::kChunks;  // rows per instruction
    const int ch = lane % Cfg::kChunks, sub = lane / Cfg::kChunks, part = warp - kWarps;
    const bool copies = ch * 16 < D * int(sizeof(elem));
    const unsigned char* kb = static_cast<const unsigned char*>(p.c.k) + ch * 16;
    const int64_t to_v = static_cast<const unsigned char*>(p.c.v) - static_cast<const unsigned char*>(p.c.k);
    // Page and slot of tokens 32 (kPL part + x) + lane of the tile that is copied next (slot -1: no token), asked for before the
    // tile in front of it is copied and not looked at until then, so that the page table's latency passes meanwhile.
    constexpr int kPL = Cfg::kPerLane;
    int page[kPL], slot[kPL];
    int64_t head_off;
    auto look_up = [&]() {
      head_off = int64_t(cur.head / p.blocks) * p.c.head_stride;
#pragma unroll
      for (int x = 0; x < kPL; x++) {
        const unsigned i = unsigned(cur.tile) * kTile + unsigned((part * kPL + x) * 32 + lane);  // may pass 31 bits, in the last tile
        page[x] = 0, slot[x] = -1;
        if (i < unsigned(cur.v.len)) {  // inside the table: the length is held to it
          const int tok = int(i < unsigned(cur.v.first) ? i : i - unsigned(cur.v.first) + unsigned(cur.v.skip));
          // tok / page_size by the reciprocal rounded down, at most one too small for tok < 2^31
          int n = int(__umulhi(unsigned(tok), p.page_recip)), r = tok - n * p.c.page_size;
          if (r >= p.c.page_size) n++, r -= p.c.page_size;
          slot[x] = r;
          page[x] = p.c.page_table[int64_t(cur.b) * p.c.table_stride + n];
        }
      }
      cursor_next<kTile>(p, cur);
    };
    look_up();
    int st = 0;
    for (int i = 0; i < n_my; i++) {
      int64_t off[kPL];  // byte offsets, -1: not there
#pragma unroll
      for (int x = 0; x < kPL; x++) {
        off[x] = -1;
        if (slot[x] >= 0) {
          if (page[x] >= 0 && page[x] < p.c.num_pages)
            off[x] = (int64_t(page[x]) * p.c.page_stride + int64_t(slot[x]) * p.c.token_stride + head_off) * int(sizeof(elem));
          else if (p.err)
            atomicExch(p.err, kErrBadIndex);
        }
      }
      if (i + 1 < n_my) look_up();
      if (i >= kSt) {
        // (the computing warps come to their arrival whatever becomes of their own waits, which p.tries bounds)
        ok = __all_sync(0xffffffffu, mbar_wait_spin(smem_u32(&empty[st]), unsigned(i / kSt - 1) & 1u, 0xffffffffu));
        if (!ok) break;
      }
#pragma unroll
      for (int x = 0; x < kPL; x++) {
        const unsigned dk = ring_u + unsigned(st) * 2 * Cfg::kTileBytes + unsigned(((part * kPL + x) * 32 + sub) * kPitch + ch * 16);
        const unsigned word = __ballot_sync(0xffffffffu, off[x] >= 0);
        if (lane == 0) there[st][part * kPL + x] = word;
#pragma unroll
        for (int r = 0; r < 32 / kPerInstr; r++) {
          const int64_t o = __shfl_sync(0xffffffffu, off[x], r * kPerInstr + sub);
          if (copies) {  // a token that is not there reads as zeros: its value must not carry anything into 0 * v
            const unsigned n = o >= 0 ? 16u : 0u;
            const unsigned char* from = kb + (o >= 0 ? o : 0);
            cp_async16(dk + unsigned(r * kPerInstr * kPitch), from, n);
            cp_async16(dk + unsigned(Cfg::kTileBytes + r * kPerInstr * kPitch), from + to_v, n);
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
  // this warp's state.  Column c of a product is query head 8 nh + c; a lane holds columns 2 c2 and 2 c2 + 1 of rows r0 and
  // r0 + 8 (tokens of the scores, channels of the output), as a right operand column r0.
  float o[kMT][NH][4];
  float base[NH][2], l[NH][2], scale[NH][2];  // maximum in use (in units of log2, less kLift), this thread's part of the sum, of the columns
  unsigned qf[NH][kKSteps][2];
  const int r0 = lane >> 2, c2 = lane & 3;
  const Cursor start = cur;
  bool fresh = true;
  int st = 0, g = 0, rows = 0, h0 = 0;
  unsigned ph = 0;

  for (int i = 0; i < n_my; i++) {
    if (fresh) {  // a new (sequence, head): its queries into registers
      fresh = false;
      g = cur.head / p.blocks;
      const int blk = cur.head - g * p.blocks;
      rows = min(kRows, p.group - blk * kRows), h0 = g * p.group + blk * kRows;
      const float ks2 = p.scale2 * (E4M3 && p.c.k_scale ? p.c.k_scale[g] : 1.f);
      const mxk_bf16* q = p.a.q + int64_t(cur.b) * p.a.q_stride + int64_t(h0) * D;
#pragma unroll
      for (int nh = 0; nh < NH; nh++) {
#pragma unroll
        for (int m = 0; m < kMT; m++) o[m][nh][0] = o[m][nh][1] = o[m][nh][2] = o[m][nh][3] = 0.f;
        base[nh][0] = base[nh][1] = -INFINITY, l[nh][0] = l[nh][1] = 0.f;
        const int r = 8 * nh + r0;
        const bool on = r < rows;
        // channels of step s: 16 s + 2 c2 + {0, 1} and + 8; of an e4m3 cache 16 s + 4 c2 + {0, 1} and {2, 3}, the order its
        // keys are read in
        float big = 0.f;
#pragma unroll
        for (int s = 0; s < kKSteps; s++)
#pragma unroll
          for (int hi = 0; hi < 2; hi++) {
            const int d = 16 * s + (E4M3 ? 4 * c2 + 2 * hi : 2 * c2 + 8 * hi);
            const unsigned x = on && d < D ? *reinterpret_cast<const unsigned*>(q + int64_t(r) * D + d) : 0u;
            qf[nh][s][hi] = x;
            if (E4M3) big = fmaxf(big, fmaxf(fabsf(bf16_lo(x)), fabsf(bf16_hi(x))));
          }
        float down = ks2;
        if (E4M3) {
          // e4m3 keys are taken as f16, which holds them exactly; so are the queries, scaled by a power of two (per head)
          // that brings their largest into [2^13, 2^14): what f16 then loses lies 2^-38 below it.
          big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
          big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
          // exponent of `big` by its bits; zero, subnormal and infinite rows keep a factor that changes nothing that matters
          int e = int((__float_as_uint(big) >> 23) & 255) - 127;
          e = e < -110 ? -110 : e > 127 ? 127 : e;
          const float up = __uint_as_float(unsigned(127 + 13 - e) << 23);
          down *= __uint_as_float(unsigned(127 - 13 + e) << 23);
#pragma unroll
          for (int s = 0; s < kKSteps; s++)
#pragma unroll
            for (int hi = 0; hi < 2; hi++) qf[nh][s][hi] = pack_f16(bf16_lo(qf[nh][s][hi]) * up, bf16_hi(qf[nh][s][hi]) * up);
        }
        // the factor of head r0 goes to the lanes whose columns it is
        scale[nh][0] = __shfl_sync(0xffffffffu, down, 8 * c2), scale[nh][1] = __shfl_sync(0xffffffffu, down, 8 * c2 + 4);
      }
    }
    // A wait that runs out does not leave the loop: the four warps go on meeting, without waiting for anything else.
    ok = ok && __all_sync(0xffffffffu, mbar_wait_spin(smem_u32(&full[st]), ph, p.tries));
    const unsigned k_u = ring_u + unsigned(st) * 2 * Cfg::kTileBytes, v_u = k_u + Cfg::kTileBytes;

    // ---- scores of this warp's tokens ----
    float s[kTT][NH][4];
#pragma unroll
    for (int t = 0; t < kTT; t++)
#pragma unroll
      for (int nh = 0; nh < NH; nh++) s[t][nh][0] = s[t][nh][1] = s[t][nh][2] = s[t][nh][3] = 0.f;
    if (!E4M3) {
      const unsigned a = k_u + unsigned((warp * kTokW + (lane & 15)) * kPitch + (lane >> 4) * 16);
#pragma unroll
      for (int ks = 0; ks < kKSteps; ks++)
#pragma unroll
        for (int t = 0; t < kTT; t++) {
          unsigned k[4];
          ldsm4(a + unsigned(t * 16 * kPitch + ks * 32), k);
#pragma unroll
          for (int nh = 0; nh < NH; nh++) mma16816<false>(s[t][nh], k, qf[nh][ks][0], qf[nh][ks][1]);
        }
    } else {
      // two 16-byte chunks of 16 tokens: a register holds four channels of one token, two pairs of one 16-channel step
      const unsigned a = k_u + unsigned((warp * kTokW + (lane & 15)) * kPitch + (lane >> 4) * 16);
#pragma unroll
      for (int ks = 0; ks < kKSteps; ks += 2)
#pragma unroll
        for (int t = 0; t < kTT; t++) {
          unsigned w[4];
          ldsm4(a + unsigned(t * 16 * kPitch + ks * 16), w);
#pragma unroll
          for (int x = 0; x < 2; x++) {
            unsigned k[4];
            e4m3x4_to_f16(w[2 * x], k[0], k[2]), e4m3x4_to_f16(w[2 * x + 1], k[1], k[3]);
#pragma unroll
            for (int nh = 0; nh < NH; nh++) mma16816<true>(s[t][nh], k, qf[nh][ks + x][0], qf[nh][ks + x][1]);
          }
        }
    }
    // the warp's bits of the tile's tokens
    const unsigned word = there[st][warp * kTokW / 32] >> (warp * kTokW % 32);
    constexpr unsigned kAll = kTokW == 32 ? 0xffffffffu : 0xffffu;
    const bool all_there = (word & kAll) == kAll;
    float mx[NH][2];
    bool grows = false;
#pragma unroll
    for (int nh = 0; nh < NH; nh++) {
#pragma unroll
      for (int t = 0; t < kTT; t++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
          s[t][nh][e] *= scale[nh][e & 1];
          if (!all_there && !(word >> (16 * t + 8 * (e >> 1) + r0) & 1u)) s[t][nh][e] = -INFINITY;
        }
#pragma unroll
      for (int c = 0; c < 2; c++) {
        mx[nh][c] = fmaxf(s[0][nh][c], s[0][nh][2 + c]);
#pragma unroll
        for (int t = 1; t < kTT; t++) mx[nh][c] = fmaxf(mx[nh][c], fmaxf(s[t][nh][c], s[t][nh][2 + c]));
        if (E4M3) mx[nh][c] -= kLift;
        grows |= mx[nh][c] > base[nh][c] + kSlack;
      }
    }
    float add[NH][2];
    auto probabilities = [&]() {
#pragma unroll
      for (int nh = 0; nh < NH; nh++) {
        const float b0 = base[nh][0] == -INFINITY ? 0.f : base[nh][0];  // nothing seen yet: exp2(-inf - 0) = 0 everywhere
        const float b1 = base[nh][1] == -INFINITY ? 0.f : base[nh][1];
        add[nh][0] = add[nh][1] = 0.f;
#pragma unroll
        for (int t = 0; t < kTT; t++)
#pragma unroll
          for (int half = 0; half < 2; half++) {
            const float p0 = ex2_approx(s[t][nh][2 * half] - b0), p1 = ex2_approx(s[t][nh][2 * half + 1] - b1);
            add[nh][0] += p0, add[nh][1] += p1;
            *reinterpret_cast<unsigned*>(&prob[i & 1][nh][warp * kTokW + 16 * t + 8 * half + r0][2 * c2]) = E4M3 ? pack_f16(p0, p1) : pack_bf16(p0, p1);
          }
      }
    };
    probabilities();
    if (vote(grows)) {  // always in a segment's first tile
#pragma unroll
      for (int nh = 0; nh < NH; nh++)
#pragma unroll
        for (int c = 0; c < 2; c++) {
#pragma unroll
          for (int x = 4; x < 32; x <<= 1) mx[nh][c] = fmaxf(mx[nh][c], __shfl_xor_sync(0xffffffffu, mx[nh][c], x));
          if (r0 == 0) wmax[warp][8 * nh + 2 * c2 + c] = mx[nh][c];
        }
      meet();
#pragma unroll
      for (int nh = 0; nh < NH; nh++)
#pragma unroll
        for (int c = 0; c < 2; c++) {
          float mn = base[nh][c];
#pragma unroll
          for (int w = 0; w < kWarps; w++) mn = fmaxf(mn, wmax[w][8 * nh + 2 * c2 + c]);
          if (mn != base[nh][c]) {
            const float f = ex2_approx(base[nh][c] - mn);  // 0 for the first maximum
            l[nh][c] *= f;
#pragma unroll
            for (int m = 0; m < kMT; m++) o[m][nh][c] *= f, o[m][nh][2 + c] *= f;
            base[nh][c] = mn;
          }
        }
      probabilities();
      meet();
    }
#pragma unroll
    for (int nh = 0; nh < NH; nh++) l[nh][0] += add[nh][0], l[nh][1] += add[nh][1];
    // ---- this warp's channels of the product with V ----
    const unsigned p_u = smem_u32(&prob[i & 1][0][lane][0]);
#pragma unroll
    for (int k2 = 0; k2 < kTile / 32; k2++) {  // 32 tokens, two steps
      unsigned pb[NH][4];
#pragma unroll
      for (int nh = 0; nh < NH; nh++) ldsm4_t(p_u + unsigned((nh * kTile + k2 * 32) * 16), pb[nh]);
      if (!E4M3) {
        const unsigned a = v_u + unsigned((k2 * 32 + (lane & 7) + ((lane >> 4) << 3)) * kPitch + (warp * kMT * 2 + ((lane >> 3) & 1)) * 16);
#pragma unroll
        for (int ks = 0; ks < 2; ks++)
#pragma unroll
          for (int m = 0; m < kMT; m++) {
            unsigned v[4];
            ldsm4_t(a + unsigned(ks * 16 * kPitch + m * 32), v);
#pragma unroll
            for (int nh = 0; nh < NH; nh++) mma16816<false>(o[m][nh], v, pb[nh][2 * ks], pb[nh][2 * ks + 1]);
          }
      } else {
        // A 16-bit transposed load of 8-bit pairs: register: (token 2c: channels 2n, 2n + 1), (token 2c + 1: the same); the
        // pairs of one channel are then its bytes 0, 2 and 1, 3: rows 0-7 of the product take the even channels of the 16,
        // rows 8-15 the odd ones.
#pragma unroll
        for (int m = 0; m < kMT; m++) {
          unsigned v[4];  // tokens 0-7, 8-15, 16-23, 24-31
          ldsm4_t(v_u + unsigned((k2 * 32 + lane) * kPitch + (warp * kMT + m) * 16), v);
#pragma unroll
          for (int ks = 0; ks < 2; ks++) {
            unsigned a[4];
            e4m3x4_to_f16(__byte_perm(v[2 * ks], 0, 0x3120), a[0], a[1]), e4m3x4_to_f16(__byte_perm(v[2 * ks + 1], 0, 0x3120), a[2], a[3]);
#pragma unroll
            for (int nh = 0; nh < NH; nh++) mma16816<true>(o[m][nh], a, pb[nh][2 * ks], pb[nh][2 * ks + 1]);
          }
        }
      }
    }
    __syncwarp();
    if (lane == 0) arrive(smem_u32(&empty[st]));
    if (++st == kSt) st = 0, ph ^= 1u;

    if (cur.left == 1) {  // the part ends: store
      const bool whole = cur.lo == 0 && cur.hi == cur.n_tiles && !joins;
#pragma unroll
      for (int nh = 0; nh < NH; nh++)
#pragma unroll
        for (int c = 0; c < 2; c++) {
#pragma unroll
          for (int x = 4; x < 32; x <<= 1) l[nh][c] += __shfl_xor_sync(0xffffffffu, l[nh][c], x);
          if (r0 == 0) wsum[warp][8 * nh + 2 * c2 + c] = l[nh][c];
        }
      meet();
      const float vs = E4M3 && p.c.v_scale ? p.c.v_scale[g] : 1.f;
      const int64_t slot = 2 * int64_t(blockIdx.x) + (cur.lo == 0 ? 1 : 0);
      // this part's place: a slot of the workspace, or this CTA's own stages, which nobody reads any more
      float* part_o = joins ? reinterpret_cast<float*>(ring) : p.part_o + slot * kRows * DP;
      float* part_ml = joins ? part_o + kRows * DP : p.part_ml + slot * kRows * 2;
#pragma unroll
      for (int nh = 0; nh < NH; nh++)
#pragma unroll
        for (int c = 0; c < 2; c++) {
          const int r = 8 * nh + 2 * c2 + c;
          if (r >= rows) continue;
          float sum = 0.f;
#pragma unroll
          for (int w = 0; w < kWarps; w++) sum += wsum[w][r];
          const float f = whole ? (sum > 0.f || sum != sum ? vs / sum : 0.f) : vs;
#pragma unroll
          for (int m = 0; m < kMT; m++) {
            // channels of o[m][nh][c] and o[m][nh][2 + c]
            const int d0 = (warp * kMT + m) * 16 + (E4M3 ? 2 * r0 : r0), d1 = E4M3 ? d0 + 1 : d0 + 8;
            const float v0 = o[m][nh][c] * f, v1 = o[m][nh][2 + c] * f;
            if (whole) {
              mxk_bf16* dst = p.a.out + (int64_t(cur.b) * p.a.H + h0 + r) * D;
              const unsigned w = pack_bf16(v0, v1);
              if (d0 < D) dst[d0] = mxk_bf16(w & 0xffffu);
              if (d1 < D) dst[d1] = mxk_bf16(w >> 16);
            } else {
              part_o[r * DP + d0] = v0, part_o[r * DP + d1] = v1;
            }
          }
          if (warp == 0 && r0 == 0) {
            if (!whole) {
              part_ml[2 * r] = base[nh][c], part_ml[2 * r + 1] = sum;
            } else if (p.a.lse) {
              p.a.lse[int64_t(cur.b) * p.a.H + h0 + r] = sum == 0.f ? -INFINITY : (base[nh][c] + log2f(sum)) * kLn2;
            }
          }
        }
      fresh = true;
    }
    cursor_next<kTile>(p, cur);
  }
  if (!ok && p.err) atomicExch(p.err, kErrBulkTimeout);
  if (joins) {
    // ---- the parts of the cluster's CTAs, in their order; each CTA adds up some of the heads, a channel per thread ----
    const int blk = start.head % p.blocks, item_h0 = start.head / p.blocks * p.group + blk * kRows, item_rows = min(kRows, p.group - blk * kRows);
    const unsigned ml_u = ring_u + unsigned(kRows * DP * sizeof(float));
    if (n_my <= 0 && tid < kRows) {
      float* part_ml = reinterpret_cast<float*>(ring) + kRows * DP;
      part_ml[2 * tid] = -INFINITY, part_ml[2 * tid + 1] = 0.f;
    }
    cluster_meet();
    for (int r = int(blockIdx.x) % p.cluster; r < item_rows; r += p.cluster) {
      float m[8], l[8], mx = -INFINITY;
#pragma unroll
      for (int c = 0; c < 8; c++) {
        m[c] = -INFINITY, l[c] = 0.f;
        if (c < p.cluster) ld_cluster2(ml_u + unsigned(r * 8), unsigned(c), m[c], l[c]);
        mx = fmaxf(mx, m[c]);
      }
      const float top = mx == -INFINITY ? 0.f : mx;
      float sum = 0.f, out = 0.f;
#pragma unroll
      for (int c = 0; c < 8; c++) {
        const float f = ex2_approx(m[c] - top);
        if (c < p.cluster && l[c] != 0.f && tid < D) {  // a part without a tile has no output
          sum = fmaf(l[c], f, sum);
          out = fmaf(ld_cluster(ring_u + unsigned((r * DP + tid) * 4), unsigned(c)), f, out);
        }
      }
      if (tid < D) {
        const int64_t at = int64_t(start.b) * p.a.H + item_h0 + r;
        p.a.out[at * D + tid] = mxk_bf16(pack_bf16(sum > 0.f || sum != sum ? out / sum : 0.f, 0.f) & 0xffffu);
        if (tid == 0 && p.a.lse) p.a.lse[at] = sum == 0.f ? -INFINITY : (mx + log2f(sum)) * kLn2;
      }
    }
    cluster_meet();  // nobody goes while its shared memory is read
  }
}

// Adds up, for each (sequence, head) that several runs share, the parts in the order of the runs: one CTA per work item and
// row, warp w taking parts w, w + 4, ... (all channels of a part per access, several parts in flight), the warps' sums in
// order at the end.
template <int DP, int TILE, int NH>
__global__ void __launch_bounds__(kConsumers) join_kernel(const __grid_constant__ DecodeLaunch p) {
  constexpr int kRows = 8 * NH;
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
  const int n_tiles = tiles_in<TILE>(view_of(p, b).len);
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

// A number as a type.
template <int N> using Int = std::integral_constant<int, N>;
// CTAs that the GPU holds at once.
template <bool E4M3, int DP, int NH, bool LONG>
int decode_ctas() {
  auto k = decode_kernel<E4M3, DP, NH, LONG>;
  allow_smem(k, DecodeCfg<E4M3, DP, LONG>::kSmem);  // a failure surfaces at the launch
  return sm_count() * resident_ctas(k, kThreadsD, DecodeCfg<E4M3, DP, LONG>::kSmem);
}

template <bool E4M3, int DP, int NH>
int launch_decode(const char* name, DecodeLaunch& p, cudaStream_t s) {
  constexpr bool kLong = DP == 64;  // of the form with runs
  constexpr int kRows = 8 * NH, kTile = DecodeCfg<E4M3, DP, kLong>::kTile, kShortTile = DecodeCfg<E4M3, DP, false>::kTile;
  p.ctas = decode_ctas<E4M3, DP, NH, kLong>();
  // tokens and tiles that a work item can have
  int64_t tokens = int64_t(p.c.max_pages) * p.c.page_size;
  if (p.a.left >= 0 && p.a.left < tokens && p.a.sinks < tokens - p.a.left) tokens = p.a.left + 1 + p.a.sinks;
  const int64_t item_tiles = ceil_div(tokens, kTile), items = int64_t(p.c.n_seqs) * p.heads;
  // no more runs than there can be tiles
  if (p.ctas > items * item_tiles) p.ctas = int(items * item_tiles < 1 ? 1 : items * item_tiles);
  const int64_t need = int64_t(2) * p.ctas * kRows * (DP + 2) * int64_t(sizeof(float));
  if (p.a.workspace_bytes < need)
    return fail(MXK_ERR_INVALID_ARG, "%s: workspace of %lld bytes, mxk_attn_decode_workspace_bytes() asks for up to %lld", name, (long long)p.a.workspace_bytes,
                (long long)need);
  p.part_o = static_cast<float*>(p.a.workspace);
  p.part_ml = p.part_o + int64_t(2) * p.ctas * kRows * DP;
  // The short form: as many CTAs per work item (1, 4, 8) as the GPU holds at once and the item has tiles.  One where it has no
  // more than kSingle tiles (16 sequences of 200 tokens, 4 heads of 64: 5.5 against 6.7 us with four, and 9.6 with two for 64 of
  // them); two, which add up no faster than eight, only where one would be too few for this form (32 of 300: 6.7 against 8.9 us
  // with two; but 24 of 1000, 8 heads of 128, e4m3: two 14.2 us, runs 15.6).  (Whole items against runs: 64 sequences of 2000
  // bf16 tokens, 512 items on 296 CTAs, 85 against 96 us; 40 of 1024, 320 items, 40 against 38 us; 200 of 1024 e4m3 tokens, 1600 items
  // on 740 CTAs, 65 against 74 us; 64 of 2000, 512 items, 49 against 45 us.)
  const int64_t resident = decode_ctas<E4M3, DP, NH, false>(), short_tiles = ceil_div(tokens, kShortTile);
  int c = 1;
  while (short_tiles > kSingle && c < 8 && items * c * 2 <= resident && c < short_tiles) c *= 2;
  if (c == 2 && short_tiles <= kShort) c = 1;
  auto one_launch = [&](auto long_tiles) {
    constexpr bool kL = long_tiles.value != 0;
    p.cluster = c;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(unsigned(items * c)), cfg.blockDim = dim3(kThreadsD), cfg.dynamicSmemBytes = DecodeCfg<E4M3, DP, kL>::kSmem, cfg.stream = s;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = unsigned(c), at[0].val.clusterDim.y = 1, at[0].val.clusterDim.z = 1;
    at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at, cfg.numAttrs = pdl_enabled() ? 2 : 1;
    cudaLaunchKernelEx(&cfg, decode_kernel<E4M3, DP, NH, kL>, p);  // errors surface through cudaGetLastError() in after_launch()
    return after_launch(name);
  };
  if (ceil_div(short_tiles, c) <= (2 * items >= 3 * resident ? kMedium : kShort) && items * c < (int64_t(1) << 31)) return one_launch(Int<0>());
  // Whole items of LONG tiles where those have two CTAs per SM to fill: 200 sequences of 2000 e4m3 tokens, 4 heads of 64, 42 against
  // 52 us by runs, of 4000 73 against 100; bf16, the same either way (54 and 97 against 53 and 98), follows the rule.
  if constexpr (kLong) {
    c = 1;
    if (item_tiles <= kMedium && 2 * items >= 3 * int64_t(decode_ctas<E4M3, DP, NH, true>()) && items < (int64_t(1) << 31)) return one_launch(Int<1>());
  }
  p.cluster = 0;
  launch_pdl(decode_kernel<E4M3, DP, NH, kLong>, dim3(unsigned(p.ctas)), dim3(kThreadsD), DecodeCfg<E4M3, DP, kLong>::kSmem, s, p);
  if (int rc = after_launch(name)) return rc;
  launch_pdl(join_kernel<DP, kTile, NH>, dim3(unsigned(items), unsigned(p.group < kRows ? p.group : kRows)), dim3(kConsumers), 0, s, p);
  return after_launch(name);
}

// The kernel for a cache and head count: f(e4m3, padded head dimension, blocks of 8 heads), as types.
template <class F>
auto pick_decode(const MxkKvCache* c, int group, F f) {
  const bool e = c->type == MXK_KV_E4M3, small = c->D <= 64;
  auto with_heads = [&](auto type, auto dp) { return group <= 8 ? f(type, dp, Int<1>()) : f(type, dp, Int<2>()); };
  if (e) return small ? with_heads(Int<1>(), Int<64>()) : with_heads(Int<1>(), Int<128>());
  return small ? with_heads(Int<0>(), Int<64>()) : with_heads(Int<0>(), Int<128>());
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
  const int64_t bytes = pick_decode(cache, H / cache->Hkv, [](auto e, auto dp, auto nh) {
    return int64_t(2) * decode_ctas<e.value != 0, dp.value, nh.value, dp.value == 64>() * (8 * nh.value) * (dp.value + 2) * int64_t(sizeof(float));
  });
  cudaGetLastError();  // without a GPU the size is that of the usual one
  return bytes;
}

int mxk_attn_decode_paged(const MxkDecodeArgs* args, const MxkKvCache* cache, mxk_stream_t stream) {
  const char* name = "attn_decode_paged";
  if (!args) return fail(MXK_ERR_INVALID_ARG, "%s: null args", name);
  if (int rc = check_cache(name, cache)) return rc;
  if (cache->n_seqs <= 0) return MXK_OK;
  if (int rc = check_heads(name, cache, args->H)) return rc;
  if (cache->max_pages > 0 && !cache->page_table) return fail(MXK_ERR_INVALID_ARG, "%s: null page table", name);
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
  if (!(a.scale > 0.f) || a.scale > 1e30f) return fail(MXK_ERR_INVALID_ARG, "%s: scale must be positive and at most 1e30", name);
  // without a page every token is left out; the copies of no bytes that stand for it then have an address that exists
  if (cache->num_pages == 0) p.c.k = p.c.v = const_cast<mxk_bf16*>(a.q);
  p.group = a.H / cache->Hkv;
  p.blocks = int(ceil_div(p.group, 16));
  p.heads = cache->Hkv * p.blocks;
  const int64_t tiles = int64_t(cache->n_seqs) * p.heads * (ceil_div(int64_t(cache->max_pages) * cache->page_size, 64) + 1);
  if (tiles >= (int64_t(1) << 30)) return fail(MXK_ERR_TOO_LARGE, "%s: n_seqs * heads * tokens too large (%lld tiles)", name, (long long)tiles);
  p.scale2 = a.scale * kLog2e;
  // A warp may have to wait while another passes over sequences without a token, one look at a length each, less than 1.5 us.
  const int64_t tries = tune(TUNE_DECODE_WAIT_TRIES, int(kSpinTries)) + 4 * int64_t(cache->n_seqs);
  p.tries = unsigned(tries < 0xffffffffll ? tries : 0xffffffffll);
  p.page_recip = 0xffffffffu / unsigned(cache->page_size);
  p.err = device_error_word();
  const cudaStream_t s = as_stream(stream);
  return pick_decode(cache, p.group, [&](auto e, auto dp, auto nh) { return launch_decode<e.value != 0, dp.value, nh.value>(name, p, s); });
}

}  // extern "C"
