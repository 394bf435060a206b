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
// Split: a tile is kTile tokens of one (sequence, key head, block of 16 query heads).  All tiles of the call in order
// (sequence, head, token) are cut into equal runs, one per resident CTA, whatever the lengths are - a CTA's run may
// end inside a sequence's tokens and cover several short sequences.  Each CTA finds the run's start itself by summing the
// lengths.  A run that covers a (sequence, head) alone writes its output; otherwise the CTA leaves its running maximum,
// sum and unnormalised output in its slots of the workspace (one for the segment its run starts in, one for the segment
// it ends in) and join_kernel, launched behind it, adds them up in order.  Results do not depend on timing.
//
// Within a CTA (4 warps): tiles of K and V come through a ring of shared-memory stages (16-byte cp.async, rows found
// through the page table one tile ahead).  For the scores each warp takes kTile / 4 tokens; for the product with V each
// warp takes D / 4 channels of all of them, so that the output stays in a few registers; maxima and probabilities pass
// through shared memory.  Scores, maxima, sums and output are fp32; probabilities are rounded to bf16 (f16 for an e4m3
// cache) for the product, as the tensor instruction needs the type of V.
#include <cuda_fp16.h>

#include "bulk_copy.cuh"
#include "common.cuh"
#include "kv_cache.cuh"

namespace mxk {
namespace {

constexpr int kRows = 16;       // query heads per work item
constexpr int kWarps = 4;
constexpr int kThreadsD = 32 * kWarps;
constexpr int kTile = 64;       // tokens per tile
constexpr int kTokW = kTile / kWarps;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct DecodeLaunch {
  MxkDecodeArgs a;
  MxkKvCache c;
  int group;       // query heads per key head
  int blocks;      // blocks of 16 of those
  int heads;       // Hkv * blocks: work items per sequence
  int ctas;        // runs
  float scale2;    // scale * log2(e)
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
__device__ __forceinline__ int tiles_of(const DecodeLaunch& p, int b) { return (view_of(p, b).len + kTile - 1) / kTile * p.heads; }

// Finds, with the whole CTA: the number of tiles of the call, and for tile `want` of the caller's choosing (a function of
// the total) the sequence it lies in and the number of tiles in front of that sequence.
template <class Want>
__device__ __forceinline__ void locate(const DecodeLaunch& p, int* red, Want want, int& total, int& seq, int& before) {
  const int n = p.c.n_seqs, t = threadIdx.x, lane = t & 31, warp = t >> 5;
  int mine = 0;  // thread t sums a contiguous share of the sequences
  const int share = (n + kThreadsD - 1) / kThreadsD, b0 = min(n, t * share), b1 = min(n, b0 + share);
  for (int b = b0; b < b1; b++) mine += tiles_of(p, b);
  int incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += x;
  }
  if (lane == 31) red[warp] = incl;
  if (t == 0) red[kWarps] = -1;
  __syncthreads();
  int base = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kWarps; w++) {
    if (w < warp) base += red[w];
    total += red[w];
  }
  int at = base + incl - mine;
  const int target = want(total);
  if (target >= at && target < at + mine) {
    int b = b0;
    for (int k = tiles_of(p, b); target >= at + k; k = tiles_of(p, b)) at += k, b++;
    red[kWarps] = b, red[kWarps + 1] = at;
  }
  __syncthreads();
  seq = red[kWarps], before = red[kWarps + 1];
}

// A place in the order of tiles.
struct Cursor {
  int b, head, tile, n_tiles;  // tile of n_tiles of work item `head` (key head * blocks + block) of sequence b
  View v;
};
__device__ __forceinline__ void cursor_sequence(const DecodeLaunch& p, Cursor& c) {  // sequences without a token are passed over
  while (c.b < p.c.n_seqs) {
    c.v = view_of(p, c.b);
    c.n_tiles = (c.v.len + kTile - 1) / kTile;
    if (c.n_tiles > 0) return;
    c.b++;
  }
}
__device__ __forceinline__ void cursor_next(const DecodeLaunch& p, Cursor& c) {
  if (++c.tile < c.n_tiles) return;
  c.tile = 0;
  if (++c.head < p.heads) return;
  c.head = 0, c.b++;
  cursor_sequence(p, c);
}

__device__ __forceinline__ void cp_async16(unsigned dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
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

// Shared-memory layout of a stage: rows of DP elements, one per token, in 16-byte chunks; chunk j of row t sits at
// chunk position chunk_at(t, j), which keeps the eight rows an ldmatrix phase (or the two rows a 128-bit load phase of
// the e4m3 keys) reads off each other's banks.
template <bool E4M3, int DP, bool IS_V>
__device__ __forceinline__ int chunk_at(int t, int j) {
  if (!E4M3) return j ^ (t & 7);                                      // rows of 256 or 128 bytes
  if (DP == 128) return IS_V ? j ^ (t & 7) : j ^ ((t & 1) << 2);      // rows of 128 bytes
  return IS_V ? j ^ ((t >> 1) & 3) : j;                               // rows of 64 bytes
}

template <bool E4M3, int DP>
struct DecodeCfg {
  static constexpr int kRowBytes = DP * (E4M3 ? 1 : 2);
  static constexpr int kChunks = kRowBytes / 16;
  static constexpr int kTileBytes = kTile * kRowBytes;
  static constexpr int kStages = E4M3 || DP == 64 ? 4 : 3;
  static constexpr int kSmem = kStages * 2 * kTileBytes;
};

template <bool E4M3, int DP>
__global__ void __launch_bounds__(kThreadsD) decode_kernel(const __grid_constant__ DecodeLaunch p) {
  using Cfg = DecodeCfg<E4M3, DP>;
  using elem = typename KvElem<E4M3>::type;
  constexpr int kSt = Cfg::kStages, kKSteps = DP / 16, kNW = DP / kWarps / 8;  // k-steps of the scores; 8-channel tiles per warp
  extern __shared__ __align__(128) unsigned char ring[];
  __shared__ int64_t offs[kSt + 1][kTile];  // element offset of each token of a tile (its head included), -1: not there
  __shared__ float wmax[kWarps][kRows], wsum[kWarps][kRows];
  __shared__ __align__(16) unsigned short prob[kRows][kTile + 8];
  __shared__ int red[kWarps + 2];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int D = p.c.D, chunks = D * int(sizeof(elem)) / 16;
  pdl_launch_dependents();
  // channels [D, DP) of every row stay zero (the copies never touch them)
  if (D < DP) {
    for (int i = tid; i < Cfg::kSmem / 16; i += kThreadsD) reinterpret_cast<uint4*>(ring)[i] = make_uint4(0u, 0u, 0u, 0u);
  }
  pdl_wait();

  int total, seq0, before;
  int per = 0;
  locate(p, red, [&](int t) { return int(blockIdx.x) * (per = (t + p.ctas - 1) / p.ctas); }, total, seq0, before);
  const int t0 = min(total, int(blockIdx.x) * per), t1 = min(total, t0 + per);
  // sequences that have no token in view: out 0, lse -inf
  for (int b = blockIdx.x; b < p.c.n_seqs; b += gridDim.x) {
    if (view_of(p, b).len > 0) continue;
    for (int i = tid; i < p.a.H * D; i += kThreadsD) p.a.out[int64_t(b) * p.a.H * D + i] = 0;
    if (p.a.lse)
      for (int i = tid; i < p.a.H; i += kThreadsD) p.a.lse[int64_t(b) * p.a.H + i] = -INFINITY;
  }
  if (t0 >= t1) return;

  Cursor cur;  // of the arithmetic
  cur.b = seq0;
  cursor_sequence(p, cur);
  cur.head = (t0 - before) / cur.n_tiles, cur.tile = (t0 - before) % cur.n_tiles;
  Cursor look = cur;  // of the page look-ups, kSt tiles ahead
  const int n_my = t1 - t0;
  int looked = 0;
  // the page look-up of one tile: thread t the tile's token t
  auto look_up = [&]() -> int64_t {
    int64_t off = -1;
    if (looked < n_my) {
      if (tid < kTile) {
        const int i = look.tile * kTile + tid;
        if (i < look.v.len) {
          const int tok = i < look.v.first ? i : i - look.v.first + look.v.skip;
          off = kv_token_offset(p.c, look.b, tok);
          if (off < 0) {
            if (p.err) atomicExch(p.err, kErrBadIndex);
          } else {
            off += int64_t(look.head / p.blocks) * p.c.head_stride;
          }
        }
      }
      cursor_next(p, look);
    }
    looked++;
    return off;
  };
  const unsigned ring_u = smem_u32(ring);
  auto copy_tile = [&](int i) {  // tile i of the run into its stage
    if (i < n_my) {
      const unsigned st = ring_u + unsigned(i % kSt) * 2 * Cfg::kTileBytes;
      const int64_t* of = offs[i % (kSt + 1)];
      for (int j = tid; j < kTile * chunks; j += kThreadsD) {
        const int t = D == DP ? j / Cfg::kChunks : j / chunks, ch = D == DP ? j % Cfg::kChunks : j - t * chunks;
        const int64_t off = of[t];
        const unsigned dk = st + unsigned(t * Cfg::kRowBytes + chunk_at<E4M3, DP, false>(t, ch) * 16);
        const unsigned dv = st + Cfg::kTileBytes + unsigned(t * Cfg::kRowBytes + chunk_at<E4M3, DP, true>(t, ch) * 16);
        if (off >= 0) {
          cp_async16(dk, static_cast<const elem*>(p.c.k) + off + ch * (16 / int(sizeof(elem))));
          cp_async16(dv, static_cast<const elem*>(p.c.v) + off + ch * (16 / int(sizeof(elem))));
        } else {  // a token that is not there: its value must not carry anything into 0 * v
          const uint4 z = make_uint4(0u, 0u, 0u, 0u);
          *reinterpret_cast<uint4*>(ring + (dk - ring_u)) = z;
          *reinterpret_cast<uint4*>(ring + (dv - ring_u)) = z;
        }
      }
    }
    cp_commit();
  };
  for (int i = 0; i < kSt; i++) {
    const int64_t off = look_up();
    if (tid < kTile) offs[i][tid] = off;
  }
  __syncthreads();
  for (int i = 0; i < kSt - 1; i++) copy_tile(i);

  // this warp's state: rows r0 = lane / 4 and r0 + 8; channel tile n of the warp: channels (warp * kNW + n) * 8 ..
  // (e4m3: see the product with V) of the output
  float o[kNW][4];
  float m[2], l[2];
  unsigned qf[kKSteps][4];
  float qs[2] = {1.f, 1.f};
  const int r0 = lane >> 2, c2 = (lane & 3) * 2;
  bool fresh = true;
  int first_tile = cur.tile;

  for (int i = 0; i < n_my; i++) {
    const int64_t next_off = look_up();  // of tile i + kSt; the page table's latency passes during this tile
    const int g = cur.head / p.blocks, blk = cur.head % p.blocks;
    const int rows = min(kRows, p.group - blk * kRows);
    const int h0 = g * p.group + blk * kRows;
    if (fresh) {  // a new (sequence, head): its queries into registers
      fresh = false, first_tile = cur.tile;
#pragma unroll
      for (int n = 0; n < kNW; n++) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
      m[0] = m[1] = -INFINITY, l[0] = l[1] = 0.f;
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
          // a 64-channel group is the one the keys are read in: step s, lane c: channels 16 c + 4 s + {0, 1 | 2, 3}.
          unsigned raw[kKSteps][2];
          float big = 0.f;
#pragma unroll
          for (int s = 0; s < kKSteps; s++)
#pragma unroll
            for (int hi = 0; hi < 2; hi++) {
              const int d = 64 * (s / 4) + 8 * c2 + 4 * (s % 4) + 2 * hi;
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
    cp_wait<kSt - 2>();
    __syncthreads();  // tile i has landed for everyone, and nobody still reads the stage that is filled next
    copy_tile(i + kSt - 1);

    // ---- scores of this warp's 16 tokens ----
    const unsigned char* kt = ring + (i % kSt) * 2 * Cfg::kTileBytes;
    const unsigned k_u = ring_u + unsigned(i % kSt) * 2 * Cfg::kTileBytes, v_u = k_u + Cfg::kTileBytes;
    float s[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
    if (!E4M3) {
      const int t = warp * kTokW + (lane & 7) + ((lane >> 4) << 3), hi = (lane >> 3) & 1;
#pragma unroll
      for (int ks = 0; ks < kKSteps; ks++) {
        unsigned b[4];
        ldsm4(k_u + unsigned(t * Cfg::kRowBytes + chunk_at<E4M3, DP, false>(t, 2 * ks + hi) * 16), b);
        mma16816<false>(s[0], qf[ks], b[0], b[1]);
        mma16816<false>(s[1], qf[ks], b[2], b[3]);
      }
    } else {
#pragma unroll
      for (int n = 0; n < 2; n++) {
        const int t = warp * kTokW + 8 * n + r0;
#pragma unroll
        for (int grp = 0; grp < DP / 64; grp++) {
          const uint4 kv = *reinterpret_cast<const uint4*>(kt + t * Cfg::kRowBytes + chunk_at<E4M3, DP, false>(t, 4 * grp + (lane & 3)) * 16);
          const unsigned w[4] = {kv.x, kv.y, kv.z, kv.w};
#pragma unroll
          for (int ks = 0; ks < 4; ks++) mma16816<true>(s[n], qf[4 * grp + ks], e4m3x2_to_f16x2(w[ks] & 0xffffu), e4m3x2_to_f16x2(w[ks] >> 16));
        }
      }
    }
    const float ks2 = p.scale2 * (E4M3 && p.c.k_scale ? p.c.k_scale[g] : 1.f);
    const int64_t* of = offs[i % (kSt + 1)] + warp * kTokW;
    float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int n = 0; n < 2; n++)
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const bool there = of[8 * n + c2 + (e & 1)] >= 0;
        s[n][e] = there ? s[n][e] * (E4M3 ? ks2 * qs[e >> 1] : ks2) : -INFINITY;
        mx[e >> 1] = fmaxf(mx[e >> 1], s[n][e]);
      }
#pragma unroll
    for (int h = 0; h < 2; h++) {
      mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 1));
      mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 2));
      if ((lane & 3) == 0) wmax[warp][r0 + 8 * h] = mx[h];
    }
    __syncthreads();
    if (tid < kTile) offs[(i + kSt) % (kSt + 1)][tid] = next_off;  // the slot of tile i - 1
    float base[2];
#pragma unroll
    for (int h = 0; h < 2; h++) {
      float mn = m[h];
#pragma unroll
      for (int w = 0; w < kWarps; w++) mn = fmaxf(mn, wmax[w][r0 + 8 * h]);
      base[h] = mn == -INFINITY ? 0.f : mn;  // nothing seen yet: exp2(-inf - 0) = 0 everywhere
      if (mn != m[h]) {
        const float f = ex2_approx(m[h] - base[h]);  // 0 for the first maximum
        l[h] *= f;
#pragma unroll
        for (int n = 0; n < kNW; n++) o[n][2 * h] *= f, o[n][2 * h + 1] *= f;
        m[h] = mn;
      }
    }
#pragma unroll
    for (int n = 0; n < 2; n++)
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const float p0 = ex2_approx(s[n][2 * h] - base[h]), p1 = ex2_approx(s[n][2 * h + 1] - base[h]);
        l[h] += p0 + p1;
        *reinterpret_cast<unsigned*>(&prob[r0 + 8 * h][warp * kTokW + 8 * n + c2]) = E4M3 ? pack_f16(p0, p1) : pack_bf16(p0, p1);
      }
    __syncthreads();
    // ---- this warp's channels of the product with V ----
#pragma unroll
    for (int ks = 0; ks < kTile / 16; ks++) {
      unsigned pa[4];
      ldsm4(smem_u32(&prob[(lane & 7) + (((lane >> 3) & 1) << 3)][16 * ks + ((lane >> 4) << 3)]), pa);
      const int t = 16 * ks + (lane & 7) + (((lane >> 3) & 1) << 3);
      if (!E4M3) {
#pragma unroll
        for (int n = 0; n < kNW; n += 2) {
          unsigned b[4];
          ldsm4_t(v_u + unsigned(t * Cfg::kRowBytes + chunk_at<E4M3, DP, true>(t, warp * kNW + n + (lane >> 4)) * 16), b);
          mma16816<false>(o[n], pa, b[0], b[1]);
          mma16816<false>(o[n + 1], pa, b[2], b[3]);
        }
      } else {
        // a 16-bit transposed load of 8-bit pairs: register: (token 2c: channels 2n, 2n + 1), (token 2c + 1: the same);
        // the pairs of one channel are then its bytes 0, 2 and 1, 3, so two channel tiles hold the even and the odd ones
        constexpr int kPairs = kNW / 2;  // 16-byte chunks of the warp (16 channels each)
        unsigned b[4];
        const int ch = kPairs == 2 ? warp * 2 + (lane >> 4) : warp;
        ldsm4_t(v_u + unsigned(t * Cfg::kRowBytes + chunk_at<E4M3, DP, true>(t, ch) * 16), b);
#pragma unroll
        for (int n = 0; n < kPairs; n++) {
          const unsigned lo = b[2 * n], hi = b[2 * n + 1];  // tokens 0-7 and 8-15 of the step
          mma16816<true>(o[2 * n], pa, e4m3x2_to_f16x2(__byte_perm(lo, 0, 0x4420)), e4m3x2_to_f16x2(__byte_perm(hi, 0, 0x4420)));
          mma16816<true>(o[2 * n + 1], pa, e4m3x2_to_f16x2(__byte_perm(lo, 0, 0x4431)), e4m3x2_to_f16x2(__byte_perm(hi, 0, 0x4431)));
        }
      }
    }

    const bool last = cur.tile + 1 == cur.n_tiles;
    if (last || i + 1 == n_my) {  // the (sequence, head) or the run ends: store
      const bool whole = last && first_tile == 0;
#pragma unroll
      for (int h = 0; h < 2; h++) {
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
        if ((lane & 3) == 0) wsum[warp][r0 + 8 * h] = l[h];
      }
      __syncthreads();
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
            p.part_ml[(slot * kRows + r) * 2] = m[h], p.part_ml[(slot * kRows + r) * 2 + 1] = sum;
          } else if (p.a.lse) {
            p.a.lse[int64_t(cur.b) * p.a.H + h0 + r] = sum == 0.f ? -INFINITY : (m[h] + log2f(sum)) * kLn2;
          }
        }
      }
      fresh = true;
    }
    cursor_next(p, cur);
  }
  cp_wait<0>();
}

// Adds up, for each (sequence, head) that several runs share, the parts in the order of the runs.
template <int DP>
__global__ void __launch_bounds__(kThreadsD) join_kernel(const __grid_constant__ DecodeLaunch p) {
  __shared__ int red[kWarps + 2];
  pdl_launch_dependents();
  pdl_wait();
  const int b = int(blockIdx.x) / p.heads, head = int(blockIdx.x) - b * p.heads;
  const int n_tiles = (view_of(p, b).len + kTile - 1) / kTile;
  // tiles in front of sequence b and in total
  int total = 0, before = 0;
  {
    const int n = p.c.n_seqs, t = threadIdx.x;
    int all = 0, front = 0;
    for (int x = t; x < n; x += kThreadsD) {
      const int k = tiles_of(p, x);
      all += k;
      if (x < b) front += k;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o), front += __shfl_xor_sync(0xffffffffu, front, o);
    __shared__ int fr[kWarps];
    if ((t & 31) == 0) red[t >> 5] = all, fr[t >> 5] = front;
    __syncthreads();
    for (int w = 0; w < kWarps; w++) total += red[w], before += fr[w];
  }
  if (n_tiles == 0) return;
  const int per = (total + p.ctas - 1) / p.ctas;
  const int s0 = before + head * n_tiles, c0 = s0 / per, c1 = (s0 + n_tiles - 1) / per;
  if (c0 == c1) return;  // one run had all of it and has written the output
  const int g = head / p.blocks, blk = head % p.blocks;
  const int rows = min(kRows, p.group - blk * kRows), h0 = g * p.group + blk * kRows, D = p.c.D;
  // slot of run c: the segment it starts in, unless the segment starts inside the run (or with it)
  auto slot = [&](int c) { return 2 * int64_t(c) + (c == c0 ? 1 : 0); };
  for (int i = threadIdx.x; i < rows * D; i += kThreadsD) {
    const int r = i / D, d = i - r * D;
    float mx = -INFINITY;
    for (int c = c0; c <= c1; c++) mx = fmaxf(mx, p.part_ml[(slot(c) * kRows + r) * 2]);
    const float base = mx == -INFINITY ? 0.f : mx;
    float sum = 0.f, o = 0.f;
    for (int c = c0; c <= c1; c++) {
      const int64_t at = slot(c) * kRows + r;
      const float f = ex2_approx(p.part_ml[at * 2] - base);
      sum = fmaf(p.part_ml[at * 2 + 1], f, sum);
      o = fmaf(p.part_o[at * DP + d], f, o);
    }
    const float res = sum > 0.f || sum != sum ? o / sum : 0.f;
    p.a.out[(int64_t(b) * p.a.H + h0 + r) * D + d] = mxk_bf16(pack_bf16(res, 0.f) & 0xffffu);
    if (d == 0 && p.a.lse) p.a.lse[int64_t(b) * p.a.H + h0 + r] = sum == 0.f ? -INFINITY : (mx + log2f(sum)) * kLn2;
  }
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
  const int64_t most = int64_t(p.c.n_seqs) * p.heads * ceil_div(int64_t(p.c.max_pages) * p.c.page_size, kTile);
  if (p.ctas > most) p.ctas = int(most < 1 ? 1 : most);
  p.part_o = static_cast<float*>(p.a.workspace);
  p.part_ml = p.part_o + int64_t(2) * p.ctas * kRows * DP;
  launch_pdl(decode_kernel<E4M3, DP>, dim3(unsigned(p.ctas)), dim3(kThreadsD), DecodeCfg<E4M3, DP>::kSmem, s, p);
  if (int rc = after_launch(name)) return rc;
  launch_pdl(join_kernel<DP>, dim3(unsigned(p.c.n_seqs * p.heads)), dim3(kThreadsD), 0, s, p);
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
  const int64_t tiles = int64_t(cache->n_seqs) * p.heads * (ceil_div(int64_t(cache->max_pages) * cache->page_size, kTile) + 1);
  if (tiles >= (int64_t(1) << 30)) return fail(MXK_ERR_TOO_LARGE, "%s: n_seqs * heads * tokens too large (%lld tiles)", name, (long long)tiles);
  p.scale2 = a.scale * kLog2e;
  p.err = device_error_word();
  const cudaStream_t s = as_stream(stream);
  if (cache->D <= 64) return cache->type == MXK_KV_E4M3 ? launch_decode<true, 64>(name, p, s) : launch_decode<false, 64>(name, p, s);
  return cache->type == MXK_KV_E4M3 ? launch_decode<true, 128>(name, p, s) : launch_decode<false, 128>(name, p, s);
}

}  // extern "C"
