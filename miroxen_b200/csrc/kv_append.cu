// qkv_norm_rope_append: per-head RMSNorm + rotary embedding of a step's q and k, q to a contiguous array, k and v into
// the pages of a key/value cache, one launch.
//
// For row t, head h of q (or k):  x = in[t, h];  with a norm weight w:  x = x * rsqrt(mean(x^2) + eps) * w;  the first
// `rot` channels turn by the row's angles, (a, b) -> (a c - b s, a s + b c), pairs (2i, 2i + 1) or (i, i + rot / 2);
// nothing is rounded before the store (one rounding to bf16, or of x / scale to e4m3 with saturation).  v is stored as
// it is (bf16) or as v / scale (e4m3).
//
// The op only streams: 2 bytes per channel in, 2 or 1 out, some ten flops between; what keeps it from the memory's rate is
// instructions and the chain sequence, position -> page, table row that stands in front of a row's work.  So
// (append_kernel) a head is held by D / 16 lanes, two vectors of eight channels each, chosen so that both members of a
// rotated pair sit in one lane; a group of lanes stays with one row, whose angles it keeps in registers, and walks heads
// g, g + groups, ... of q, k and v, the next two heads' vectors on their way while it works on the last two.  Few rows get
// many groups each, so that a single token's heads all go at once.  Head dimensions and rotations that do not split
// into such vectors take append_any_kernel.
//
// Measured: 33272 rows, 40 + 40 + 40 heads of 128 from a packed projection, bf16 pages and k_out, 424 us = 5660 GB/s (first
// form, a vector per lane and a CTA per 32 heads: 765 us); 8704 rows of 24 + 24 + 24 heads 72.5 us; 250 rows of 32 + 8 + 8 heads
// into e4m3 pages 5.1 us, one row 2.9 us.  Two heads per lane in flight and four CTAs per SM: one head takes 504 us on the
// largest, five CTAs (96 registers, spills) 501 us.  Into e4m3 pages the division counts: 8704 rows of 24 + 24 + 24 heads of 128
// without k_out 72 us against 67 into bf16 pages.  append_any_kernel, the same rows with heads of 72: 174 us; of 80, which append_kernel
// takes, 60.
#include "common.cuh"
#include "kv_cache.cuh"

namespace mxk {
namespace {

constexpr int kHeadsPerLane = 2;     // independent heads a lane has in flight
constexpr int kAppendThreads = 128;
constexpr int kAnyThreads = 256;     // of append_any_kernel, at most

struct AppendLaunch {
  MxkAppendArgs a;
  MxkKvCache c;
  int heads;          // H + 2 Hkv
  int groups;         // append_kernel: groups of lanes per row, a power of two
  int chunks;         // append_any_kernel: CTAs per row
  int heads_per_cta;  // of those
  float inv_d;
  int* err;
};

// Eight values / scale as e4m3.  A product with 1 / scale, which is rounded itself, would put quotients that lie exactly between two
// codes (scales of few significant bits have many) on the wrong side.  So the quotient's remainder, which one fma gives
// exactly, is divided as well (Markstein, IBM J. Res. Dev. 34, 1990: correctly rounded where the reciprocal is).  Both sides are
// taken times a power of two that brings the scale into [1, 4), where nothing on the way leaves the normal numbers but quotients that
// are the code 0.  Saturating, infinite and NaN quotients stay as they are; a zero keeps its sign.  8704 rows of 3 x 24 heads of 128:
// 71.5 us, with __fdiv_rn 86, with the reciprocal alone 65.
__device__ __forceinline__ uint2 pack8_e4m3(const float* f, float scale) {
  const float up = __uint_as_float(0x7f000000u - min(__float_as_uint(scale) & 0x7f800000u, 0x7e800000u));
  const float m = scale * up, inv = __frcp_rn(m);
  unsigned w[2] = {0u, 0u};
#pragma unroll
  for (int i = 0; i < 4; i++) {
    float q[2];
#pragma unroll
    for (int e = 0; e < 2; e++) {
      const float x = f[2 * i + e] * up, y = x * inv, rest = fmaf(y, m, -x);
      q[e] = fabsf(y) < 512.f ? fmaf(rest, -inv, y) : y;
    }
    w[i >> 1] |= unsigned(__nv_cvt_float2_to_fp8x2(make_float2(q[0], q[1]), __NV_SATFINITE, __NV_E4M3)) << (16 * (i & 1));
  }
  return make_uint2(w[0], w[1]);
}

__device__ __forceinline__ void load8(const float* p, float* o) {
  const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
  o[0] = a.x, o[1] = a.y, o[2] = a.z, o[3] = a.w, o[4] = b.x, o[5] = b.y, o[6] = b.z, o[7] = b.w;
}
__device__ __forceinline__ void unpack8_at(const uint4& v, float* o) {
  float f[8];
  unpack8(v, f);
#pragma unroll
  for (int i = 0; i < 8; i++) o[i] = f[i];
}
__device__ __forceinline__ uint4 pack8_at(const float* f) {
  return make_uint4(pack_bf16(f[0], f[1]), pack_bf16(f[2], f[3]), pack_bf16(f[4], f[5]), pack_bf16(f[6], f[7]));
}

// LPH >= D / 16 lanes hold a head; lane l its vectors (of eight channels) va and vb.
template <int LPH, bool E4M3, bool INTER>
__global__ void __launch_bounds__(kAppendThreads, 4) append_kernel(const __grid_constant__ AppendLaunch p) {
  using elem = typename KvElem<E4M3>::type;
  constexpr int U = kHeadsPerLane, kGroups = kAppendThreads / LPH;
  const MxkAppendArgs& a = p.a;
  const MxkKvCache& c = p.c;
  pdl_launch_dependents();
  pdl_wait();
  const int D = c.D, H = a.H, Hkv = c.Hkv, G = p.groups;
  const int unit = int(blockIdx.x) * kGroups + int(threadIdx.x) / LPH, l = int(threadIdx.x) % LPH;
  const int row = unit / G, g = unit - row * G;
  if (__all_sync(0xffffffffu, row >= a.T)) return;
  const bool on = row < a.T && 16 * l < D;
  const int half = a.mode == MXK_ROPE_NONE ? 0 : a.rot >> 1;
  // Vectors of lane l.  Pairs (i, i + half): the first half / 8 lanes hold partners, the others two vectors that do not turn;
  // adjacent pairs lie within a vector.
  const int hv = half >> 3;
  const int va = INTER ? l : l < hv ? l : 2 * l, vb = INTER ? l + D / 16 : l < hv ? l + hv : 2 * l + 1;

  // Turns of the group: heads of q, then k, then v; each kind starts with the group after the one that the last kind's heads
  // ended with, so that a row with as many groups as heads does all of them in its first turn.
  auto first = [&](int kind) { return kind == 0 ? g : kind == 1 ? (g - H) & (G - 1) : (g - H - Hkv) & (G - 1); };
  auto turns = [&](int kind) {
    const int n = (kind == 0 ? H : Hkv) - first(kind);
    return n <= 0 ? 0 : (n + G * U - 1) / (G * U);
  };
  const int t1 = turns(0), t2 = t1 + turns(1), t3 = t2 + turns(2);
  // (turn counts of the groups of a warp differ by one at most; the exchanges below are made by all of them)
  int last = t3;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) last = max(last, __shfl_xor_sync(0xffffffffu, last, o));
  auto kind_of = [&](int t) { return t < t1 ? 0 : t < t2 ? 1 : 2; };
  auto load = [&](int t, uint4 (&raw)[U][2]) {
    const int kind = kind_of(t), i0 = first(kind) + (t - (kind == 0 ? 0 : kind == 1 ? t1 : t2)) * G * U;
    const int n = kind == 0 ? H : Hkv;
    const mxk_bf16* src = kind == 0 ? a.q + int64_t(row) * a.q_stride : kind == 1 ? a.k + int64_t(row) * a.k_stride : a.v + int64_t(row) * a.v_stride;
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int h = i0 + u * G;
      raw[u][0] = raw[u][1] = make_uint4(0u, 0u, 0u, 0u);
      if (on && t < t3 && h < n) {
        const mxk_bf16* s = src + int64_t(h) * D;
        raw[u][0] = ld_stream(reinterpret_cast<const uint4*>(s + 8 * va));
        raw[u][1] = ld_stream(reinterpret_cast<const uint4*>(s + 8 * vb));
      }
    }
  };
  uint4 raw[U][2];
  load(0, raw);

  // where the row goes, and its angles
  const int row_c = min(row, int(a.T) - 1);
  const int seq = a.seq_ids ? a.seq_ids[row_c] : row_c, pos = a.positions[row_c];
  const int trow = half > 0 ? (a.rope_rows ? a.rope_rows[row_c] : pos) : 0;
  const int64_t at = kv_token_offset(c, seq, pos);
  const bool table_ok = half == 0 || (trow >= 0 && trow < a.table_rows);
  const bool bad = seq >= 0 && (at < 0 || !table_ok);
  const bool live = on && seq >= 0 && !bad;  // a negative sequence: a padding row
  if (bad && on && l == 0 && p.err) atomicExch(p.err, kErrBadIndex);
  float cs[8], sn[8];
#pragma unroll
  for (int i = 0; i < 8; i++) cs[i] = 1.f, sn[i] = 0.f;
  const bool turn_a = live && (INTER ? 8 * va < 2 * half : l < hv), turn_b = live && INTER && 8 * vb < 2 * half;
  {
    const float* cr = a.cos + int64_t(trow) * half;
    const float* sr = a.sin + int64_t(trow) * half;
    if (INTER) {  // cs[0..3] of va's pairs, cs[4..7] of vb's
      if (turn_a) {
        const float4 x = *reinterpret_cast<const float4*>(cr + 4 * va), y = *reinterpret_cast<const float4*>(sr + 4 * va);
        cs[0] = x.x, cs[1] = x.y, cs[2] = x.z, cs[3] = x.w, sn[0] = y.x, sn[1] = y.y, sn[2] = y.z, sn[3] = y.w;
      }
      if (turn_b) {
        const float4 x = *reinterpret_cast<const float4*>(cr + 4 * vb), y = *reinterpret_cast<const float4*>(sr + 4 * vb);
        cs[4] = x.x, cs[5] = x.y, cs[6] = x.z, cs[7] = x.w, sn[4] = y.x, sn[5] = y.y, sn[6] = y.z, sn[7] = y.w;
      }
    } else if (turn_a) {
      load8(cr + 8 * l, cs), load8(sr + 8 * l, sn);
    }
  }

  float wt[16];
  int wt_kind = 2;
#pragma unroll 1
  for (int t = 0; t < last; t++) {
    uint4 next[U][2];
    load(t + 1, next);
    const int kind = kind_of(t), n = kind == 0 ? H : Hkv;
    const int i0 = first(kind) + (t - (kind == 0 ? 0 : kind == 1 ? t1 : t2)) * G * U;
    const float* w = kind == 0 ? a.q_norm_w : kind == 1 ? a.k_norm_w : nullptr;
    if (w && on && kind != wt_kind) load8(w + 8 * va, wt), load8(w + 8 * vb, wt + 8), wt_kind = kind;
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int h = i0 + u * G;
      float v[16];
      unpack8_at(raw[u][0], v), unpack8_at(raw[u][1], v + 8);
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < 16; i++) ss = fmaf(v[i], v[i], ss);
      ss = group_sum<LPH>(ss);
      const bool mine = live && t < t3 && h < n;
      if (!mine) continue;
      if (kind < 2) {
        if (w) {
          const float rstd = rsqrtf(fmaf(ss, p.inv_d, a.eps));
#pragma unroll
          for (int i = 0; i < 16; i++) v[i] *= rstd * wt[i];
        }
        if (INTER) {  // vectors that do not turn have cosine 1 and sine 0
#pragma unroll
          for (int i = 0; i < 8; i++) {
            const float x = v[2 * i], y = v[2 * i + 1];
            if (i < 4 ? turn_a : turn_b) v[2 * i] = x * cs[i] - y * sn[i], v[2 * i + 1] = fmaf(x, sn[i], y * cs[i]);
          }
        } else if (turn_a) {
#pragma unroll
          for (int i = 0; i < 8; i++) {
            const float x = v[i], y = v[8 + i];
            v[i] = x * cs[i] - y * sn[i], v[8 + i] = fmaf(x, sn[i], y * cs[i]);
          }
        }
      }
      if (kind == 0) {
        mxk_bf16* dst = a.q_out + (int64_t(row) * H + h) * D;
        st_stream(reinterpret_cast<uint4*>(dst + 8 * va), pack8_at(v));
        st_stream(reinterpret_cast<uint4*>(dst + 8 * vb), pack8_at(v + 8));
        continue;
      }
      elem* dst = static_cast<elem*>(kind == 1 ? c.k : c.v) + at + int64_t(h) * c.head_stride;
      if (E4M3) {
        const float* sc = kind == 1 ? c.k_scale : c.v_scale;
        const float scale = sc ? sc[h] : 1.f;
        *reinterpret_cast<uint2*>(dst + 8 * va) = pack8_e4m3(v, scale);
        *reinterpret_cast<uint2*>(dst + 8 * vb) = pack8_e4m3(v + 8, scale);
      } else {
        *reinterpret_cast<uint4*>(dst + 8 * va) = kind == 2 ? raw[u][0] : pack8_at(v);
        *reinterpret_cast<uint4*>(dst + 8 * vb) = kind == 2 ? raw[u][1] : pack8_at(v + 8);
      }
      if (kind == 1 && a.k_out) {
        mxk_bf16* ko = a.k_out + (int64_t(row) * Hkv + h) * D;
        *reinterpret_cast<uint4*>(ko + 8 * va) = pack8_at(v);
        *reinterpret_cast<uint4*>(ko + 8 * vb) = pack8_at(v + 8);
      }
    }
#pragma unroll
    for (int u = 0; u < U; u++) raw[u][0] = next[u][0], raw[u][1] = next[u][1];
  }
}

// Any D that is a multiple of 8 and any even rotation: LPH >= D / 8 lanes hold a head, each channel looks its own pair up, its
// partner through shared memory; a CTA has one row's heads [chunk * heads_per_cta, + heads_per_cta).
template <int LPH, bool E4M3>
__global__ void __launch_bounds__(kAnyThreads) append_any_kernel(const __grid_constant__ AppendLaunch p) {
  using elem = typename KvElem<E4M3>::type;
  const MxkAppendArgs& a = p.a;
  const MxkKvCache& c = p.c;
  pdl_launch_dependents();
  pdl_wait();
  const int row = int(blockIdx.x) / p.chunks, chunk = int(blockIdx.x) - row * p.chunks;
  const int groups = int(blockDim.x) / LPH, group = int(threadIdx.x) / LPH, l = int(threadIdx.x) % LPH;
  const int D = c.D, H = a.H, Hkv = c.Hkv;
  const bool lane_on = 8 * l < D;
  const int h_end = min(p.heads, (chunk + 1) * p.heads_per_cta);

  // the vectors of this lane's heads
  uint4 raw[kHeadsPerLane];
  int head[kHeadsPerLane];
#pragma unroll
  for (int u = 0; u < kHeadsPerLane; u++) {
    const int h = head[u] = chunk * p.heads_per_cta + group + u * groups;
    raw[u] = make_uint4(0u, 0u, 0u, 0u);
    if (lane_on && h < h_end) {
      const mxk_bf16* src = h < H ? a.q + int64_t(row) * a.q_stride + int64_t(h) * D
                            : h < H + Hkv ? a.k + int64_t(row) * a.k_stride + int64_t(h - H) * D
                                          : a.v + int64_t(row) * a.v_stride + int64_t(h - H - Hkv) * D;
      raw[u] = ld_stream(reinterpret_cast<const uint4*>(src + 8 * l));
    }
  }

  // where the row goes
  const int seq = a.seq_ids ? a.seq_ids[row] : row;
  if (seq < 0) return;  // a padding row (the whole CTA)
  const int pos = a.positions[row];
  const int half = a.mode == MXK_ROPE_NONE ? 0 : a.rot >> 1;
  const int trow = half > 0 ? (a.rope_rows ? a.rope_rows[row] : pos) : 0;
  const int64_t at = kv_token_offset(c, seq, pos);
  if (at < 0 || (half > 0 && (trow < 0 || trow >= a.table_rows))) {
    if (threadIdx.x == 0 && p.err) atomicExch(p.err, kErrBadIndex);
    return;
  }

  // this lane's cosines and signed sines: channel i of the lane becomes v[i] * cs[i] + partner * sn[i]
  const bool inter = a.mode == MXK_ROPE_INTERLEAVED;
  const bool rotates = 8 * l < 2 * half;
  float cs[8], sn[8];
#pragma unroll
  for (int i = 0; i < 8; i++) cs[i] = 1.f, sn[i] = 0.f;
  if (rotates) {
    const float* cr = a.cos + int64_t(trow) * half;
    const float* sr = a.sin + int64_t(trow) * half;
#pragma unroll
      for (int i = 0; i < 8; i++) {
        const int ch = 8 * l + i;
        if (ch < 2 * half) {
          const bool first = inter ? (ch & 1) == 0 : ch < half;
          const int pair = inter ? ch >> 1 : first ? ch : ch - half;
          cs[i] = cr[pair], sn[i] = first ? -sr[pair] : sr[pair];
        }
      }
  }
  __shared__ float xch[kAnyThreads * 8];
#pragma unroll
  for (int u = 0; u < kHeadsPerLane; u++) {
    const int h = head[u];
    const bool on = lane_on && h < h_end, is_q = h < H, is_v = h >= H + Hkv;
    float v[8];
    unpack8(raw[u], v);
    const float* w = is_q ? a.q_norm_w : is_v ? nullptr : a.k_norm_w;
    float ss = 0.f;  // every lane of the warp takes part in the exchanges
#pragma unroll
    for (int i = 0; i < 8; i++) ss = fmaf(v[i], v[i], ss);
    ss = group_sum<LPH>(ss);
    if (w && on) {
      const float rstd = rsqrtf(fmaf(ss, p.inv_d, a.eps));
#pragma unroll
      for (int i = 0; i < 8; i++) v[i] *= rstd * w[8 * l + i];
    }
    if (half > 0) {  // the same for the whole launch
      float o[8];
      if (inter) {
#pragma unroll
        for (int i = 0; i < 8; i++) o[i] = v[i ^ 1];
      } else {
        float* mine = xch + (threadIdx.x - l) * 8;  // the head's channels
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 8; i++) mine[8 * l + i] = v[i];
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 8; i++) {
          const int ch = 8 * l + i;
          o[i] = ch < half ? mine[ch + half] : ch < 2 * half ? mine[ch - half] : 0.f;
        }
      }
      if (!is_v) {
#pragma unroll
        for (int i = 0; i < 8; i++)
          if (8 * l + i < 2 * half) v[i] = fmaf(o[i], sn[i], v[i] * cs[i]);
      }
    }
    if (!on) continue;
    if (is_q) {
      st_stream(reinterpret_cast<uint4*>(a.q_out + (int64_t(row) * H + h) * D + 8 * l), pack8(v));
      continue;
    }
    const int g = is_v ? h - H - Hkv : h - H;
    elem* dst = static_cast<elem*>(is_v ? c.v : c.k) + at + int64_t(g) * c.head_stride + 8 * l;
    if (E4M3) {
      const float* sc = is_v ? c.v_scale : c.k_scale;
      *reinterpret_cast<uint2*>(dst) = pack8_e4m3(v, sc ? sc[g] : 1.f);
    } else {
      *reinterpret_cast<uint4*>(dst) = is_v ? raw[u] : pack8(v);
    }
    if (!is_v && a.k_out) *reinterpret_cast<uint4*>(a.k_out + (int64_t(row) * Hkv + g) * D + 8 * l) = pack8(v);
  }
}

template <int LPH, bool E4M3>
int launch_any(const char* name, AppendLaunch& p, cudaStream_t s) {
  // whole heads per CTA, an even share of the row's heads for each
  const int most = kAnyThreads / LPH * kHeadsPerLane;
  p.chunks = int(ceil_div(p.heads, most));
  p.heads_per_cta = int(ceil_div(p.heads, p.chunks));
  const int threads = int(ceil_div(ceil_div(p.heads_per_cta, kHeadsPerLane) * LPH, 32)) * 32;
  const int64_t ctas = p.a.T * p.chunks;
  if (ctas >= (int64_t(1) << 31)) return fail(MXK_ERR_TOO_LARGE, "%s: T=%lld rows of %d heads", name, (long long)p.a.T, p.heads);
  launch_pdl(append_any_kernel<LPH, E4M3>, dim3(unsigned(ctas)), dim3(unsigned(threads)), 0, s, p);
  return after_launch(name);
}

template <int LPH, bool E4M3>
int launch_append(const char* name, AppendLaunch& p, cudaStream_t s) {
  // Groups per row: as many as the GPU holds at once (four CTAs an SM), at least four, at most one per head.
  const int64_t fill = int64_t(sm_count()) * 4 * kAppendThreads / LPH / p.a.T;
  p.groups = 4;
  while (2 * p.groups <= fill && p.groups < p.heads) p.groups *= 2;
  const int64_t ctas = ceil_div(p.a.T * p.groups, kAppendThreads / LPH);
  if (ctas >= (int64_t(1) << 31) / (kAppendThreads / LPH)) return fail(MXK_ERR_TOO_LARGE, "%s: T=%lld rows of %d heads", name, (long long)p.a.T, p.heads);
  launch_pdl(p.a.mode == MXK_ROPE_INTERLEAVED ? append_kernel<LPH, E4M3, true> : append_kernel<LPH, E4M3, false>, dim3(unsigned(ctas)), dim3(kAppendThreads), 0, s,
             p);
  return after_launch(name);
}

}  // namespace
}  // namespace mxk

using namespace mxk;

extern "C" int mxk_qkv_norm_rope_append(const MxkAppendArgs* args, const MxkKvCache* cache, mxk_stream_t stream) {
  const char* name = "qkv_norm_rope_append";
  if (!args) return fail(MXK_ERR_INVALID_ARG, "%s: null args", name);
  if (args->T <= 0) return MXK_OK;
  if (int rc = check_cache(name, cache)) return rc;
  if (int rc = check_cache_pointers(name, cache)) return rc;
  AppendLaunch p{};
  p.a = *args, p.c = *cache;
  const MxkAppendArgs& a = p.a;
  if (!a.q || !a.k || !a.v || !a.q_out || !a.positions) return fail(MXK_ERR_INVALID_ARG, "%s: null q, k, v, q_out or positions", name);
  if (a.H <= 0) return fail(MXK_ERR_INVALID_ARG, "%s: H=%d", name, a.H);
  if (a.T >= (int64_t(1) << 31)) return fail(MXK_ERR_TOO_LARGE, "%s: T=%lld", name, (long long)a.T);
  if (a.q_stride % 8 != 0 || a.k_stride % 8 != 0 || a.v_stride % 8 != 0 || a.q_stride < 0 || a.k_stride < 0 || a.v_stride < 0)
    return fail(MXK_ERR_INVALID_ARG, "%s: strides must be multiples of 8", name);
  if (!aligned(a.q, 16) || !aligned(a.k, 16) || !aligned(a.v, 16) || !aligned(a.q_out, 16) || !aligned(a.k_out, 16))
    return fail(MXK_ERR_INVALID_ARG, "%s: q, k, v, q_out and k_out must be 16-byte aligned", name);
  if (a.mode != MXK_ROPE_NONE && a.mode != MXK_ROPE_INTERLEAVED && a.mode != MXK_ROPE_HALF)
    return fail(MXK_ERR_INVALID_ARG, "%s: unknown rope mode %d", name, a.mode);
  const bool rope = a.mode != MXK_ROPE_NONE;
  if (rope && (a.rot < 0 || a.rot > cache->D || a.rot % 2 != 0))
    return fail(MXK_ERR_INVALID_ARG, "%s: rot=%d must be even and <= D=%d", name, a.rot, cache->D);
  if (rope && a.rot > 0 && (!a.cos || !a.sin)) return fail(MXK_ERR_INVALID_ARG, "%s: rotary mode needs cos and sin tables", name);
  const int64_t heads = int64_t(a.H) + 2 * int64_t(cache->Hkv);
  if (heads >= (int64_t(1) << 30)) return fail(MXK_ERR_TOO_LARGE, "%s: H=%d and Hkv=%d heads", name, a.H, cache->Hkv);
  p.heads = int(heads);
  p.inv_d = 1.f / float(cache->D);
  p.err = device_error_word();
  const int half = rope ? a.rot / 2 : 0;
  // append_kernel needs a head in pairs of vectors (D % 16 == 0), and table rows, weights and pair partners in whole aligned
  // vectors: half % 8 == 0 puts the partners of a vector into one other vector, half % 4 == 0 is enough for adjacent pairs.
  const bool vec = cache->D % 16 == 0 && half % (a.mode == MXK_ROPE_HALF ? 8 : 4) == 0 && aligned(a.cos, 16) && aligned(a.sin, 16) &&
                   aligned(a.q_norm_w, 16) && aligned(a.k_norm_w, 16);
  const cudaStream_t s = as_stream(stream);
  const bool e = cache->type == MXK_KV_E4M3, small = cache->D <= 64;
  if (vec) return small ? (e ? launch_append<4, true>(name, p, s) : launch_append<4, false>(name, p, s)) : (e ? launch_append<8, true>(name, p, s) : launch_append<8, false>(name, p, s));
  return small ? (e ? launch_any<8, true>(name, p, s) : launch_any<8, false>(name, p, s)) : (e ? launch_any<16, true>(name, p, s) : launch_any<16, false>(name, p, s));
}
