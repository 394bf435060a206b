// qkv_norm_rope_append: per-head RMSNorm + rotary embedding of a step's q and k, q to a contiguous array, k and v into
// the pages of a key/value cache, one launch.
//
// For row t, head h of q (or k):  x = in[t, h];  with a norm weight w:  x = x * rsqrt(mean(x^2) + eps) * w;  the first
// `rot` channels turn by the row's angles, (a, b) -> (a c - b s, a s + b c), pairs (2i, 2i + 1) or (i, i + rot / 2);
// nothing is rounded before the store (one rounding to bf16, or of x / scale to e4m3 with saturation).  v is stored as
// it is (bf16) or as v / scale (e4m3).
//
// The op only streams: 2 bytes per channel in, 2 or 1 out, some ten flops between.  So its form is that of the other
// streaming ops here: one tile per CTA and as many CTAs as that takes.  A tile is one row's heads [h0, h0 + heads per
// CTA) of q | k | v; D / 8 lanes (rounded up to a power of two) hold a head, eight channels - one 128-bit access - per
// lane, and each lane has the vectors of two heads in flight.  The row's sequence, position and page are looked up by
// every lane (the same addresses: one L1 transaction each) while its vectors are on the way.
#include "common.cuh"
#include "kv_cache.cuh"

namespace mxk {
namespace {

constexpr int kHeadsPerLane = 2;     // independent vectors a lane has in flight
constexpr int kAppendThreads = 256;  // at most

struct AppendLaunch {
  MxkAppendArgs a;
  MxkKvCache c;
  int heads;          // H + 2 Hkv
  int chunks;         // CTAs per row
  int heads_per_cta;  // of those
  float inv_d;
  int* err;
};

__device__ __forceinline__ uint2 pack8_e4m3(const float (&f)[8], float scale) {
  unsigned w[2] = {0u, 0u};
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const __nv_fp8x2_storage_t p = __nv_cvt_float2_to_fp8x2(make_float2(__fdiv_rn(f[2 * i], scale), __fdiv_rn(f[2 * i + 1], scale)), __NV_SATFINITE, __NV_E4M3);
    w[i >> 1] |= unsigned(p) << (16 * (i & 1));
  }
  return make_uint2(w[0], w[1]);
}

// LPH lanes hold a head.  VEC: the lane's table entries (and, in half mode, its pair partners) are whole aligned vectors
// of another lane; otherwise every channel looks its own pair up.
template <int LPH, bool E4M3, bool VEC>
__global__ void __launch_bounds__(kAppendThreads) append_kernel(const __grid_constant__ AppendLaunch p) {
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
    if (VEC && inter) {
      const float4 cc = *reinterpret_cast<const float4*>(cr + 4 * l), ss = *reinterpret_cast<const float4*>(sr + 4 * l);
      cs[0] = cs[1] = cc.x, cs[2] = cs[3] = cc.y, cs[4] = cs[5] = cc.z, cs[6] = cs[7] = cc.w;
      sn[0] = -ss.x, sn[1] = ss.x, sn[2] = -ss.y, sn[3] = ss.y, sn[4] = -ss.z, sn[5] = ss.z, sn[6] = -ss.w, sn[7] = ss.w;
    } else if (VEC) {
      const bool first = 8 * l < half;
      const int i0 = first ? 8 * l : 8 * l - half;
      const float4 c0 = *reinterpret_cast<const float4*>(cr + i0), c1 = *reinterpret_cast<const float4*>(cr + i0 + 4);
      const float4 s0 = *reinterpret_cast<const float4*>(sr + i0), s1 = *reinterpret_cast<const float4*>(sr + i0 + 4);
      const float f = first ? -1.f : 1.f;
      cs[0] = c0.x, cs[1] = c0.y, cs[2] = c0.z, cs[3] = c0.w, cs[4] = c1.x, cs[5] = c1.y, cs[6] = c1.z, cs[7] = c1.w;
      sn[0] = f * s0.x, sn[1] = f * s0.y, sn[2] = f * s0.z, sn[3] = f * s0.w, sn[4] = f * s1.x, sn[5] = f * s1.y, sn[6] = f * s1.z, sn[7] = f * s1.w;
    } else {
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
  }
  const int lane = int(threadIdx.x) & 31, base = lane & ~(LPH - 1);
  const int partner = base + (!rotates || inter ? l : 8 * l < half ? l + (half >> 3) : l - (half >> 3));

  __shared__ float xch[VEC ? 1 : kAppendThreads * 8];
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
      if (VEC) {
        const float4 w0 = *reinterpret_cast<const float4*>(w + 8 * l), w1 = *reinterpret_cast<const float4*>(w + 8 * l + 4);
        v[0] *= rstd * w0.x, v[1] *= rstd * w0.y, v[2] *= rstd * w0.z, v[3] *= rstd * w0.w;
        v[4] *= rstd * w1.x, v[5] *= rstd * w1.y, v[6] *= rstd * w1.z, v[7] *= rstd * w1.w;
      } else {
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] *= rstd * w[8 * l + i];
      }
    }
    if (half > 0) {  // the same for the whole launch
      float o[8];
      if (inter) {
#pragma unroll
        for (int i = 0; i < 8; i++) o[i] = v[i ^ 1];
      } else if (VEC) {
#pragma unroll
        for (int i = 0; i < 8; i++) o[i] = __shfl_sync(0xffffffffu, v[i], partner);
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
          if (VEC ? rotates : 8 * l + i < 2 * half) v[i] = fmaf(o[i], sn[i], v[i] * cs[i]);
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
int launch_append(const char* name, AppendLaunch& p, bool vec, cudaStream_t s) {
  // whole heads per CTA, an even share of the row's heads for each
  const int most = kAppendThreads / LPH * kHeadsPerLane;
  p.chunks = int(ceil_div(p.heads, most));
  p.heads_per_cta = int(ceil_div(p.heads, p.chunks));
  const int threads = int(ceil_div(ceil_div(p.heads_per_cta, kHeadsPerLane) * LPH, 32)) * 32;
  const int64_t ctas = p.a.T * p.chunks;
  if (ctas >= (int64_t(1) << 31)) return fail(MXK_ERR_TOO_LARGE, "%s: T=%lld rows of %d heads", name, (long long)p.a.T, p.heads);
  launch_pdl(vec ? append_kernel<LPH, E4M3, true> : append_kernel<LPH, E4M3, false>, dim3(unsigned(ctas)), dim3(unsigned(threads)), 0, s, p);
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
  p.heads = a.H + 2 * cache->Hkv;
  p.inv_d = 1.f / float(cache->D);
  p.err = device_error_word();
  const int half = rope ? a.rot / 2 : 0;
  // The vector form needs table rows, weights and pair partners in whole aligned vectors: half % 8 == 0 puts a half-mode
  // lane's partners into one other lane, half % 4 == 0 is enough for adjacent pairs.
  const bool vec = half % (a.mode == MXK_ROPE_HALF ? 8 : 4) == 0 && aligned(a.cos, 16) && aligned(a.sin, 16) && aligned(a.q_norm_w, 16) &&
                   aligned(a.k_norm_w, 16);
  const cudaStream_t s = as_stream(stream);
  if (cache->D <= 64)
    return cache->type == MXK_KV_E4M3 ? launch_append<8, true>(name, p, vec, s) : launch_append<8, false>(name, p, vec, s);
  return cache->type == MXK_KV_E4M3 ? launch_append<16, true>(name, p, vec, s) : launch_append<16, false>(name, p, vec, s);
}
