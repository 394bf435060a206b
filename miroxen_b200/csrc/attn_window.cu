// attn_window: attention of a packed batch of sequences with a sliding window and first tokens that stay visible.
//
//   s_ij = scale * q_i . k_j over the keys j that row i sees,  m_i = max_j s_ij,
//   out_i = sum_j exp(s_ij - m_i) v_j / sum_j exp(s_ij - m_i),   lse_i = m_i + ln sum_j exp(s_ij - m_i)
//
// Row i of a sequence of Lq rows and Lk keys stands at p = i + Lk - Lq and sees j <= p + right (right >= 0) that are
// j >= p - left (left >= 0) or j < sinks.
#include "common.cuh"
#include "kv_cache.cuh"

namespace mxk {
namespace {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct AttnLaunch {
  MxkAttnArgs a;
  int group;     // query heads per key head
  float scale2;  // scale * log2(e)
  int* err;
};

// First row of sequence b, held inside [0, rows] and not before `least` whatever the array holds.
__device__ __forceinline__ int cu_at(const int32_t* cu, int b, int64_t rows, int least, int* err) {
  const int v = cu[b];
  if (v < least || v > rows) {
    if (err) atomicExch(err, kErrBadIndex);
    return v < least ? least : int(rows);
  }
  return v;
}

// Keys that a row at position p of a sequence of nk keys sees: [0, first) and [lo, hi).
struct Seen {
  int first, lo, hi;
};
__device__ __forceinline__ Seen seen_by(const MxkAttnArgs& a, int64_t p, int nk) {
  Seen s{0, 0, nk};
  if (a.right >= 0 && p + a.right + 1 < nk) s.hi = p + a.right + 1 < 0 ? 0 : int(p + a.right + 1);
  if (a.left >= 0 && p - a.left > 0) s.lo = p - a.left > nk ? nk : int(p - a.left);
  s.first = a.sinks < s.lo ? int(a.sinks) : s.lo;
  if (s.first > s.hi) s.first = s.hi;
  if (s.lo > s.hi) s.lo = s.hi;
  return s;
}

// One row and head by one warp, 32 keys at a time: a lane takes a key's product with q, then the warp adds the keys'
// values, each lane holding channels 2 lane, 2 lane + 1, + 64.  `qs`: the warp's 128 floats of shared memory.
__device__ void row_attention(const AttnLaunch& L, int64_t row, int h, int64_t k0, int64_t p, int nk, float* qs) {
  const MxkAttnArgs& a = L.a;
  const int lane = threadIdx.x & 31, D = a.D, g = h / L.group;
  const Seen seen = seen_by(a, p, nk);
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

__global__ void __launch_bounds__(256) attn_rows_kernel(const __grid_constant__ AttnLaunch L) {
  __shared__ float qs[8][MXK_ATTN_MAX_HEAD_DIM];
  const MxkAttnArgs& a = L.a;
  pdl_launch_dependents();
  pdl_wait();
  const int warp = threadIdx.x >> 5;
  const int64_t row = int64_t(blockIdx.x) * 8 + warp;
  if (a.cu_q && blockIdx.x == 0 && blockIdx.y == 0)  // every end, those that no row looks at too
    for (int b = threadIdx.x; b < a.n_seqs; b += blockDim.x) {
      cu_at(a.cu_q, b + 1, a.q_rows, cu_at(a.cu_q, b, a.q_rows, 0, L.err), L.err);
      cu_at(a.cu_k, b + 1, a.k_rows, cu_at(a.cu_k, b, a.k_rows, 0, L.err), L.err);
    }
  if (row >= a.q_rows) return;
  int q0 = 0, q1 = int(a.q_rows), k0 = 0, k1 = int(a.k_rows);
  if (a.cu_q) {
    // the sequence that the row lies in: the first whose end lies behind it
    int b = 0, lo = 0, hi = a.n_seqs;
    while (lo < hi) {
      const int mid = (lo + hi) / 2;
      if (a.cu_q[mid + 1] > row) hi = mid;
      else lo = mid + 1;
    }
    b = lo;
    if (b >= a.n_seqs || a.cu_q[b] > row) return;  // a row of no sequence
    q0 = cu_at(a.cu_q, b, a.q_rows, 0, L.err), q1 = cu_at(a.cu_q, b + 1, a.q_rows, q0, L.err);
    k0 = cu_at(a.cu_k, b, a.k_rows, 0, L.err), k1 = cu_at(a.cu_k, b + 1, a.k_rows, k0, L.err);
  }
  const int nk = k1 - k0;
  row_attention(L, row, int(blockIdx.y), k0, row - q0 + nk - (q1 - q0), nk, qs[warp]);
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
  if (a.H <= 0 || a.Hkv <= 0 || a.H % a.Hkv != 0 || a.H > 65535)
    return fail(MXK_ERR_INVALID_ARG, "%s: H=%d must be a positive multiple of Hkv=%d", name, a.H, a.Hkv);
  if (a.D < 8 || a.D > MXK_ATTN_MAX_HEAD_DIM || a.D % 8 != 0)
    return fail(MXK_ERR_INVALID_ARG, "%s: head dimension %d must be a multiple of 8 and at most %d", name, a.D, MXK_ATTN_MAX_HEAD_DIM);
  if ((a.cu_q == nullptr) != (a.cu_k == nullptr) || (!a.cu_q && a.n_seqs != 1))
    return fail(MXK_ERR_INVALID_ARG, "%s: cu_q and cu_k come together, and several sequences need them (n_seqs=%d)", name, a.n_seqs);
  if (a.q_rows >= (int64_t(1) << 31) || a.k_rows >= (int64_t(1) << 31))
    return fail(MXK_ERR_TOO_LARGE, "%s: q_rows=%lld k_rows=%lld", name, (long long)a.q_rows, (long long)a.k_rows);
  if (a.q_stride % 8 != 0 || a.k_stride % 8 != 0 || a.v_stride % 8 != 0 || a.out_stride % 8 != 0)
    return fail(MXK_ERR_INVALID_ARG, "%s: strides must be multiples of 8", name);
  if ((a.q_rows > 1 && (a.q_stride < int64_t(a.H) * a.D || a.out_stride < int64_t(a.H) * a.D)) ||
      (a.k_rows > 1 && (a.k_stride < int64_t(a.Hkv) * a.D || a.v_stride < int64_t(a.Hkv) * a.D)))
    return fail(MXK_ERR_INVALID_ARG, "%s: row strides smaller than a row's heads", name);
  if (!aligned(a.q, 16) || !aligned(a.k, 16) || !aligned(a.v, 16) || !aligned(a.out, 16))
    return fail(MXK_ERR_INVALID_ARG, "%s: q, k, v and out must be 16-byte aligned", name);
  if (a.sinks < 0) return fail(MXK_ERR_INVALID_ARG, "%s: sinks=%lld", name, (long long)a.sinks);
  if (!(a.scale > 0.f) || a.scale > 3.0e38f) return fail(MXK_ERR_INVALID_ARG, "%s: scale must be positive and finite", name);
  L.group = a.H / a.Hkv;
  L.scale2 = a.scale * kLog2e;
  L.err = device_error_word();
  launch_pdl(attn_rows_kernel, dim3(unsigned(ceil_div(a.q_rows, 8)), unsigned(a.H)), dim3(256), 0, as_stream(stream), L);
  return after_launch(name);
}
