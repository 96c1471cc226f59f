// Per-head RMSNorm of Q and K, RoPE, and K / V quantised into the paged pool, in one pass over the
// token rows of a layer's qkv.
//
// For every token row and every head x of d values (halves a = x[i], b = x[i + d/2]):
//   n     = x * r * w,  r = 1 / sqrt(mean(x^2) + eps)        (no weight given: n = x; V: n = x, no rotation)
//   rot   = (a c - b s, b c + a s) with c, s = cos / sin of the row's position
//   q_rot = bf16(rot)
//   K, V  = codes: scale = f32(max |rot| / top), code = sign * floor(|rot| / scale + 1/2), top = 7 | 127
// The 4-bit pool keeps code + 8 in a nibble, the even dim in the low half of its byte, [Hk][stride][d / 2];
// the 8-bit pool is the one rope_kv.cu writes, [Hk][stride][d]. Both have f32 scales [Hk][stride].
//
// The one rounding of a code is its own: K is normed and rotated in double from its bf16 values and the f32
// tables, so that a code does not depend on the order in which a kernel rounds its way there. What is left
// of a double between the value and the border of two codes is 1e-15 of the scale.
#include "g4_host.h"
#include "g4_math.cuh"

#include "../../include/granite4_b200.h"

namespace g4 {
namespace {

struct QkNormParams {
  const uint16_t* qkv;  // [rows][(Hq + 2 Hk) d]
  const uint16_t* wq;   // [d] or NULL
  const uint16_t* wk;   // [d] or NULL
  float eps;
  const float* cos_tbl;  // [max_pos][d / 2]
  const float* sin_tbl;
  const int* pos_rows;
  const int* kv_rows;
  uint16_t* q_rot;
  uint8_t* cache_k;
  uint8_t* cache_v;
  float* k_scale;
  float* v_scale;
  int rows, Hq, Hk, max_pos;
  long long stride;
};

constexpr int kQkThreads = 128;

// sign * floor(|x| / s + 1/2) of a value whose quotient by the scale is at most top (but for a rounding)
template <int TOP>
__device__ __forceinline__ int code_of(double x, double s) {
  const double t = floor(fabs(x) / s + 0.5);
  const int m = static_cast<int>(fmin(t, static_cast<double>(TOP)));
  return x < 0.0 ? -m : m;
}

// d / 16 lanes own a head: lane j has columns [8j, 8j + 8) of both halves, i.e. both sides of its eight
// rotation pairs, so the rotation needs no exchange and the head's sums are log2(d / 16) shuffles.
template <int D, int BITS>
__global__ void __launch_bounds__(kQkThreads) qk_norm_rope_kv_kernel(const QkNormParams p) {
  pdl_begin();
  constexpr int kLanes = D / 16, kHeads = kQkThreads / kLanes, kTop = BITS == 4 ? 7 : 127;
  const int g = threadIdx.x / kLanes + blockIdx.y * kHeads, step = gridDim.y * kHeads, j = threadIdx.x % kLanes;
  const unsigned mask = ((1u << kLanes) - 1u) << (threadIdx.x & 31 & ~(kLanes - 1));
  const int heads = p.Hq + 2 * p.Hk, r = blockIdx.x;
  const int pos = __ldg(p.pos_rows + r), kv_row = __ldg(p.kv_rows + r);
  // a bad index skips the row instead of touching memory outside the tables or the pool
  if (pos < 0 || pos >= p.max_pos || kv_row < 0 || kv_row >= p.stride) return;
  float c[8], s[8];
#pragma unroll
  for (int e = 0; e < 8; e += 4) {
    const float4 cv = __ldg(reinterpret_cast<const float4*>(p.cos_tbl + static_cast<size_t>(pos) * (D / 2) + 8 * j + e));
    const float4 sv = __ldg(reinterpret_cast<const float4*>(p.sin_tbl + static_cast<size_t>(pos) * (D / 2) + 8 * j + e));
    c[e] = cv.x, c[e + 1] = cv.y, c[e + 2] = cv.z, c[e + 3] = cv.w;
    s[e] = sv.x, s[e + 1] = sv.y, s[e + 2] = sv.z, s[e + 3] = sv.w;
  }
  for (int head = g; head < heads; head += step) {
    const uint4* src = reinterpret_cast<const uint4*>(p.qkv + (static_cast<size_t>(r) * heads + head) * D);
    float lo[8], hi[8], wl[8], wh[8];
    unpack8(ld_stream(src + j), lo);
    unpack8(ld_stream(src + kLanes + j), hi);
    const bool is_q = head < p.Hq, is_k = !is_q && head < p.Hq + p.Hk;
    const uint16_t* w = is_q ? p.wq : p.wk;
    if (w != nullptr) {
      unpack8(__ldg(reinterpret_cast<const uint4*>(w) + j), wl);
      unpack8(__ldg(reinterpret_cast<const uint4*>(w) + kLanes + j), wh);
    }
    if (is_q) {
      if (w != nullptr) {
        float ss = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) ss += lo[e] * lo[e] + hi[e] * hi[e];
#pragma unroll
        for (int o = 1; o < kLanes; o <<= 1) ss += __shfl_xor_sync(mask, ss, o);
        const float rn = 1.0f / sqrtf(ss / D + p.eps);
#pragma unroll
        for (int e = 0; e < 8; ++e) lo[e] *= rn * wl[e], hi[e] *= rn * wh[e];
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float a = lo[e], b = hi[e];
        lo[e] = a * c[e] - b * s[e], hi[e] = b * c[e] + a * s[e];
      }
      uint4* dst = reinterpret_cast<uint4*>(p.q_rot + (static_cast<size_t>(r) * p.Hq + head) * D);
      st_stream(dst + j, pack8(lo));
      st_stream(dst + kLanes + j, pack8(hi));
      continue;
    }
    double dl[8], dh[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) dl[e] = lo[e], dh[e] = hi[e];
    if (is_k) {
      if (w != nullptr) {
        double ss = 0.0;
#pragma unroll
        for (int e = 0; e < 8; ++e) ss += dl[e] * dl[e] + dh[e] * dh[e];
#pragma unroll
        for (int o = 1; o < kLanes; o <<= 1) ss += __shfl_xor_sync(mask, ss, o);
        const double rn = 1.0 / sqrt(ss / D + static_cast<double>(p.eps));
#pragma unroll
        for (int e = 0; e < 8; ++e) dl[e] = dl[e] * rn * wl[e], dh[e] = dh[e] * rn * wh[e];
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const double a = dl[e], b = dh[e];
        dl[e] = a * c[e] - b * s[e], dh[e] = b * c[e] + a * s[e];
      }
    }
    double amax = 0.0;
#pragma unroll
    for (int e = 0; e < 8; ++e) amax = fmax(amax, fmax(fabs(dl[e]), fabs(dh[e])));
#pragma unroll
    for (int o = 1; o < kLanes; o <<= 1) amax = fmax(amax, __shfl_xor_sync(mask, amax, o));
    const float sc = static_cast<float>(amax / kTop);
    const int hkv = is_k ? head - p.Hq : head - p.Hq - p.Hk;
    const size_t srow = static_cast<size_t>(hkv) * p.stride + kv_row;
    if (j == 0) (is_k ? p.k_scale : p.v_scale)[srow] = sc;
    uint8_t* cache = (is_k ? p.cache_k : p.cache_v) + srow * (D * BITS / 8);
    int cl[8], ch[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      cl[e] = sc > 0.0f ? code_of<kTop>(dl[e], sc) : 0;
      ch[e] = sc > 0.0f ? code_of<kTop>(dh[e], sc) : 0;
    }
    if (BITS == 4) {
      uint32_t a = 0, b = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) a |= static_cast<uint32_t>(cl[e] + 8) << (4 * e), b |= static_cast<uint32_t>(ch[e] + 8) << (4 * e);
      reinterpret_cast<uint32_t*>(cache)[j] = a;
      reinterpret_cast<uint32_t*>(cache)[kLanes + j] = b;
    } else {
      uint32_t a[2] = {0, 0}, b[2] = {0, 0};
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        a[e >> 2] |= static_cast<uint32_t>(cl[e] & 0xff) << (8 * (e & 3));
        b[e >> 2] |= static_cast<uint32_t>(ch[e] & 0xff) << (8 * (e & 3));
      }
      reinterpret_cast<uint2*>(cache)[j] = make_uint2(a[0], a[1]);
      reinterpret_cast<uint2*>(cache)[kLanes + j] = make_uint2(b[0], b[1]);
    }
  }
}

template <int D, int BITS>
int launch_qk_norm(const char* fn, const QkNormParams& p) {
  constexpr int heads_per_cta = kQkThreads / (D / 16);
  const int heads = p.Hq + 2 * p.Hk;
  const unsigned parts = p.rows <= 16 ? static_cast<unsigned>((heads + heads_per_cta - 1) / heads_per_cta) : 1u;
  G4_LAUNCH_PDL(fn, (qk_norm_rope_kv_kernel<D, BITS>), dim3(static_cast<unsigned>(p.rows), parts), dim3(kQkThreads), 0,
                current_stream(), p);
  return 0;
}

}  // namespace
}  // namespace g4

extern "C" int granite4_kernel_qk_norm_rope_kv_paged(const uint16_t* d_qkv, const uint16_t* d_q_norm,
                                                     const uint16_t* d_k_norm, float eps, const float* d_cos,
                                                     const float* d_sin, const int* d_pos_rows, const int* d_kv_rows,
                                                     int rows, int Hq, int Hk, int d, int stride, int max_pos, int bits,
                                                     uint16_t* d_q_rot, void* d_cache_k, void* d_cache_v,
                                                     float* d_k_scale, float* d_v_scale) {
  const char* fn = "granite4_kernel_qk_norm_rope_kv_paged";
  if (d_qkv == nullptr || d_cos == nullptr || d_sin == nullptr || d_pos_rows == nullptr || d_kv_rows == nullptr ||
      d_q_rot == nullptr || d_cache_k == nullptr || d_cache_v == nullptr || d_k_scale == nullptr ||
      d_v_scale == nullptr || rows <= 0 || Hq <= 0 || Hk <= 0 || Hq > 65535 || Hk > 65535 || stride <= 0 || max_pos <= 0 ||
      !std::isfinite(eps) || eps <= 0.0f)
    return g4::fail(fn, "invalid arguments");
  if ((d != 64 && d != 128) || (bits != 4 && bits != 8)) return g4::fail(fn, "head dims of 64 and 128, pools of 4 and 8 bits");
  if (!g4::aligned16(d_qkv) || !g4::aligned16(d_q_norm) || !g4::aligned16(d_k_norm) || !g4::aligned16(d_cos) ||
      !g4::aligned16(d_sin) || !g4::aligned16(d_q_rot) || !g4::aligned16(d_cache_k) || !g4::aligned16(d_cache_v))
    return g4::fail(fn, "pointers must be 16-byte aligned");
  g4::QkNormParams p{};
  p.qkv = d_qkv, p.wq = d_q_norm, p.wk = d_k_norm, p.eps = eps, p.cos_tbl = d_cos, p.sin_tbl = d_sin;
  p.pos_rows = d_pos_rows, p.kv_rows = d_kv_rows, p.q_rot = d_q_rot;
  p.cache_k = static_cast<uint8_t*>(d_cache_k), p.cache_v = static_cast<uint8_t*>(d_cache_v);
  p.k_scale = d_k_scale, p.v_scale = d_v_scale;
  p.rows = rows, p.Hq = Hq, p.Hk = Hk, p.max_pos = max_pos, p.stride = stride;
  if (d == 128) return bits == 4 ? g4::launch_qk_norm<128, 4>(fn, p) : g4::launch_qk_norm<128, 8>(fn, p);
  return bits == 4 ? g4::launch_qk_norm<64, 4>(fn, p) : g4::launch_qk_norm<64, 8>(fn, p);
}
