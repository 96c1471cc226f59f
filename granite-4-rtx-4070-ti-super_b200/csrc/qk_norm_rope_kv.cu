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
// Doubles are short: 80 of them a key element's lane and head, no division. The code itself is found in f32 (value
// times the scale's reciprocal, off by 2^-22 of it at most) wherever that is further from a border than 2^-14;
// where it is not, the sign of fma(-(code +- 1/2), scale, |x|) decides, which an fma gives exactly.
//
#include "g4_host.h"
#include "g4_math.cuh"

#include "../../include/granite4_b200.h"

#include <algorithm>

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
constexpr float kNearBorder = 0.5f - 1.0f / 16384.0f;

// |x| against the borders of code c: the code itself.
__device__ __forceinline__ float settle(float c, float x, float s) {
  if (fmaf(-(c + 0.5f), s, x) >= 0.0f) return c + 1.0f;
  return c > 0.0f && fmaf(-(c - 0.5f), s, x) < 0.0f ? c - 1.0f : c;
}
__device__ __forceinline__ float settle(float c, double x, float s) {
  if (fma(-static_cast<double>(c + 0.5f), static_cast<double>(s), x) >= 0.0) return c + 1.0f;
  return c > 0.0f && fma(-static_cast<double>(c - 0.5f), static_cast<double>(s), x) < 0.0 ? c - 1.0f : c;
}

// A code under a scale whose reciprocal, or the fma's difference, may lie outside of f32 (or that is zero).
__device__ __noinline__ float code_by_division(double x, float s, float top) {
  if (!(s > 0.0f)) return 0.0f;
  const double ax = fabs(x);
  const float c = settle(fminf(rintf(static_cast<float>(ax / static_cast<double>(s))), top), ax, s);
  return x < 0.0 ? -c : c;
}

// Codes of a lane's values x (xf: the same in f32) under scale s, as the words of the pool: 4 bits, code + 8, or 8.
template <int BITS, typename T>
__device__ __forceinline__ uint2 encode8(const T (&x)[8], const float (&xf)[8], float s, bool plain, float inv) {
  // adding 1.5 2^23 (and the 8) leaves the integer in the low bits of the sum
  constexpr float kMagic = 12582912.0f + (BITS == 4 ? 8.0f : 0.0f);
  float z[8], far = plain ? 0.0f : 1.0f;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float t = xf[e] * inv;
    z[e] = t + kMagic;
    far = fmaxf(far, fabsf(t - (z[e] - kMagic)));
  }
  if (!(far < kNearBorder)) {
    if (plain) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float code = settle(fabsf(z[e] - kMagic), x[e] < T(0) ? -x[e] : x[e], s);
        z[e] = (x[e] < T(0) ? -code : code) + kMagic;
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) z[e] = code_by_division(x[e], s, BITS == 4 ? 7.0f : 127.0f) + kMagic;
    }
  }
  // sum of (z - magic's bits) 2^(BITS e): the magic's bits are taken out of the sum
  uint2 w = make_uint2(0u, 0u);
  if (BITS == 4) {
#pragma unroll
    for (int e = 0; e < 8; ++e) w.x += __float_as_uint(z[e]) << (4 * e);
    w.x -= 0x4b400000u * 0x11111111u;
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      w.x |= (__float_as_uint(z[e]) & 0xffu) << (8 * e);
      w.y |= (__float_as_uint(z[4 + e]) & 0xffu) << (8 * e);
    }
  }
  return w;
}

__device__ __forceinline__ void copy16_async(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(dst))), "l"(src)
               : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// d / 16 lanes own a head: lane j has columns [8j, 8j + 8) of both halves, i.e. both sides of its eight
// rotation pairs, so the rotation needs no exchange and the head's sums are log2(d / 16) shuffles. An item is the heads
// that a warp takes at once (four of 128); the items of all rows are one line, of which every warp has an equal run:
// query, key and value heads cost 1 : 3 : 1.5, so runs, not strides, keep the warps even, and a row's tables are
// loaded once. A lane's 32 bytes of the next three items are on their way by asynchronous copies into slots of
// its own, so nothing is synchronised. What bounds the kernel is memory, 22 KB a row of 48 heads in and out.
constexpr int kQkDepth = 4, kQkCtas = 6;
template <int D, int BITS>
__global__ void __launch_bounds__(kQkThreads, kQkCtas) qk_norm_rope_kv_kernel(const QkNormParams p, int per_row, int items) {
  pdl_begin();
  constexpr int kLanes = D / 16, kHeads = 32 / kLanes, kTop = BITS == 4 ? 7 : 127;
  __shared__ uint4 s_raw[kQkDepth][2][kQkThreads];
  const int lane = threadIdx.x & 31, g = lane / kLanes, j = lane % kLanes;
  const unsigned mask = ((1u << kLanes) - 1u) << (lane & ~(kLanes - 1));
  const int heads = p.Hq + 2 * p.Hk;
  const unsigned warps = gridDim.x * (kQkThreads / 32), warp = blockIdx.x * (kQkThreads / 32) + (threadIdx.x >> 5);
  const int begin = static_cast<int>(static_cast<unsigned long long>(warp) * items / warps);
  const int end = static_cast<int>(static_cast<unsigned long long>(warp + 1) * items / warps);
  if (begin >= end) return;
  // (row, part) of the item to work on and of the item to fetch
  int row = begin / per_row, part = begin - row * per_row, f_row = row, f_part = part;
  auto fetch = [&](int item) {
    if (item < end) {
      const int head = f_part * kHeads + g;
      if (head < heads) {
        const uint4* src = reinterpret_cast<const uint4*>(p.qkv + (static_cast<size_t>(f_row) * heads + head) * D) + j;
        copy16_async(&s_raw[item % kQkDepth][0][threadIdx.x], src);
        copy16_async(&s_raw[item % kQkDepth][1][threadIdx.x], src + kLanes);
      }
      if (++f_part == per_row) f_part = 0, ++f_row;
    }
    copies_commit();
  };
#pragma unroll
  for (int i = 0; i < kQkDepth - 1; ++i) fetch(begin + i);
  int next_pos = __ldg(p.pos_rows + row), next_kv = __ldg(p.kv_rows + row), pos = 0, kv_row = 0;
  float c[8], s[8];
  bool fresh = true, sound = false;
#pragma unroll 1
  for (int item = begin; item < end; ++item) {
    if (fresh) {
      pos = next_pos, kv_row = next_kv;
      if (row + 1 < p.rows) next_pos = __ldg(p.pos_rows + row + 1), next_kv = __ldg(p.kv_rows + row + 1);
      // a bad index skips the row instead of touching memory outside the tables or the pool
      sound = pos >= 0 && pos < p.max_pos && kv_row >= 0 && kv_row < p.stride;
      if (sound) {
#pragma unroll
        for (int e = 0; e < 8; e += 4) {
          const float4 cv = __ldg(reinterpret_cast<const float4*>(p.cos_tbl + static_cast<size_t>(pos) * (D / 2) + 8 * j + e));
          const float4 sv = __ldg(reinterpret_cast<const float4*>(p.sin_tbl + static_cast<size_t>(pos) * (D / 2) + 8 * j + e));
          c[e] = cv.x, c[e + 1] = cv.y, c[e + 2] = cv.z, c[e + 3] = cv.w;
          s[e] = sv.x, s[e + 1] = sv.y, s[e + 2] = sv.z, s[e + 3] = sv.w;
        }
      }
    }
    fetch(item + kQkDepth - 1);
    copies_wait<kQkDepth - 1>();
    const int head = part * kHeads + g, r = row;
    fresh = ++part == per_row;
    if (fresh) part = 0, ++row;
    if (!sound || head >= heads) continue;
    float lo[8], hi[8];
    unpack8(s_raw[item % kQkDepth][0][threadIdx.x], lo);
    unpack8(s_raw[item % kQkDepth][1][threadIdx.x], hi);
    const bool is_q = head < p.Hq, is_k = !is_q && head < p.Hq + p.Hk;
    const uint16_t* wt = is_q ? p.wq : p.wk;
    if (is_q) {
      if (wt != nullptr) {
        float wl[8], wh[8];
        unpack8(__ldg(reinterpret_cast<const uint4*>(wt) + j), wl);
        unpack8(__ldg(reinterpret_cast<const uint4*>(wt) + kLanes + j), wh);
        float ss = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) ss += lo[e] * lo[e] + hi[e] * hi[e];
#pragma unroll
        for (int o = 1; o < kLanes; o <<= 1) ss += __shfl_xor_sync(mask, ss, o);
        const float rn = rsqrtf(ss * (1.0f / D) + p.eps);
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
    const int hkv = is_k ? head - p.Hq : head - p.Hq - p.Hk;
    const size_t srow = static_cast<size_t>(hkv) * p.stride + kv_row;
    float sc;
    uint2 cl, ch;
    if (is_k) {
      double dl[8], dh[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) dl[e] = lo[e], dh[e] = hi[e];
      if (wt != nullptr) {
        double ss = 0.0;
#pragma unroll
        for (int e = 0; e < 8; ++e) ss += dl[e] * dl[e] + dh[e] * dh[e];
#pragma unroll
        for (int o = 1; o < kLanes; o <<= 1) ss += __shfl_xor_sync(mask, ss, o);
        const double rn = 1.0 / sqrt(ss * (1.0 / D) + static_cast<double>(p.eps));
        float wl[8], wh[8];
        unpack8(__ldg(reinterpret_cast<const uint4*>(wt) + j), wl);
        unpack8(__ldg(reinterpret_cast<const uint4*>(wt) + kLanes + j), wh);
#pragma unroll
        for (int e = 0; e < 8; ++e) dl[e] *= rn * wl[e], dh[e] *= rn * wh[e];
      }
      double amax = 0.0;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const double a = dl[e], b = dh[e];
        dl[e] = a * c[e] - b * s[e], dh[e] = b * c[e] + a * s[e];
        const double x = fabs(dl[e]), y = fabs(dh[e]);
        amax = x > amax ? x : amax;
        amax = y > amax ? y : amax;
        lo[e] = static_cast<float>(dl[e]), hi[e] = static_cast<float>(dh[e]);
      }
#pragma unroll
      for (int o = 1; o < kLanes; o <<= 1) {
        const double x = __shfl_xor_sync(mask, amax, o);
        amax = x > amax ? x : amax;
      }
      sc = static_cast<float>(amax / kTop);
      const bool plain = sc > 1e-30f;
      const float inv = plain ? 1.0f / sc : 0.0f;
      cl = encode8<BITS>(dl, lo, sc, plain, inv), ch = encode8<BITS>(dh, hi, sc, plain, inv);
    } else {
      float amax = 0.0f;
#pragma unroll
      for (int e = 0; e < 8; ++e) amax = fmaxf(amax, fmaxf(fabsf(lo[e]), fabsf(hi[e])));
#pragma unroll
      for (int o = 1; o < kLanes; o <<= 1) amax = fmaxf(amax, __shfl_xor_sync(mask, amax, o));
      sc = __fdiv_rn(amax, static_cast<float>(kTop));  // eight significant bits over 7 or 127: never half way between floats
      const bool plain = sc > 1e-30f;
      const float inv = plain ? 1.0f / sc : 0.0f;
      cl = encode8<BITS>(lo, lo, sc, plain, inv), ch = encode8<BITS>(hi, hi, sc, plain, inv);
    }
    if (j == 0) (is_k ? p.k_scale : p.v_scale)[srow] = sc;
    uint8_t* cache = (is_k ? p.cache_k : p.cache_v) + srow * (D * BITS / 8);
    if (BITS == 4) {
      reinterpret_cast<uint32_t*>(cache)[j] = cl.x;
      reinterpret_cast<uint32_t*>(cache)[kLanes + j] = ch.x;
    } else {
      reinterpret_cast<uint2*>(cache)[j] = cl;
      reinterpret_cast<uint2*>(cache)[kLanes + j] = ch;
    }
  }
}

template <int D, int BITS>
int launch_qk_norm(const char* fn, const QkNormParams& p) {
  constexpr int heads_per_item = 32 / (D / 16), warps = kQkThreads / 32;
  const int per_row = (p.Hq + 2 * p.Hk + heads_per_item - 1) / heads_per_item;
  const long long items = static_cast<long long>(p.rows) * per_row;
  if (items > INT_MAX - kQkDepth) return fail(fn, "too many rows");
  const long long grid = std::min((items + warps - 1) / warps, static_cast<long long>(kQkCtas) * sm_count());
  G4_LAUNCH_PDL(fn, (qk_norm_rope_kv_kernel<D, BITS>), dim3(static_cast<unsigned>(grid)), dim3(kQkThreads), 0, current_stream(), p,
                per_row, static_cast<int>(items));
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
