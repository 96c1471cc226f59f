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
// The one rounding of a code is its own: a code is the one that exact arithmetic on the bf16 inputs and the f32 tables
// gives (in double where it matters: 1e-15 of the scale), so that it does not depend on the order in which a kernel
// rounds its way there. Doubles are few: with y = rot(x w) (products of two bf16 are exact in f32) rot(n) = r y, the
// scale is f32(r max |y| / top) and the quotients are y (r / scale). r is a double, y is f32, off by at most 2^-22 of the
// head's max |y|. In double are only y of the pairs that may hold the maximum (those within 2^-19 of it: hardly ever
// more than one a head), and y of a pair with a quotient so near to the border of two codes that f32 may be wrong, where
// the sign of fma(-(code +- 1/2), scale, |r y|) decides, which an fma gives exactly. A head whose y may leave f32 on the way
// (max |y| not in [2^-100, 2^126)) is all doubles. A key or value head that holds an infinity or a NaN has codes 0 and a scale
// that is not finite, so that whoever reads it gets NaN.
// V: value and amax have eight significant bits each, so a quotient top v / amax is a border exactly or further from it
// than 1 / (2 top 255) >= 2^-16 of itself. Exact ones (v = amax / 2 is one in every third head) fall to the side that the
// rounding of the scale pushes them to: the scale's reciprocal, moved by 2^-19 of itself to that side, decides all.
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
// An f32 quotient further than this from its code may belong to the next: y and r / scale are off by 5.5 2^-24 of the
// quotients' range, 2.3e-6 (4 bits) and 4.2e-5.
template <int BITS>
constexpr float kNearBorder = 0.5f - (BITS == 4 ? 1.0f / 131072.0f : 1.0f / 16384.0f);

// |x| against the borders of code c: the code itself.
__device__ __forceinline__ float settle(float c, double x, float s) {
  if (fma(-static_cast<double>(c + 0.5f), static_cast<double>(s), x) >= 0.0) return c + 1.0f;
  return c > 0.0f && fma(-static_cast<double>(c - 0.5f), static_cast<double>(s), x) < 0.0 ? c - 1.0f : c;
}

// A code under a scale whose reciprocal, or the fma's difference, may lie outside of f32 (or that is zero or not finite).
__device__ __noinline__ float code_by_division(double x, float s, float top) {
  if (!(s > 0.0f && s < INFINITY)) return 0.0f;
  const double ax = fabs(x);
  const float c = fminf(settle(fminf(rintf(static_cast<float>(ax / static_cast<double>(s))), top), ax, s), top);  // (a subnormal scale may be short)
  return x < 0.0 ? -c : c;
}

// The larger, NaN where either is.
__device__ __forceinline__ float max_or_nan(float x, float y) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(x), "f"(y));
  return r;
}
// Float bits of the largest |y| of a key head for which f32 does: [2^-100, 2^126), the products of weights and tables
// included (what overflows shows as an infinity or NaN, what underflows is 2^-149 of 2^-100).
constexpr unsigned kLeastY = (127u - 100u) << 23, kPastY = (127u + 126u) << 23;

// Eight quotients x inv rounded to the nearest integer, as z = code + magic in f32: 1.5 2^23 (and the 8 of a nibble)
// leaves the integer in the low bits of the sum. Returns the largest distance |quotient - code|.
template <int BITS>
constexpr float kMagic = 12582912.0f + (BITS == 4 ? 8.0f : 0.0f);
template <int BITS>
__device__ __forceinline__ float round8(const float (&x)[8], float inv, float (&z)[8]) {
  const F32x2 inv2 = f32x2(inv, inv), magic2 = f32x2(kMagic<BITS>, kMagic<BITS>), one2 = f32x2(1.0f, 1.0f);
  const F32x2 less2 = f32x2(-kMagic<BITS>, -kMagic<BITS>), minus2 = f32x2(-1.0f, -1.0f);
  float far = 0.0f;
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    const F32x2 t = mul2(f32x2(x[e], x[e + 1]), inv2), zz = fma2(t, one2, magic2);
    const F32x2 off = fma2(fma2(zz, one2, less2), minus2, t);
    float u, v;
    f32x2_split(off, u, v);
    f32x2_split(zz, z[e], z[e + 1]);
    far = fmaxf(far, fmaxf(fabsf(u), fabsf(v)));
  }
  return far;
}
// z of a key settled against its exact value x.
template <int BITS>
__device__ __forceinline__ float settled(float z, double x, float s, bool plain) {
  if (!plain) return code_by_division(x, s, BITS == 4 ? 7.0f : 127.0f) + kMagic<BITS>;
  const float c = settle(fabsf(z - kMagic<BITS>), fabs(x), s);
  return (x < 0.0 ? -c : c) + kMagic<BITS>;
}
// The words of the pool: 4 bits, code + 8, or 8.
template <int BITS>
__device__ __forceinline__ uint2 pack_codes(const float (&z)[8]) {
  uint2 w = make_uint2(0u, 0u);
  if (BITS == 4) {  // sum of (bits of z - bits of 1.5 2^23) 16^e
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

// y of pair e of a lane in double, from where its inputs lie. Out of line: the kernel's instructions have to stay in the cache.
__device__ __noinline__ double2 key_pair(const uint16_t* a, const uint16_t* b, const uint16_t* wa, const uint16_t* wb,
                                         const float* c, const float* s, int e) {
  float x = bf16_to_f32(a[e]), y = bf16_to_f32(b[e]);
  if (wa != nullptr) x *= bf16_to_f32(__ldg(wa + e)), y *= bf16_to_f32(__ldg(wb + e));
  const double cd = __ldg(c + e), sd = __ldg(s + e);
  return make_double2(x * cd - y * sd, y * cd + x * sd);
}

// A lane's part of a key head whose y may leave f32: everything in double, codes by division. (Doubles in key_pair instead:
// 16384 rows 1.3 us more, for the registers of its callers.)
struct FarHead {
  uint2 lo, hi;
  float scale;
};
template <int D, int BITS>
__device__ __noinline__ FarHead far_key_head(const uint16_t* a, const uint16_t* b, const uint16_t* wa, const uint16_t* wb,
                                             const float* c, const float* s, double rn, unsigned mask) {
  constexpr float kTop = BITS == 4 ? 7.0f : 127.0f;
  const auto pair = [&](int e) {
    const double x = static_cast<double>(bf16_to_f32(a[e])) * (wa != nullptr ? bf16_to_f32(__ldg(wa + e)) : 1.0f);
    const double y = static_cast<double>(bf16_to_f32(b[e])) * (wa != nullptr ? bf16_to_f32(__ldg(wb + e)) : 1.0f);
    const double cd = __ldg(c + e), sd = __ldg(s + e);
    return make_double2((x * cd - y * sd) * rn, (y * cd + x * sd) * rn);
  };
  double amax = 0.0;
  bool numbers = true;
#pragma unroll 1
  for (int e = 0; e < 8; ++e) {
    const double2 y = pair(e);
    amax = fmax(amax, fmax(fabs(y.x), fabs(y.y)));
    numbers = numbers && fabs(y.x) < INFINITY && fabs(y.y) < INFINITY;
  }
  numbers = __all_sync(mask, numbers);
#pragma unroll
  for (int o = 1; o < D / 16; o <<= 1) amax = fmax(amax, __shfl_xor_sync(mask, amax, o));
  FarHead h;
  h.scale = numbers ? static_cast<float>(amax * (1.0 / kTop)) : __int_as_float(0x7fc00000);
  float lo[8], hi[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const double2 y = pair(e);
    lo[e] = code_by_division(y.x, h.scale, kTop) + kMagic<BITS>, hi[e] = code_by_division(y.y, h.scale, kTop) + kMagic<BITS>;
  }
  h.lo = pack_codes<BITS>(lo), h.hi = pack_codes<BITS>(hi);
  return h;
}

__device__ __forceinline__ void copy16_async(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// d / 16 lanes own a head: lane j has columns [8j, 8j + 8) of both halves, i.e. both sides of its eight
// rotation pairs, so the rotation needs no exchange and the head's sums are log2(d / 16) shuffles. An item is the heads
// that a warp takes at once (four of 128), of q or of k and v; the items of all rows are one line, of which every warp has
// an equal run: the kinds cost 1 : 3 : 2, so runs, not strides, keep the warps even, and what depends on the row alone
// (the products of norm weights and tables for q) is worked out once. A lane's 32 bytes of the next three items are on
// their way by asynchronous copies into slots of its own, so nothing is synchronised. Arithmetic is on pairs of f32 where
// it can be. What bounds the kernel is memory, 22 KB a row of 48 heads in and out, and close behind it the issue slots:
// 16384 such rows with norms into the 4-bit pool take 66 - 69 us on the GPU, 5.3 TB/s, 2400 warp instructions a row; six CTAs
// per SM leave 80 registers a thread, of which 28 - 32 bytes are spilled. (With every key in double 79 us, 3080; rows unrolled in
// the code 210 us, waiting for instructions.)
constexpr int kQkDepth = 4, kQkCtas = 6;
// WHOLE: query heads and key / value heads fill their items, so the items of all rows lie one behind the other in qkv.
template <int D, int BITS, bool WHOLE>
__global__ void __launch_bounds__(kQkThreads, kQkCtas) qk_norm_rope_kv_kernel(const QkNormParams p, int q_parts, int per_row, int run, int longer) {
  pdl_begin();
  constexpr int kLanes = D / 16, kHeads = 32 / kLanes, kTop = BITS == 4 ? 7 : 127;
  __shared__ uint4 s_raw[kQkDepth][2][kQkThreads];
  const int lane = threadIdx.x & 31, g = lane / kLanes, j = lane % kLanes;
  const unsigned mask = ((1u << kLanes) - 1u) << (lane & ~(kLanes - 1));
  const int heads = p.Hq + 2 * p.Hk;
  // the first `longer` warps have run + 1 items, the others run
  const int warp = blockIdx.x * (kQkThreads / 32) + (threadIdx.x >> 5);
  const int begin = warp * run + min(warp, longer), end = begin + run + (warp < longer ? 1 : 0);
  if (begin >= end) return;
  int row = begin / per_row, part = begin - row * per_row, f_left = end - begin, f_part = part;
  constexpr unsigned kSlot = 2 * kQkThreads * 16;  // bytes
  unsigned slot = 0, f_slot = 0;
  unsigned char* const raw_bytes = reinterpret_cast<unsigned char*>(&s_raw[0][0][threadIdx.x]);
  const uint32_t raw_at = static_cast<uint32_t>(__cvta_generic_to_shared(raw_bytes));
  // where the next item's values lie (WHOLE), or its row's
  const uint4* f_src = reinterpret_cast<const uint4*>(p.qkv) + (WHOLE ? static_cast<size_t>(begin) * (kHeads * D / 8) : static_cast<size_t>(row) * heads * (D / 8)) + g * (D / 8) + j;
  auto fetch = [&]() {  // the next item that is not on its way yet
    if (f_left > 0) {
      if (WHOLE) {
        copy16_async(raw_at + f_slot, f_src);
        copy16_async(raw_at + f_slot + kQkThreads * 16, f_src + kLanes);
        f_src += kHeads * D / 8;
      } else {
        const bool q = f_part < q_parts;
        const int first = (q ? f_part : f_part - q_parts) * kHeads;  // of the item's heads, counted from the first q or k head
        if (first + g < (q ? p.Hq : 2 * p.Hk)) {
          const uint4* src = f_src + (q ? first : p.Hq + first) * (D / 8);
          copy16_async(raw_at + f_slot, src);
          copy16_async(raw_at + f_slot + kQkThreads * 16, src + kLanes);
        }
        if (++f_part == per_row) f_part = 0, f_src += heads * (D / 8);
      }
    }
    --f_left, f_slot = (f_slot + kSlot) % (kQkDepth * kSlot);
    copies_commit();
  };
  int next_pos = __ldg(p.pos_rows + row), next_kv = __ldg(p.kv_rows + row);
#pragma unroll
  for (int i = 0; i < kQkDepth - 1; ++i) fetch();
  for (int item = begin; item < end; ++row, part = 0) {
    const int pos = next_pos, kv_row = next_kv, stop = min(end, item + per_row - part);  // this row's items of the run
    if (row + 1 < p.rows) next_pos = __ldg(p.pos_rows + row + 1), next_kv = __ldg(p.kv_rows + row + 1);
    // a bad index skips the row instead of touching memory outside the tables or the pool
    const bool sound = pos >= 0 && pos < p.max_pos && kv_row >= 0 && kv_row < p.stride;
    const float4* cp = reinterpret_cast<const float4*>(p.cos_tbl + static_cast<size_t>(sound ? pos : 0) * (D / 2) + 8 * j);
    const float4* sp = reinterpret_cast<const float4*>(p.sin_tbl + static_cast<size_t>(sound ? pos : 0) * (D / 2) + 8 * j);

    if (part < q_parts) {
      F32x2 ac[4], as[4], bc[4], bs[4];  // rot = (a ac - b bs, b bc + a as), bs kept negative
      {
        const float4 c0 = __ldg(cp), c1 = __ldg(cp + 1), s0 = __ldg(sp), s1 = __ldg(sp + 1);
        ac[0] = f32x2(c0.x, c0.y), ac[1] = f32x2(c0.z, c0.w), ac[2] = f32x2(c1.x, c1.y), ac[3] = f32x2(c1.z, c1.w);
        as[0] = f32x2(s0.x, s0.y), as[1] = f32x2(s0.z, s0.w), as[2] = f32x2(s1.x, s1.y), as[3] = f32x2(s1.z, s1.w);
        const uint4 one = make_uint4(0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u);
        const uint4 a4 = p.wq != nullptr ? __ldg(reinterpret_cast<const uint4*>(p.wq) + j) : one;
        const uint4 b4 = p.wq != nullptr ? __ldg(reinterpret_cast<const uint4*>(p.wq) + kLanes + j) : one;
        const uint32_t aw[4] = {a4.x, a4.y, a4.z, a4.w}, bw[4] = {b4.x, b4.y, b4.z, b4.w};
        const F32x2 minus = f32x2(-1.0f, -1.0f);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const F32x2 a = bf16x2_f32(aw[e]), b = bf16x2_f32(bw[e]);
          bc[e] = mul2(b, ac[e]), bs[e] = mul2(mul2(b, as[e]), minus);
          ac[e] = mul2(a, ac[e]), as[e] = mul2(a, as[e]);
        }
      }
      uint4* dst = reinterpret_cast<uint4*>(p.q_rot) + (static_cast<size_t>(row) * p.Hq + part * kHeads + g) * (D / 8) + j;
      const int q_stop = min(q_parts - part, stop - item);
#pragma unroll 1
      for (int i = 0; i < q_stop; ++i, dst += kHeads * D / 8) {
        fetch();
        copies_wait<kQkDepth - 1>();
        const uint4 a4 = *reinterpret_cast<const uint4*>(raw_bytes + slot);
        const uint4 b4 = *reinterpret_cast<const uint4*>(raw_bytes + slot + kQkThreads * 16);
        slot = (slot + kSlot) % (kQkDepth * kSlot);
        if (!sound || (!WHOLE && (part + i) * kHeads + g >= p.Hq)) continue;
        const F32x2 a[4] = {bf16x2_f32(a4.x), bf16x2_f32(a4.y), bf16x2_f32(a4.z), bf16x2_f32(a4.w)};
        const F32x2 b[4] = {bf16x2_f32(b4.x), bf16x2_f32(b4.y), bf16x2_f32(b4.z), bf16x2_f32(b4.w)};
        float rn = 1.0f;
        if (p.wq != nullptr) {
          F32x2 s2 = mul2(a[0], a[0]), t2 = mul2(b[0], b[0]);
#pragma unroll
          for (int e = 1; e < 4; ++e) s2 = fma2(a[e], a[e], s2), t2 = fma2(b[e], b[e], t2);
          float s0, s1, t0, t1;
          f32x2_split(s2, s0, s1);
          f32x2_split(t2, t0, t1);
          float ss = (s0 + s1) + (t0 + t1);
#pragma unroll
          for (int o = 1; o < kLanes; o <<= 1) ss += __shfl_xor_sync(mask, ss, o);
          rn = rsqrtf(ss * (1.0f / D) + p.eps);
        }
        const F32x2 rn2 = f32x2(rn, rn);
        uint32_t lo[4], hi[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float x, y;
          f32x2_split(mul2(fma2(b[e], bs[e], mul2(a[e], ac[e])), rn2), x, y);
          lo[e] = pack_bf16x2(x, y);
          f32x2_split(mul2(fma2(a[e], as[e], mul2(b[e], bc[e])), rn2), x, y);
          hi[e] = pack_bf16x2(x, y);
        }
        st_stream(dst, make_uint4(lo[0], lo[1], lo[2], lo[3]));
        st_stream(dst + kLanes, make_uint4(hi[0], hi[1], hi[2], hi[3]));
      }
      part += q_stop, item += q_stop;
    }

#pragma unroll 1
    for (; item < stop; ++part, ++item) {
      fetch();
      copies_wait<kQkDepth - 1>();
      const int head = (part - q_parts) * kHeads + g;  // of k, then of v
      const uint4* const raw = reinterpret_cast<const uint4*>(raw_bytes + slot);
      slot = (slot + kSlot) % (kQkDepth * kSlot);
      if (!sound || (!WHOLE && head >= 2 * p.Hk)) continue;
      const bool is_k = head < p.Hk;
      const size_t srow = static_cast<size_t>(is_k ? head : head - p.Hk) * p.stride + kv_row;
      float lo[8], hi[8], zl[8], zh[8], sc;
      uint2 cl, ch;
      bool far_head = false;
      unpack8(raw[0], lo);
      unpack8(raw[kQkThreads], hi);
      if (is_k) {
        double rn = 1.0;
        const uint16_t* const wa = p.wk != nullptr ? p.wk + 8 * j : nullptr;
        if (wa != nullptr) {
          double ss = 0.0, st = 0.0;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const double x = lo[e], y = hi[e];
            ss += x * x, st += y * y;
          }
          ss += st;
#pragma unroll
          for (int o = 1; o < kLanes; o <<= 1) ss += __shfl_xor_sync(mask, ss, o);
          rn = rsqrt(ss * (1.0 / D) + static_cast<double>(p.eps));
          float w[8];  // products of two bf16 are exact in f32
          unpack8(__ldg(reinterpret_cast<const uint4*>(wa)), w);
#pragma unroll
          for (int e = 0; e < 8; ++e) lo[e] *= w[e];
          unpack8(__ldg(reinterpret_cast<const uint4*>(wa + D / 2)), w);
#pragma unroll
          for (int e = 0; e < 8; ++e) hi[e] *= w[e];
        }
        // the largest |y| of a pair, its last three bits the pair's number; the lane's largest and second
        unsigned best = 0, second = 0;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float4 c4 = __ldg(cp + h), s4 = __ldg(sp + h);
          const float c[4] = {c4.x, c4.y, c4.z, c4.w}, s[4] = {s4.x, s4.y, s4.z, s4.w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int e = 4 * h + i;
            const float a = lo[e], b = hi[e];
            lo[e] = fmaf(a, c[i], -(b * s[i])), hi[e] = fmaf(b, c[i], a * s[i]);
            const unsigned key = (__float_as_uint(max_or_nan(fabsf(lo[e]), fabsf(hi[e]))) & ~7u) | e;
            second = max(second, min(best, key)), best = max(best, key);
          }
        }
        unsigned top = best;
#pragma unroll
        for (int o = 1; o < kLanes; o <<= 1) top = max(top, __shfl_xor_sync(mask, top, o));
        const uint16_t* const ra = reinterpret_cast<const uint16_t*>(raw);
        const uint16_t* const rb = reinterpret_cast<const uint16_t*>(raw + kQkThreads);
        const float* const ct = reinterpret_cast<const float*>(cp);
        const float* const st = reinterpret_cast<const float*>(sp);
        far_head = top - kLeastY >= kPastY - kLeastY;
        if (far_head) {
          const FarHead h = far_key_head<D, BITS>(ra, rb, wa, wa + D / 2, ct, st, rn, mask);
          cl = h.lo, ch = h.hi, sc = h.scale;
        } else {
          const unsigned floor_key = top - 32u;  // what y lost, and the three bits
          double amax = 0.0;
          if (best >= floor_key) {
            const bool several = second >= floor_key;
            const int from = several ? 0 : best & 7, to = several ? 7 : from;
#pragma unroll 1
            for (int e = from; e <= to; ++e) {
              const double2 y = key_pair(ra, rb, wa, wa + D / 2, ct, st, e);
              amax = fmax(amax, fmax(fabs(y.x), fabs(y.y)));
            }
          }
          __syncwarp(mask);
#pragma unroll
          for (int o = 1; o < kLanes; o <<= 1) {
            const double x = __shfl_xor_sync(mask, amax, o);
            amax = x > amax ? x : amax;
          }
          sc = static_cast<float>(amax * rn * (1.0 / kTop));
          const bool plain = sc > 1e-30f;
          const float inv = plain ? static_cast<float>(rn) / sc : 0.0f;
          const float far = fmaxf(round8<BITS>(lo, inv, zl), round8<BITS>(hi, inv, zh));
          if (!plain || !(far < kNearBorder<BITS>)) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const float dl = fabsf(lo[e] * inv - (zl[e] - kMagic<BITS>)), dh = fabsf(hi[e] * inv - (zh[e] - kMagic<BITS>));
              if (!plain || !(fmaxf(dl, dh) < 2.0f * kNearBorder<BITS> - 0.5f)) {  // (these products may be rounded elsewhere)
                const double2 y = key_pair(ra, rb, wa, wa + D / 2, ct, st, e);
                zl[e] = settled<BITS>(zl[e], y.x * rn, sc, plain), zh[e] = settled<BITS>(zh[e], y.y * rn, sc, plain);
              }
            }
          }
        }
      } else {
        float amax = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) amax = max_or_nan(amax, max_or_nan(fabsf(lo[e]), fabsf(hi[e])));
#pragma unroll
        for (int o = 1; o < kLanes; o <<= 1) amax = max_or_nan(amax, __shfl_xor_sync(mask, amax, o));
        sc = __fdiv_rn(amax, static_cast<float>(kTop));  // eight significant bits over 7 or 127: never half way between floats
        const bool plain = sc > 1e-30f && sc < INFINITY;
        const float side = fmaf(sc, static_cast<float>(kTop), -amax) > 0.0f ? 1.0f - 1.0f / 524288.0f : 1.0f + 1.0f / 524288.0f;
        const float inv = plain ? __fdividef(side, sc) : 0.0f;
        round8<BITS>(lo, inv, zl);
        round8<BITS>(hi, inv, zh);
        if (!plain) {
#pragma unroll
          for (int e = 0; e < 8; ++e) zl[e] = code_by_division(lo[e], sc, kTop) + kMagic<BITS>, zh[e] = code_by_division(hi[e], sc, kTop) + kMagic<BITS>;
        }
      }
      if (!far_head) cl = pack_codes<BITS>(zl), ch = pack_codes<BITS>(zh);
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
}

template <int D, int BITS>
int launch_qk_norm(const char* fn, const QkNormParams& p) {
  constexpr int heads_per_item = 32 / (D / 16), warps = kQkThreads / 32;
  const int q_parts = (p.Hq + heads_per_item - 1) / heads_per_item;
  const int per_row = q_parts + (2 * p.Hk + heads_per_item - 1) / heads_per_item;
  const long long items = static_cast<long long>(p.rows) * per_row;
  if (items > INT_MAX - kQkDepth) return fail(fn, "too many rows");
  const int grid = static_cast<int>(std::min((items + warps - 1) / warps, static_cast<long long>(kQkCtas) * sm_count()));
  const int run = static_cast<int>(items / (grid * warps)), longer = static_cast<int>(items % (grid * warps));
  if (p.Hq % heads_per_item == 0 && 2 * p.Hk % heads_per_item == 0)
    G4_LAUNCH_PDL(fn, (qk_norm_rope_kv_kernel<D, BITS, true>), dim3(static_cast<unsigned>(grid)), dim3(kQkThreads), 0, current_stream(), p,
                  q_parts, per_row, run, longer);
  else
    G4_LAUNCH_PDL(fn, (qk_norm_rope_kv_kernel<D, BITS, false>), dim3(static_cast<unsigned>(grid)), dim3(kQkThreads), 0, current_stream(), p,
                  q_parts, per_row, run, longer);
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
