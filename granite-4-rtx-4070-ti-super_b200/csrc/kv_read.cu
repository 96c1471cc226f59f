// Rows of the quantised paged pool read back: as bf16 values, or (for the prefill attention over a 4-bit
// pool) as an 8-bit pool with the sequence's positions in order.
//
//   out[i][h][:] = bf16(code * scale) of pool row kv_rows[i]
//
// A 4-bit code is an 8-bit code as it stands (both mean code * scale), so the second form loses nothing.
#include "g4_host.h"
#include "g4_math.cuh"

#include "../../include/granite4_b200.h"

namespace g4 {
namespace {

constexpr int kReadThreads = 256;

// Eight codes of a 4-bit word as signed bytes: nibble - 8 in each byte.
__device__ __forceinline__ uint2 nibbles_to_bytes(uint32_t w) {
  const uint32_t even = w & 0x0f0f0f0fu, odd = (w >> 4) & 0x0f0f0f0fu;
  const uint32_t lo = __byte_perm(even, odd, 0x5140), hi = __byte_perm(even, odd, 0x7362);
  // bytewise nibble - 8: the subtraction never borrows across bytes when the top bit is set first
  return make_uint2(((lo | 0x80808080u) - 0x08080808u) ^ 0x80808080u, ((hi | 0x80808080u) - 0x08080808u) ^ 0x80808080u);
}

__device__ __forceinline__ float byte_value(uint32_t w, int i) {
  return static_cast<float>(static_cast<int8_t>(w >> (8 * i)));
}

struct ReadParams {
  const uint8_t* ck;
  const uint8_t* cv;
  const float* ks;
  const float* vs;
  const int* kv_rows;
  uint16_t* k_out;
  uint16_t* v_out;
  int Hk;
  long long stride, n;
};

// A thread reads eight codes of K and V and writes 16 bytes of each, N times; consecutive threads follow the output.
// The N rows' indices, then their codes and scales, are all on their way before the first is used. Bound by memory, four
// fifths of it writes: 65536 rows of 8 heads of 128 take 56 us replayed from a graph, 6.0 TB/s, and 57 - 59 called one by one (74
// with one row a thread).
template <int D, int BITS, int N>
__global__ void __launch_bounds__(kReadThreads) kv_read_kernel(const ReadParams p) {
  pdl_begin();
  constexpr int kParts = D / 8;
  const long long items = p.n * p.Hk * kParts, first = static_cast<long long>(blockIdx.x) * (kReadThreads * N) + threadIdx.x;
  int row[N];
  size_t srow[N];
#pragma unroll
  for (int u = 0; u < N; ++u) {
    const long long i = first + u * kReadThreads;
    row[u] = -1;
    if (i < items) {
      // (row, head) pairs of a call fit 32 bits: checked by the launcher
      const unsigned rh = static_cast<unsigned>(i / kParts), r = rh / static_cast<unsigned>(p.Hk);
      row[u] = __ldg(p.kv_rows + r);
      srow[u] = static_cast<size_t>(rh - r * static_cast<unsigned>(p.Hk)) * p.stride;
    }
  }
  uint2 w[N][2];
  float s[N][2];
#pragma unroll
  for (int u = 0; u < N; ++u) {
    const int part = static_cast<int>((first + u * kReadThreads) % kParts);
    const bool have = row[u] >= 0 && row[u] < p.stride;
    if (have) srow[u] += row[u];
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      w[u][kv] = make_uint2(0u, 0u), s[u][kv] = 0.0f;
      if (have) {
        const uint8_t* cache = (kv ? p.cv : p.ck) + srow[u] * (D * BITS / 8);
        if (BITS == 4) w[u][kv].x = __ldg(reinterpret_cast<const uint32_t*>(cache) + part);
        else w[u][kv] = __ldg(reinterpret_cast<const uint2*>(cache) + part);
        s[u][kv] = __ldg((kv ? p.vs : p.ks) + srow[u]);
      }
    }
  }
#pragma unroll
  for (int u = 0; u < N; ++u) {
    const long long i = first + u * kReadThreads;
    if (i >= items) break;
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      const uint2 b = BITS == 4 ? nibbles_to_bytes(w[u][kv].x) : w[u][kv];
      float v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = byte_value(e < 4 ? b.x : b.y, e & 3) * s[u][kv];
      st_stream(reinterpret_cast<uint4*>(kv ? p.v_out : p.k_out) + i, pack8(v));
    }
  }
}

struct WidenParams {
  const uint8_t* ck;
  const uint8_t* cv;
  const float* ks;
  const float* vs;
  const int* pt;
  int8_t* ok;
  int8_t* ov;
  float* oks;
  float* ovs;
  float* tops;
  int blocks;  // of a head
  long long stride, n;
};

// Positions [0, n) of a sequence out of the 4-bit pool into an 8-bit pool [Hk][n][128] in their order; a block's 32 positions
// of a head also leave their largest value scale.
constexpr int kWidenPositions = kReadThreads / 8;
__global__ void __launch_bounds__(kReadThreads) kv_widen_kernel(const WidenParams p) {
  pdl_begin();
  __shared__ unsigned s_top[kReadThreads / 32];
  constexpr int kParts = 128 / 16;  // a thread: 8 bytes in, 16 out
  const int h = blockIdx.x / p.blocks, part = threadIdx.x % kParts;
  const long long pos = static_cast<long long>(blockIdx.x - h * p.blocks) * kWidenPositions + threadIdx.x / kParts;
  unsigned top = 0;
  if (pos < p.n) {
    long long row = p.pt != nullptr ? __ldg(p.pt + pos) : pos;
    row = row < 0 ? 0 : (row >= p.stride ? p.stride - 1 : row);
    const size_t srow = static_cast<size_t>(h) * p.stride + row, hp = static_cast<size_t>(h) * p.n + pos;
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      const uint2 w = __ldg(reinterpret_cast<const uint2*>((kv ? p.cv : p.ck) + srow * 64) + part);
      const uint2 a = nibbles_to_bytes(w.x), b = nibbles_to_bytes(w.y);
      reinterpret_cast<uint4*>(kv ? p.ov : p.ok)[hp * kParts + part] = make_uint4(a.x, a.y, b.x, b.y);
    }
    if (part == 0) {
      // A value scale that is not finite, or takes values past fp16's range (V's type in those kernels), goes over to the
      // key's: as a logit it is masked for the rows that do not see the position, as an element of V it would reach them
      // (0 times infinity), and who sees it gets NaN either way.
      const float ks = __ldg(p.ks + srow), vs = __ldg(p.vs + srow);
      const bool sound = fabsf(vs) * 7.0f <= 65504.0f;
      p.oks[hp] = sound ? ks : __int_as_float(0x7fc00000), p.ovs[hp] = sound ? vs : 0.0f;
      if (sound) top = __float_as_uint(fabsf(vs));
    }
  }
  top = __reduce_max_sync(0xffffffffu, top);
  if (threadIdx.x % 32 == 0) s_top[threadIdx.x / 32] = top;
  __syncthreads();
  if (threadIdx.x < 32) {
    top = __reduce_max_sync(0xffffffffu, threadIdx.x < kReadThreads / 32 ? s_top[threadIdx.x] : 0u);
    if (threadIdx.x == 0) p.tops[blockIdx.x] = __uint_as_float(top);
  }
}

template <int D, int BITS>
int launch_read(const char* fn, const ReadParams& p) {
  if (p.n * p.Hk > INT_MAX) return fail(fn, "too many rows");
  const long long items = p.n * p.Hk * (D / 8);
  // one item a thread while that does not fill the card twice over: latency is what counts
  const bool few = items <= 2ll * 2048 * sm_count();
  const long long per = kReadThreads * (few ? 1 : 4), blocks = (items + per - 1) / per;
  if (few) G4_LAUNCH_PDL(fn, (kv_read_kernel<D, BITS, 1>), dim3(static_cast<unsigned>(blocks)), dim3(kReadThreads), 0, current_stream(), p);
  else G4_LAUNCH_PDL(fn, (kv_read_kernel<D, BITS, 4>), dim3(static_cast<unsigned>(blocks)), dim3(kReadThreads), 0, current_stream(), p);
  return 0;
}

}  // namespace

// Used by the prefill attention over a 4-bit pool (attn_int4.cu); out: codes [2][Hk][n][128], scales [2][Hk][n], and the
// largest value scales of every 32 positions [Hk][widen_tops(n)].
int widen_tops(long long n) { return static_cast<int>((n + kWidenPositions - 1) / kWidenPositions); }
int widen_int4(const char* fn, const uint8_t* ck, const uint8_t* cv, const float* ks, const float* vs, const int* pt,
               int Hk, long long stride, long long n, int8_t* ok, int8_t* ov, float* oks, float* ovs, float* tops) {
  WidenParams p{ck, cv, ks, vs, pt, ok, ov, oks, ovs, tops, widen_tops(n), stride, n};
  const long long blocks = static_cast<long long>(p.blocks) * Hk;
  if (blocks > INT_MAX) return fail(fn, "too many positions");
  G4_LAUNCH_PDL(fn, kv_widen_kernel, dim3(static_cast<unsigned>(blocks)), dim3(kReadThreads), 0, current_stream(), p);
  return 0;
}

}  // namespace g4

extern "C" int granite4_kernel_kv_read_paged(const void* d_cache_k, const void* d_cache_v, const float* d_k_scale,
                                             const float* d_v_scale, const int* d_kv_rows, int rows, int bits, int Hk,
                                             int d, int stride, uint16_t* d_k_out, uint16_t* d_v_out) {
  const char* fn = "granite4_kernel_kv_read_paged";
  if (d_cache_k == nullptr || d_cache_v == nullptr || d_k_scale == nullptr || d_v_scale == nullptr ||
      d_kv_rows == nullptr || d_k_out == nullptr || d_v_out == nullptr || rows <= 0 || Hk <= 0 || Hk > 65535 || stride <= 0)
    return g4::fail(fn, "invalid arguments");
  if ((d != 64 && d != 128) || (bits != 4 && bits != 8)) return g4::fail(fn, "head dims of 64 and 128, pools of 4 and 8 bits");
  if (!g4::aligned16(d_cache_k) || !g4::aligned16(d_cache_v) || !g4::aligned16(d_k_out) || !g4::aligned16(d_v_out))
    return g4::fail(fn, "pointers must be 16-byte aligned");
  g4::ReadParams p{};
  p.ck = static_cast<const uint8_t*>(d_cache_k), p.cv = static_cast<const uint8_t*>(d_cache_v);
  p.ks = d_k_scale, p.vs = d_v_scale, p.kv_rows = d_kv_rows, p.k_out = d_k_out, p.v_out = d_v_out;
  p.Hk = Hk, p.stride = stride, p.n = rows;
  if (d == 128) return bits == 4 ? g4::launch_read<128, 4>(fn, p) : g4::launch_read<128, 8>(fn, p);
  return bits == 4 ? g4::launch_read<64, 4>(fn, p) : g4::launch_read<64, 8>(fn, p);
}
