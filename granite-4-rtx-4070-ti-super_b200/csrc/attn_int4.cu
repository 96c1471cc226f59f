// Attention of new tokens over the 4-bit paged KV pool: one token or a few rows of every sequence (decode,
// verify), split over the length of the cache and joined; and prompt chunks.
//
//   query row r at position pos[r] sees cache positions t in (pos - window, pos] (window 0: [0, pos]);
//   position t lives in pool row table[t]; k_t = code * k_scale, v_t = code * v_scale, codes c in [-7, 7]
//   l_t = scale * q . k_t,   out = sum_t softmax(l)_t v_t,   no position seen: out = 0
//
// A position costs d + 8 bytes a kv head and 4 d multiply-adds a query head: memory bounds it as long as the
// conversion of the codes stays cheap, so nothing is converted that need not be:
//  * A nibble u = c + 8 masked out of a word IS a number of the mma's operand type. K: in the low half of a byte it is a
//    u8; two ANDs and a shift give the eight operand elements of a word. V: in bits 4-7 of a half it is the fp16
//    subnormal u 2^-20, and the power of two comes out of the output, exactly. The tensor cores line products up by the
//    operands' exponent fields, and a subnormal's is that of 2^-14: of a sum they keep what is above 2^-24 of p 2^-14. With
//    nibbles in bits 0-3 too, as u 2^-24 (two shifts a word less: 16 sessions 65.5 us instead of 67), sums were off by 2^-13 of the
//    largest p v_scale, more than the other positions of a peaked softmax are worth; in bits 4-7 it is 2^-17.
//  * The 8 of u = c + 8 is one number per column: sum_d q_d (u_d - 8) = sum q u - 8 sum q, and
//    sum_t p_t (u_t - 8) = sum p u - 8 sum p, with sum p from one more mma against ones.
//  * The row scales multiply a logit (K) and a probability (V), never an element.
//  * Both contractions have the cache positions on the 16-row side (S^T = K Q^T, m16n8k32 u8 x s8) or the 16-deep side
//    (O^T = V^T P^T, m16n8k16 fp16) and the (query row, head) pairs on the 8-column side. Which dims a lane's fragment
//    elements stand for is free as long as q's match, so a lane's K elements are 16 consecutive bytes of a row, and
//    V's come out of ldmatrix.trans on 16-bit units: four dims of two positions in a register, ready for the masks.
//  * q is two s8 columns, the digits of a 16-bit integer round(q 32639 / max |q| of the head) = 256 hi + lo: the pair's
//    logit is 256 times one accumulator element of a lane plus its neighbour, in exact integers. q is off by at most
//    2^-17 of the head's range 2 max |q| (half a step): of N(0, 1) values, logits by 3e-5 of their spread, under the
//    2^-11 that P is rounded by. (Measured at 16 sessions of up to 24000: fp16 operands, which take five instructions
//    instead of three per eight codes and twice the mma, 86 us; two e4m3 columns, which sm_100 widens to fp16 instruction
//    by instruction, 82; u8 x s8 72, the rest alike.)
// What goes into the second contraction is p v_scale, rounded to fp16 (11 bits; everything else is f32). So what a column's
// probabilities are taken against, p = exp2(l - m - under), is not its largest logit but its largest l + log2(v_scale) of the
// positions that it sees, less 10: the largest p v_scale so far is kept at 2^10, whatever its magnitude, and a scale at a position
// that a column does not see, or gives no weight to, takes no bits from the others. That moves only when a position passes it by
// 14: products reach 2^14, fp16 ends at 2^16, and most tiles leave the accumulators as they are. m is a logit, and everything
// else a difference to it, so that large logits cost no bits of the rest. p reaches 2^94 where v_scale is small: a scale, a
// zero too, counts as 2^-80 at least, so that a sum of p stays within f32. Scales up to 2^100 are as good.
//
// Work split, by size: a (group, kv head, column block) segment is one CTA's; or a cluster's, whose CTAs take equal parts
// and join them through distributed shared memory; or, for long caches, the segments' tiles of 32 positions form one line,
// cut into equal shares, one CTA each, whatever the sequences' lengths (read on the device), and pieces of a segment that
// more than one CTA worked on are joined by a second small kernel, in order of the CTAs. A CTA's four warps take every
// fourth tile of a piece, each with its own ring of asynchronous copies and its own running (max, sum, O); they merge in
// shared memory.
//
// 16 sessions of up to 24000 positions (32 / 8 heads of 128, 302 MB): 64 us, rows at 6 TB/s once they stream, 4 us before
// and 4 to join; one session at 131072 (143 MB): 36 us; without the two contractions 4 us less each. One session of 37
// positions 3.6 us, five groups of three rows at 4100 15 us, 16 groups of four at 16000 100, 118 where the softmax is so
// peaked that the base moves all the time. (GPU time, replayed from a graph; called one by one 0.3 - 2 us more.)
#include "g4_cluster.cuh"
#include "g4_host.h"
#include "g4_math.cuh"

#include "../../include/granite4_b200.h"

#include <cuda_fp16.h>

#include <algorithm>

namespace g4 {

// kv_read.cu
int widen_tops(long long n);
int widen_int4(const char* fn, const uint8_t* ck, const uint8_t* cv, const float* ks, const float* vs, const int* pt,
               int Hk, long long stride, long long n, int8_t* ok, int8_t* ov, float* oks, float* ovs, float* tops);
// attn_prefill.cu
int attn_prefill_flash(const char* fn, const uint16_t* d_q, float scale, int Hq, int Hk, int base_pos, int rows,
                       int stride, uint16_t* d_out, const int8_t* d_ck, const int8_t* d_cv, const float* d_ks,
                       const float* d_vs, const int* d_pt, const float* d_v_tops, int n_tops);

namespace {

constexpr int kTile = 32;     // positions a warp works on at a time
constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kMaxGroups = 256;   // of a launch that cuts the line of tiles
constexpr int kMaxShares = 640;   // it is cut into
constexpr int kMaxColumns = 64;   // rows of a group x query heads of a kv head
constexpr float kNone = -1e38f;  // the m of what has seen nothing: below every logit, and differences of two are finite
constexpr float kUnset = -1e30f;  // the same of `under`
constexpr float kLift = 10.0f, kSlack = 14.0f, kLeastLogScale = -80.0f;

struct Int4AttnParams {
  const uint16_t* q;
  const uint8_t* ck;
  const uint8_t* cv;
  const float* ks;
  const float* vs;
  const int* row_pos;  // NULL: row r is at base_pos + r
  int base_pos;
  const int* const* row_pt;
  const int* pt;
  uint16_t* out;
  float* part_o;   // [slots][columns][D]
  float* part_ml;  // [slots][columns][2]
  int* prefix;     // [groups + 1] tiles or chunks before each group, then the shares of a straight cut (0: chunks)
  int rows, per, groups, Hq, Hk, G, blocks;  // blocks: column blocks of a segment
  unsigned g_inv;  // ceil(65536 / G): c / G = c * g_inv >> 16 for c < 256
  long long stride;
  int max_len, window;
  float scale_log2;
  int split;    // the line of tiles is cut into gridDim.x shares
  int cluster;  // else: CTAs of a segment, a cluster (1: one CTA)
};

__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_u8s8(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void load_8x8_trans(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(at)
               : "memory");
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float log2_fast(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t halves(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// A row's value over the sum of its probabilities; 0 where it saw nothing. What is not a number stays one.
__device__ __forceinline__ uint16_t quotient_bf16(float acc, float l) {
  return static_cast<uint16_t>(pack_bf16x2(l == 0.0f ? 0.0f : __fdividef(acc, l), 0.0f));
}

// First and last position that any row of a group sees; last < first: none.
__device__ __forceinline__ void group_span(const Int4AttnParams& p, int grp, int& lo, int& hi) {
  lo = INT_MAX, hi = -1;
  const int r0 = grp * p.per, nr = min(p.per, p.rows - r0);
  for (int j = 0; j < nr; ++j) {
    const int raw = p.row_pos != nullptr ? __ldg(p.row_pos + r0 + j) : p.base_pos + r0 + j;
    if (raw < 0) continue;
    const int pos = min(raw, p.max_len - 1);
    hi = max(hi, pos);
    lo = min(lo, p.window > 0 ? max(0, pos + 1 - p.window) : 0);
  }
}
// Sum over the lanes before this one; `all` gets the sum over all lanes.
__device__ __forceinline__ int sum_before(int v, int& all) {
  const int lane = threadIdx.x & 31;
  int inc = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += u;
  }
  all = __shfl_sync(0xffffffffu, inc, 31);
  return inc - v;
}

// a / d for quotients below 2^21: a float quotient is then off by less than one.
__device__ __forceinline__ int quotient(int a, int d) {
  int q = static_cast<int>(__fdividef(static_cast<float>(a), static_cast<float>(d)));
  const int r = a - q * d;
  q += (r >= d ? 1 : 0) - (r < 0 ? 1 : 0);
  return q;
}
constexpr int kMaxQuotient = 1 << 21;

// The line of all tiles is cut straight, into shares that differ by a tile at most, whatever segments they cross, or,
// where a share would be short and the segments are few, into chunks of equal parts of each segment: a CTA that crosses
// from one segment to the next pays the start of a piece (a chain of dependent loads, 2 us) and its end twice. In the
// straight cut that start and end count as kStartTiles tiles at the head of every segment. `chunk` is a chunk's largest
// length, 0 for the straight cut.
struct Cut {
  int shares, quot, rest, chunk;
};
constexpr int kShortShare = 64;  // tiles
constexpr int kStartTiles = 8;
__device__ __forceinline__ Cut cut_line(int all, int segments, int ctas) {
  Cut c;
  c.shares = all >= ctas * kWarps ? ctas : max(1, all / kWarps);  // a tile for each warp
  c.quot = quotient(all, c.shares), c.rest = all - c.quot * c.shares;
  c.chunk = ctas >= 2 * segments && c.quot < kShortShare ? max(kWarps, quotient(all + ctas - segments - 1, ctas - segments)) : 0;
  return c;
}
// The share of a straight cut that holds tile x.
__device__ __forceinline__ int share_of(const Cut& c, int x) {
  const int big = c.rest * (c.quot + 1);
  return x < big ? quotient(x, c.quot + 1) : c.rest + quotient(x - big, c.quot);
}

__device__ __forceinline__ void copy16_async(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy4_async(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
// All of this thread's copies have landed.
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// A warp's ring of raw tiles: 32 K rows, 32 V rows, their scales, as they are in the pool (for positions that no
// row sees, the nearest that one sees). The 16-byte pieces of a row lie exchanged, so that neither the copies (two lanes a row),
// nor the eight rows of an ldmatrix piece, nor the lanes' reads of K meet a bank more often than their width asks for.
template <int D>
__device__ __forceinline__ int piece_at(int row, int piece) {
  return D == 128 ? piece ^ ((row >> 1) & 3) : piece ^ ((row >> 2) & 1);
}
constexpr int kStages = 2;
template <int D>
constexpr int kRowBytes = D / 2;
template <int D>
constexpr int kStageBytes = 2 * kTile * kRowBytes<D> + 2 * kTile * 4;
template <int D>
constexpr int kWarpBytes = kStages * kStageBytes<D>;
constexpr int kPad = 4;  // floats after a parked row of O

// NS logit tiles of four columns each: column 4 i + t of column block cb is pair c = 4 NS cb + 4 i + t, query row c / G,
// query head c % G. P and O have a tile of eight columns for two of them: column 2 t + e of tile n is pair 4 (2 n + e) + t
// (an odd NS: the odd columns of the last tile are zero).
// Registers: 128 a thread for one or two logit tiles, 168 for three or four; four tiles of wide heads spill 176 bytes of them.
// Four tiles at two CTAs per SM: 16 groups of four rows at 16000 5 % slower, two of them at 33 positions 6 %
// faster.
constexpr int ctas_per_sm(int ns) { return ns >= 3 ? 3 : 4; }
template <int D, int NS>
__global__ void __launch_bounds__(kThreads, ctas_per_sm(NS)) attn_int4_kernel(const Int4AttnParams p) {
  pdl_begin();
  constexpr int kC = 4 * NS, kNP = (NS + 1) / 2;
  constexpr int kW = D / 32 /* K words of a row per lane */, kM = D / 16 /* 16-dim tiles of O^T */;
  constexpr int kRB = kRowBytes<D>, kVAt = kTile * kRB, kSAt = 2 * kTile * kRB;
  static_assert(kWarpBytes<D> >= kC * (D + kPad) * 4 + kC * 8, "a warp parks its state in its ring");
  __shared__ __align__(16) unsigned char s_q[8 * NS][D + 16];  // a row per column of the logit tiles
  __shared__ float s_scale[4 * NS];                            // of a pair's logits
  __shared__ float2 s_cta[4 * NS];                             // (m, sum) of the CTA, where it is one of a cluster
  extern __shared__ __align__(128) unsigned char s_ring[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  unsigned char* const ring = s_ring + warp * kWarpBytes<D>;
  const uint32_t ring_at = static_cast<uint32_t>(__cvta_generic_to_shared(ring));
  const int per_group = p.Hk * p.blocks;
  // Every warp lays out the line for itself: lane L has groups [L n, L n + n), their tiles (or chunks) and those before.
  int x = 0, x_end = 1, chunk = 0;  // this CTA's share of the line, or its chunk
  const int lane_groups = (p.groups + 31) >> 5, lane_first = lane * lane_groups;
  int lane_units = 0, lane_before = 0, lane_lo = 0, lane_hi = -1;
  const int* lane_pt = nullptr;  // span and table of a lane's only group
  auto units_of = [&](int grp) -> int {
    int lo = lane_lo, hi = lane_hi;
    if (lane_groups > 1) group_span(p, grp, lo, hi);
    const int n = hi < 0 ? 0 : hi / kTile - lo / kTile + 1;
    return chunk > 0 ? quotient(n + chunk - 1, chunk) : n > 0 ? n + kStartTiles : 0;
  };
  if (p.split) {
    const int lane_end = min(lane_first + lane_groups, p.groups);
    if (lane_groups == 1 && lane_first < lane_end) {
      lane_pt = p.row_pt != nullptr ? p.row_pt[lane_first * p.per] : p.pt;
      group_span(p, lane_first, lane_lo, lane_hi);
    }
    int all;
#pragma unroll 1
    for (int gi = lane_first; gi < lane_end; ++gi) lane_units += units_of(gi);
    lane_before = sum_before(lane_units, all);
    const Cut cut = cut_line(all * per_group, p.groups * per_group, gridDim.x);
    chunk = cut.chunk;
    if (chunk > 0) {
      lane_units = 0;
#pragma unroll 1
      for (int gi = lane_first; gi < lane_end; ++gi) lane_units += units_of(gi);
      lane_before = sum_before(lane_units, all);
      x = blockIdx.x;
      x_end = min(x + 1, all * per_group);
    } else {
      x = blockIdx.x * cut.quot + min(static_cast<int>(blockIdx.x), cut.rest);
      x_end = static_cast<int>(blockIdx.x) < cut.shares ? x + cut.quot + (static_cast<int>(blockIdx.x) < cut.rest ? 1 : 0) : x;
    }
    if (blockIdx.x == 0 && warp == 0) {
      int before = lane_before;
#pragma unroll 1
      for (int gi = lane_first; gi < lane_end; ++gi) p.prefix[gi] = before, before += units_of(gi);
      if (lane == 0) p.prefix[p.groups] = all, p.prefix[p.groups + 1] = chunk > 0 ? 0 : cut.shares;
    }
  }

  while (true) {
    int grp, sub, n_tiles, first_tile, piece_begin, piece_end;  // of this segment's tiles
    int span_lo, span_hi;
    const int* pt;
    if (p.split) {
      if (x >= x_end) return;
      const int at = quotient(x, per_group);  // the group that holds the line's unit x
      const int owner = 31 - __clz(__ballot_sync(0xffffffffu, lane_units > 0 && lane_before <= at));
      int found = lane_first, before = lane_before, units = lane_units;
      if (lane_groups > 1 && lane == owner) {
#pragma unroll 1
        for (int gi = lane_first, next = lane_before; gi < min(lane_first + lane_groups, p.groups) && next <= at; ++gi) {
          const int n = units_of(gi);
          if (n > 0) found = gi, before = next, units = n;
          next += n;
        }
      }
      grp = __shfl_sync(0xffffffffu, found, owner);
      before = __shfl_sync(0xffffffffu, before, owner), units = __shfl_sync(0xffffffffu, units, owner);
      const int in = x - before * per_group;
      sub = quotient(in, units);
      piece_begin = in - sub * units, piece_end = units;
      if (lane_groups == 1) {
        span_lo = __shfl_sync(0xffffffffu, lane_lo, owner), span_hi = __shfl_sync(0xffffffffu, lane_hi, owner);
        pt = reinterpret_cast<const int*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(lane_pt), owner));
      }
    } else {
      const int segment = p.cluster == 1 ? blockIdx.x : blockIdx.x / p.cluster;
      grp = segment / per_group, sub = segment - grp * per_group;
      piece_begin = 0, piece_end = 1;
    }
    if (!p.split || lane_groups > 1) {
      pt = p.row_pt != nullptr ? p.row_pt[grp * p.per] : p.pt;
      group_span(p, grp, span_lo, span_hi);
    }
    const int hkv = p.blocks == 1 ? sub : sub / p.blocks, c0 = p.blocks == 1 ? 0 : (sub % p.blocks) * kC;
    const int r0 = grp * p.per, nrows = min(p.per, p.rows - r0), columns = min(kC, nrows * p.G - c0);
    // what the piece needs first and does not depend on one another: q, positions, the table's address
    uint32_t q_raw[NS][D / 64];
    int pos_raw[NS];
#pragma unroll
    for (int i = 0; i < NS; ++i) {
      const int cq = i * kWarps + warp, cp = 4 * i + t;
      const int j = (c0 + cq) * p.g_inv >> 16, hl = c0 + cq - j * p.G;
#pragma unroll
      for (int e = 0; e < D / 64; ++e)
        q_raw[i][e] = cq < columns ? __ldg(reinterpret_cast<const uint32_t*>(p.q + (static_cast<size_t>(r0 + j) * p.Hq + static_cast<size_t>(hkv) * p.G + hl) * D + lane * (D / 32)) + e) : 0u;
      const int row = r0 + ((c0 + cp) * p.g_inv >> 16);
      pos_raw[i] = cp < columns ? (p.row_pos != nullptr ? __ldg(p.row_pos + row) : p.base_pos + row) : INT_MAX;
    }
    first_tile = span_hi < 0 ? 0 : span_lo / kTile;
    n_tiles = span_hi < 0 ? 0 : span_hi / kTile - first_tile + 1;
    if (!p.split) {
      const int rank = p.cluster == 1 ? 0 : blockIdx.x % p.cluster;
      piece_begin = p.cluster == 1 ? 0 : rank * n_tiles / p.cluster, piece_end = p.cluster == 1 ? n_tiles : (rank + 1) * n_tiles / p.cluster;
    } else if (chunk > 0) {
      const int k = piece_begin, n = piece_end;
      piece_begin = quotient(k * n_tiles, n), piece_end = quotient((k + 1) * n_tiles, n);
      x = x_end;
    } else {
      const int past = piece_begin + x_end - x - kStartTiles;  // of the segment's tiles, the first that is not this CTA's
      piece_begin = max(0, piece_begin - kStartTiles), piece_end = min(n_tiles, past);
      x = past >= n_tiles ? x_end - (past - n_tiles) : x_end;
      if (piece_end <= 0) return;  // the share ends in the head
    }
    const size_t head_row0 = static_cast<size_t>(hkv) * p.stride;
    const uint8_t* ck = p.ck + head_row0 * kRB;
    const uint8_t* cv = p.cv + head_row0 * kRB;
    const float* ks = p.ks + head_row0;
    const float* vs = p.vs + head_row0;

    // pool row of the lane's position of a tile (past the end of what the group sees: the end's)
    auto table_row = [&](int tile) -> int {
      const int pos = min(max(tile * kTile + lane, span_lo), span_hi);
      const int row = pt != nullptr ? __ldg(pt + pos) : pos;
      return min(max(row, 0), static_cast<int>(p.stride) - 1);
    };
    // A row takes 16 bytes of two lanes (32: a sector) at a time.
    auto fetch = [&](int stage, int row) {
      const uint32_t at = ring_at + stage * kStageBytes<D>;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = 16 * i + (lane >> 1);
        const size_t off = static_cast<size_t>(static_cast<unsigned>(__shfl_sync(0xffffffffu, row, r))) * kRB + (lane & 1) * 16;
        const uint8_t *src_k = ck + off, *src_v = cv + off;
#pragma unroll
        for (int c = 0; c < kRB / 32; ++c) {
          const uint32_t dst = at + r * kRB + piece_at<D>(r, 2 * c + (lane & 1)) * 16;
          copy16_async(dst, src_k + 32 * c);
          copy16_async(dst + kVAt, src_v + 32 * c);
        }
      }
      copy4_async(at + kSAt + lane * 4, ks + row);
      copy4_async(at + kSAt + kTile * 4 + lane * 4, vs + row);
    };
    const int tile_end = first_tile + piece_end;
    int tile = first_tile + piece_begin + warp;
    int row_next = 0;
    if (tile < tile_end) {
      const int row = table_row(tile);
      if (tile + kWarps < tile_end) row_next = table_row(tile + kWarps);
      fetch(0, row);
    }

    // q's digits into shared memory: a warp per pair, D / 32 dims a lane. Bytes follow the nibbles of K's words: of
    // eight dims first 0, 2, 4, 6, then 1, 3, 5, 7.
#pragma unroll
    for (int i = 0; i < NS; ++i) {
      const int c = i * kWarps + warp;
      constexpr int kPer = D / 32;
      float f[kPer];
#pragma unroll
      for (int e = 0; e < kPer; e += 2) f[e] = bf16_lo(q_raw[i][e >> 1]), f[e + 1] = bf16_hi(q_raw[i][e >> 1]);
      unsigned top_bits = 0;
#pragma unroll
      for (int e = 0; e < kPer; ++e) top_bits = max(top_bits, __float_as_uint(f[e]) & 0x7fffffffu);
      top_bits = __reduce_max_sync(0xffffffffu, top_bits);
      const bool sound = top_bits < 0x7f800000u;  // a head that holds an infinity or a NaN gives NaN
      const float top = fmaxf(__uint_as_float(top_bits), 1e-30f), to_int = sound ? 32639.0f / top : 0.0f;
      uint32_t hi[2] = {0, 0}, lo[2] = {0, 0};  // even dims, odd dims
#pragma unroll
      for (int e = 0; e < kPer; ++e) {
        const int v = __float2int_rn(f[e] * to_int), h = (v + 128) >> 8;
        hi[e & 1] |= static_cast<uint32_t>(h & 0xff) << (8 * (e >> 1)), lo[e & 1] |= static_cast<uint32_t>((v - 256 * h) & 0xff) << (8 * (e >> 1));
      }
      unsigned char* dst = s_q[2 * c] + (lane * kPer / 8) * 8 + lane * kPer % 8 / 2;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        if (kPer == 4) {
          *reinterpret_cast<uint16_t*>(dst + 4 * u) = static_cast<uint16_t>(hi[u]);
          *reinterpret_cast<uint16_t*>(dst + 4 * u + sizeof(s_q[0])) = static_cast<uint16_t>(lo[u]);
        } else {
          dst[4 * u] = static_cast<unsigned char>(hi[u]), dst[4 * u + sizeof(s_q[0])] = static_cast<unsigned char>(lo[u]);
        }
      }
      if (lane == 0) s_scale[c] = sound ? p.scale_log2 * top / 32639.0f : __int_as_float(0x7fc00000);
    }
    __syncthreads();
    uint32_t qb[NS][kW][2];  // the lane's column g of tile i: pair 4 i + g / 2, hi (g even) or lo
    float l_scale[NS];       // of the lane's accumulator pairs 4 i + t
    int l_off[NS], pos_col[NS];
    int all_lo = 0, all_hi = INT_MAX;  // positions that every column sees
#pragma unroll
    for (int i = 0; i < NS; ++i) {
#pragma unroll
      for (int w = 0; w < kW; w += 2) {
        const uint4 v = *reinterpret_cast<const uint4*>(s_q[8 * i + g] + t * (D / 4) + 8 * w);
        qb[i][w][0] = v.x, qb[i][w][1] = v.y, qb[i][w + 1][0] = v.z, qb[i][w + 1][1] = v.w;
      }
      const int c = 4 * i + t;
      l_scale[i] = s_scale[c];
      int sums[4] = {0, 0, 0, 0};  // a K of codes 0 (u = 8) gives what the 8 of every u adds
#pragma unroll
      for (int w = 0; w < kW; ++w) mma_u8s8(sums, 0x08080808u, 0x08080808u, 0x08080808u, 0x08080808u, qb[i][w][0], qb[i][w][1]);
      l_off[i] = sums[0] * 256 + sums[1];
      // a column that is not there sees everything and is dropped
      pos_col[i] = pos_raw[i] < 0 ? -1 : c < columns ? min(pos_raw[i], p.max_len - 1) : INT_MAX;
      all_hi = min(all_hi, pos_col[i]);
      if (c < columns && p.window > 0) all_lo = max(all_lo, pos_col[i] + 1 - p.window);
    }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
      all_hi = min(all_hi, __shfl_xor_sync(0xffffffffu, all_hi, o));
      all_lo = max(all_lo, __shfl_xor_sync(0xffffffffu, all_lo, o));
    }

    float o[kNP][kM][4], osum[kNP][4], m_ref[NS], under[NS], l_run[NS];  // p = exp2(l - m_ref - under)
#pragma unroll
    for (int n = 0; n < kNP; ++n) {
#pragma unroll
      for (int b = 0; b < kM; ++b) o[n][b][0] = o[n][b][1] = o[n][b][2] = o[n][b][3] = 0.0f;
      osum[n][0] = osum[n][1] = osum[n][2] = osum[n][3] = 0.0f;
    }
#pragma unroll
    for (int i = 0; i < NS; ++i) m_ref[i] = l_run[i] = 0.0f, under[i] = kUnset;

    for (int stage = 0; tile < tile_end; tile += kWarps, stage ^= 1) {
      copies_wait();
      __syncwarp();
      if (tile + kWarps < tile_end) fetch(stage ^ 1, row_next);
      if (tile + 2 * kWarps < tile_end) row_next = table_row(tile + 2 * kWarps);
      const unsigned char* const raw = ring + stage * kStageBytes<D>;
      const float* const raw_ks = reinterpret_cast<const float*>(raw + kSAt);
      const float* const raw_vs = raw_ks + kTile;
      const int t0 = tile * kTile;

      // S^T = K Q^T for the tile's two halves
      int s[NS][2][4];
#pragma unroll
      for (int i = 0; i < NS; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h) s[i][h][0] = s[i][h][1] = s[i][h][2] = s[i][h][3] = 0;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t k[2][kW];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int r = g + 8 * i + 16 * h;
          const unsigned char* src = raw + r * kRB + (D == 128 ? piece_at<D>(r, t) * 16 : piece_at<D>(r, t >> 1) * 16 + (t & 1) * 8);
          if (D == 128) {
            const uint4 w = *reinterpret_cast<const uint4*>(src);
            k[i][0] = w.x, k[i][1] = w.y, k[i][kW - 2] = w.z, k[i][kW - 1] = w.w;
          } else {
            const uint2 w = *reinterpret_cast<const uint2*>(src);
            k[i][0] = w.x, k[i][1] = w.y;
          }
        }
#pragma unroll
        for (int w = 0; w < kW; ++w) {
          const uint32_t a0 = k[0][w] & 0x0f0f0f0fu, a1 = k[1][w] & 0x0f0f0f0fu;
          const uint32_t a2 = (k[0][w] >> 4) & 0x0f0f0f0fu, a3 = (k[1][w] >> 4) & 0x0f0f0f0fu;
#pragma unroll
          for (int i = 0; i < NS; ++i) mma_u8s8(s[i][h], a0, a1, a2, a3, qb[i][w][0], qb[i][w][1]);
        }
      }
      float fk[4], fv[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) fk[i] = raw_ks[g + 8 * i], fv[i] = raw_vs[g + 8 * i];
      float dl[NS][4];  // logits in powers of two, less m_ref, of pair 4 i + t at positions g + 8 u
#pragma unroll
      for (int i = 0; i < NS; ++i)
#pragma unroll
        for (int u = 0; u < 4; ++u)
          dl[i][u] = fmaf(static_cast<float>(s[i][u >> 1][2 * (u & 1)] * 256 + s[i][u >> 1][2 * (u & 1) + 1] - l_off[i]), fk[u] * l_scale[i], -m_ref[i]);
      const bool masked = !(t0 >= all_lo && t0 + kTile - 1 <= all_hi);  // the same for the whole warp
      if (masked) {
        asm volatile("" ::: "memory");  // (a branch, not selects)
#pragma unroll
        for (int i = 0; i < NS; ++i)
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const int pos = t0 + g + 8 * u;
            if (pos > pos_col[i] || (p.window > 0 && pos_col[i] != INT_MAX && pos <= pos_col[i] - p.window)) dl[i][u] = -INFINITY;
          }
      }
      float lv[4], z_top[NS];
#pragma unroll
      for (int u = 0; u < 4; ++u) lv[u] = fminf(fmaxf(log2_fast(fabsf(fv[u])), kLeastLogScale), 127.0f);  // (of what is not finite: 127 or the least)
      bool moves = false;
#pragma unroll
      for (int i = 0; i < NS; ++i) {
        z_top[i] = fmaxf(fmaxf(dl[i][0] + lv[0], dl[i][1] + lv[1]), fmaxf(dl[i][2] + lv[2], dl[i][3] + lv[3]));
        moves |= z_top[i] > under[i] + kSlack;
      }
      if (__any_sync(0xffffffffu, moves)) {
        float corr[2 * kNP];
        corr[2 * kNP - 1] = 1.0f;
        const auto over_positions = [](float x) {
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
          return fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
        };
#pragma unroll
        for (int i = 0; i < NS; ++i) {  // each column by what it sees itself
          const bool grows = over_positions(z_top[i]) > under[i] + kSlack;
          const float top = over_positions(fmaxf(fmaxf(dl[i][0], dl[i][1]), fmaxf(dl[i][2], dl[i][3])));
          const float m_new = grows ? m_ref[i] + top : m_ref[i], up = m_new - m_ref[i];
          float z = -INFINITY;
#pragma unroll
          for (int u = 0; u < 4; ++u) dl[i][u] -= up, z = fmaxf(z, dl[i][u] + lv[u]);
          z = over_positions(z);
          const float next = grows ? z - kLift : under[i];
          const float down = under[i] - next - up, half = exp2_fast(0.5f * down);
          corr[i] = exp2_fast(down);
          l_run[i] *= half, l_run[i] *= half;  // (a sum of 2^94 outlives a factor under f32's range)
          m_ref[i] = m_new, under[i] = next;
        }
#pragma unroll
        for (int n = 0; n < kNP; ++n) {
#pragma unroll
          for (int m = 0; m < kM; ++m) {
            o[n][m][0] *= corr[2 * n], o[n][m][2] *= corr[2 * n];
            if (2 * n + 1 < NS) o[n][m][1] *= corr[2 * n + 1], o[n][m][3] *= corr[2 * n + 1];
          }
          osum[n][0] *= corr[2 * n];
          if (2 * n + 1 < NS) osum[n][1] *= corr[2 * n + 1];
        }
      }
      uint32_t pb[kNP][2][2];
#pragma unroll
      for (int n = 0; n < kNP; ++n) {
        float pv[2][4];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int i = 2 * n + e;
          if (i >= NS) break;
          float pr[4];
#pragma unroll
          for (int u = 0; u < 4; ++u) pr[u] = exp2_fast(dl[i][u] - under[i]), pv[e][u] = pr[u] * fv[u];
          l_run[i] += (pr[0] + pr[1]) + (pr[2] + pr[3]);
          if (masked) {  // a scale that is not finite stays with the columns that see it
            asm volatile("" ::: "memory");
#pragma unroll
            for (int u = 0; u < 4; ++u)
              if (dl[i][u] == -INFINITY) pv[e][u] = 0.0f;
          }
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) pb[n][u >> 1][u & 1] = transpose8x8(halves(pv[0][u], 2 * n + 1 < NS ? pv[1][u] : 0.0f));
      }
      // O^T += V^T P^T
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int r = 16 * h + (lane & 15);
        const uint32_t at = ring_at + stage * kStageBytes<D> + kVAt + r * kRB;
#pragma unroll
        for (int c = 0; c < D / 32; c += 2) {
          uint32_t v[4];  // positions 0-7 and 8-15 of the half, dims 32 c ..; the same, dims 32 (c + 1) ..
          load_8x8_trans(v, at + piece_at<D>(r, c + (lane >> 4)) * 16);
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const uint32_t a = v[2 * u], b = v[2 * u + 1];
            constexpr uint32_t kNibble = 0x00f000f0u;
#pragma unroll
            for (int n = 0; n < kNP; ++n) {
              mma16816(o[n][2 * (c + u)], (a << 4) & kNibble, a & kNibble, (b << 4) & kNibble, b & kNibble, pb[n][h][0],
                       pb[n][h][1]);
              mma16816(o[n][2 * (c + u) + 1], (a >> 4) & kNibble, (a >> 8) & kNibble, (b >> 4) & kNibble, (b >> 8) & kNibble,
                       pb[n][h][0], pb[n][h][1]);
            }
          }
        }
#pragma unroll
        for (int n = 0; n < kNP; ++n)
          mma16816(osum[n], 0x3c003c00u, 0x3c003c00u, 0x3c003c00u, 0x3c003c00u, pb[n][h][0], pb[n][h][1]);
      }
    }

    // the four warps' states meet in shared memory, each parked in the warp's own ring
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    __syncwarp();
    float* const park = reinterpret_cast<float*>(ring);  // [kC][D + kPad], then [kC][2] (m, sum), as of p = exp2(l - m), 1 <= sum < 2
#pragma unroll
    for (int i = 0; i < NS; ++i) {
      const int n = i >> 1, e = i & 1, c = 4 * i + t;
      float l = l_run[i];
      l += __shfl_xor_sync(0xffffffffu, l, 4);
      l += __shfl_xor_sync(0xffffffffu, l, 8);
      l += __shfl_xor_sync(0xffffffffu, l, 16);
      const int ex = ((__float_as_int(l) >> 23) & 0xff) - 127;
      const float shift = __int_as_float((127 - ex) << 23);
      if (g == 0) park[kC * (D + kPad) + 2 * c] = l == 0.0f ? kNone : m_ref[i] + (under[i] + static_cast<float>(ex)), park[kC * (D + kPad) + 2 * c + 1] = l * shift;
      const float off = osum[n][e] * (8.0f / 1048576.0f);
#pragma unroll
      for (int m = 0; m < kM; ++m)  // rows g, g + 8: dims 32 (m / 2) + 4 g + 2 (m % 2), + 1
        *reinterpret_cast<float2*>(park + c * (D + kPad) + 32 * (m >> 1) + 4 * g + 2 * (m & 1)) =
            make_float2((o[n][m][e] - off) * 1048576.0f * shift, (o[n][m][2 + e] - off) * 1048576.0f * shift);
    }
    __syncthreads();
    const bool whole = piece_begin == 0 && piece_end == n_tiles;
    const size_t slot = blockIdx.x + (chunk > 0 ? 0 : static_cast<size_t>(grp) * per_group + sub);
    constexpr int kPer = D / 32;  // a warp merges every fourth column, a lane so many of its dims
    for (int c = warp; c < columns; c += kWarps) {
      float mw[kWarps], m = kNone, l = 0.0f, acc[kPer];
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        mw[w] = reinterpret_cast<const float*>(s_ring + w * kWarpBytes<D>)[kC * (D + kPad) + 2 * c];
        m = fmaxf(m, mw[w]);
      }
#pragma unroll
      for (int e = 0; e < kPer; ++e) acc[e] = 0.0f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float* parked = reinterpret_cast<const float*>(s_ring + w * kWarpBytes<D>);
        const float f = exp2_fast(mw[w] - m);
        l += f * parked[kC * (D + kPad) + 2 * c + 1];
#pragma unroll
        for (int e = 0; e < kPer; e += 2) {
          const float2 v = *reinterpret_cast<const float2*>(parked + c * (D + kPad) + lane * kPer + e);
          acc[e] += f * v.x, acc[e + 1] += f * v.y;
        }
      }
      if (p.cluster > 1) {  // (the values of warp 0's state are read by this lane alone)
#pragma unroll
        for (int e = 0; e < kPer; e += 2)
          *reinterpret_cast<float2*>(reinterpret_cast<float*>(s_ring) + c * (D + kPad) + lane * kPer + e) = make_float2(acc[e], acc[e + 1]);
        if (lane == 0) s_cta[c] = make_float2(m, l);
      } else if (whole) {
        const int j = (c0 + c) * p.g_inv >> 16, hl = c0 + c - j * p.G;
        uint16_t* const out = p.out + (static_cast<size_t>(r0 + j) * p.Hq + static_cast<size_t>(hkv) * p.G + hl) * D + lane * kPer;
        uint16_t v[kPer];
#pragma unroll
        for (int e = 0; e < kPer; ++e) v[e] = quotient_bf16(acc[e], l);
        if ((reinterpret_cast<uintptr_t>(p.out) & 3u) == 0) {
#pragma unroll
          for (int e = 0; e < kPer; e += 2) *reinterpret_cast<uint32_t*>(out + e) = v[e] | static_cast<uint32_t>(v[e + 1]) << 16;
        } else {
#pragma unroll
          for (int e = 0; e < kPer; ++e) out[e] = v[e];
        }
      } else {
#pragma unroll
        for (int e = 0; e < kPer; e += 2)
          *reinterpret_cast<float2*>(p.part_o + (slot * kC + c) * D + lane * kPer + e) = make_float2(acc[e], acc[e + 1]);
        if (lane == 0) *reinterpret_cast<float2*>(p.part_ml + (slot * kC + c) * 2) = make_float2(m, l);
      }
    }
    if (p.cluster > 1) {
      // the cluster's CTAs share the outputs out: each adds every CTA's part of its own
      namespace cg = cooperative_groups;
      cg::cluster_group cluster = cg::this_cluster();
      cluster.sync();
      const int rank = blockIdx.x % p.cluster;
      for (int i = rank * kThreads + threadIdx.x; i < columns * D; i += p.cluster * kThreads) {
        const int c = i / D, at = c * (D + kPad) + i % D;
        float m = kNone, l = 0.0f, acc = 0.0f;
#pragma unroll 1
        for (int r0_ = 0; r0_ < p.cluster; r0_ += 8) {
          float2 ml[8];
          float v[8];
#pragma unroll
          for (int u = 0; u < 8; ++u) {
            ml[u] = make_float2(kNone, 0.0f), v[u] = 0.0f;
            if (r0_ + u < p.cluster) {
              ml[u] = *cluster.map_shared_rank(s_cta + c, r0_ + u);
              v[u] = *cluster.map_shared_rank(reinterpret_cast<const float*>(s_ring) + at, r0_ + u);
            }
          }
          float top = m;
#pragma unroll
          for (int u = 0; u < 8; ++u) top = fmaxf(top, ml[u].x);
          const float keep = exp2_fast(m - top);
          l *= keep, acc *= keep, m = top;
#pragma unroll
          for (int u = 0; u < 8; ++u) {
            const float f = exp2_fast(ml[u].x - top);
            l += f * ml[u].y, acc += f * v[u];
          }
        }
        const int j = (c0 + c) * p.g_inv >> 16, hl = c0 + c - j * p.G;
        p.out[(static_cast<size_t>(r0 + j) * p.Hq + static_cast<size_t>(hkv) * p.G + hl) * D + i % D] =
            quotient_bf16(acc, l);
      }
      cluster.sync();  // nobody leaves while its memory is read
      return;
    }
    if (!p.split) return;
    __syncthreads();
  }
}

// Joins the pieces of segments that several CTAs worked on. W warps take a column of a segment: each adds every W-th
// piece, eight loads of a lane in flight, the weights exp2(m - max) worked out beside them (W = 4: once, into shared
// memory, where the four sums meet too). Four warps where there are few columns, which then have many pieces; one where
// the columns alone fill the card. The order of the sum depends on the number of pieces alone.
template <int D, int NS, int W>
__global__ void __launch_bounds__(kThreads) attn_int4_join_kernel(const Int4AttnParams p, int ctas) {
  pdl_begin();
  constexpr int kC = 4 * NS, kPer = D / 32, kFly = 8;
  __shared__ float s_w[W == 4 ? kMaxShares : 1];
  __shared__ float s_red[2][kWarps];
  __shared__ float s_acc[W == 4 ? kWarps : 1][D];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int per_group = p.Hk * p.blocks, grp = blockIdx.x / per_group, sub = blockIdx.x - grp * per_group;
  const int c = W == 4 ? blockIdx.y : blockIdx.y * kWarps + warp, first = W == 4 ? warp : 0;
  const int hkv = p.blocks == 1 ? sub : sub / p.blocks, c0 = p.blocks == 1 ? 0 : (sub % p.blocks) * kC;
  const int r0 = grp * p.per, nrows = min(p.per, p.rows - r0);
  if (c >= min(kC, nrows * p.G - c0)) return;
  const int before = __ldcg(p.prefix + grp), units = __ldcg(p.prefix + grp + 1) - before;
  const int all = __ldcg(p.prefix + p.groups) * per_group, shares = __ldcg(p.prefix + p.groups + 1);
  int n = units, slot = before * per_group + sub * units;  // pieces of the segment, and the first one's place
  if (n > 0 && shares > 0) {
    const Cut cut = cut_line(all, p.groups * per_group, ctas);
    const int i0 = share_of(cut, slot + kStartTiles);
    n = share_of(cut, slot + units - 1) - i0 + 1, slot = i0 + blockIdx.x;
  }
  if (n == 1) return;  // written by the one CTA
  const float* const part_ml = p.part_ml + (static_cast<size_t>(slot) * kC + c) * 2;
  const float* const part_o = p.part_o + (static_cast<size_t>(slot) * kC + c) * D + lane * kPer;
  float v[kFly][kPer];
  auto load = [&](int i) {
#pragma unroll
    for (int u = 0; u < kFly; ++u) {
      const int s = i + u * W;
#pragma unroll
      for (int e = 0; e < kPer; e += 2) {
        const float2 w = s < n ? __ldcg(reinterpret_cast<const float2*>(part_o + static_cast<size_t>(s) * (kC * D) + e)) : make_float2(0.0f, 0.0f);
        v[u][e] = w.x, v[u][e + 1] = w.y;
      }
    }
  };
  auto ml_of = [&](int i) {
    return i < n ? __ldcg(reinterpret_cast<const float2*>(part_ml + static_cast<size_t>(i) * (kC * 2))) : make_float2(kNone, 0.0f);
  };
  load(first);
  float m = kNone, l = 0.0f;
  if (W == 4) {
    constexpr int kEach = (kMaxShares + kThreads - 1) / kThreads;
    float2 ml[kEach];
#pragma unroll
    for (int k = 0; k < kEach; ++k) ml[k] = ml_of(threadIdx.x + k * kThreads), m = fmaxf(m, ml[k].x);
    m = warp_max(m);
    if (lane == 0) s_red[0][warp] = m;
    __syncthreads();
    m = fmaxf(fmaxf(s_red[0][0], s_red[0][1]), fmaxf(s_red[0][2], s_red[0][3]));
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
      const int i = threadIdx.x + k * kThreads;
      const float f = exp2_fast(ml[k].x - m);
      if (i < n) s_w[i] = f;
      l += f * ml[k].y;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
    if (lane == 0) s_red[1][warp] = l;
    __syncthreads();
    l = (s_red[1][0] + s_red[1][1]) + (s_red[1][2] + s_red[1][3]);
  } else {
    for (int i = lane; i < n; i += 32) m = fmaxf(m, ml_of(i).x);
    m = warp_max(m);
  }
  float acc[kPer];
#pragma unroll
  for (int e = 0; e < kPer; ++e) acc[e] = 0.0f;
  for (int i = first; i < n; i += kFly * W) {
    if (i != first) load(i);
#pragma unroll
    for (int u = 0; u < kFly; ++u) {
      float f = 0.0f;
      if (W == 4) {
        if (i + u * W < n) f = s_w[i + u * W];
      } else {
        const float2 ml = ml_of(i + u);
        f = exp2_fast(ml.x - m);
        l += f * ml.y;
      }
#pragma unroll
      for (int e = 0; e < kPer; ++e) acc[e] += f * v[u][e];
    }
  }
  if (W == 4) {
#pragma unroll
    for (int e = 0; e < kPer; ++e) s_acc[warp][lane * kPer + e] = acc[e];
    __syncthreads();
  }
  const int j = (c0 + c) * p.g_inv >> 16, hl = c0 + c - j * p.G;
  uint16_t* const out = p.out + (static_cast<size_t>(r0 + j) * p.Hq + static_cast<size_t>(hkv) * p.G + hl) * D;
  if (W == 4) {
    const int dim = threadIdx.x;
    if (dim < D) {
      const float sum = (s_acc[0][dim] + s_acc[1 % W][dim]) + (s_acc[2 % W][dim] + s_acc[3 % W][dim]);
      out[dim] = quotient_bf16(sum, l);
    }
  } else {
#pragma unroll
    for (int e = 0; e < kPer; ++e)  // (the output may lie on any 2-byte boundary)
      out[lane * kPer + e] = quotient_bf16(acc[e], l);
  }
}

// How a launch is cut: `shares` CTAs over the line of tiles, or (shares 0) `cluster` CTAs per segment.
struct Int4Plan {
  int ns, blocks, groups, shares, cluster;
  long long segments;
};

Int4Plan plan_int4(int rows, int per, int Hq, int Hk, int d, int max_len) {
  Int4Plan s{};
  const int columns = per * (Hq / Hk);
  s.ns = columns <= 4 ? 1 : columns <= 8 ? 2 : columns <= 12 ? 3 : 4;
  s.blocks = (columns + 4 * s.ns - 1) / (4 * s.ns);
  s.groups = rows / per + (rows % per != 0);
  s.segments = static_cast<long long>(s.groups) * Hk * s.blocks;
  s.cluster = 1;
  if (s.segments > kMaxQuotient || max_len <= kTile * kWarps) return s;
  const long long resident = std::min(static_cast<long long>(ctas_per_sm(s.ns)) * sm_count(), static_cast<long long>(kMaxShares));
  const long long per_segment = (static_cast<long long>(max_len) + kTile - 1) / kTile, tiles = s.segments * per_segment;
  // Costs in ns, fitted to measured calls (segments of 7 - 4096 tiles, 2 - 512 of them; within 15 % but for a few): a CTA
  // starts and ends in 4 us; its four warps take a tile in 0.2 us, in twice that with the card full, more with more columns,
  // less with narrow heads. A cluster's join costs 1.6 us; clusters leave an SM's last places empty here and there, those
  // of more than eight CTAs a quarter of the card. The line cut: a start for every segment that a CTA meets, an equal share
  // of the tiles (sequences are seldom all as long as the longest), 4.5 us for the join.
  // 64 segments of 129 tiles: clusters 12 us, cut 14. 32 of 375: 21 (clusters of 13) and 15. 40 of 47: 9 and 12.
  const auto tile_ns = [&](long long ctas) {
    return (200 + 225 * std::min(ctas, resident) / resident) * (3 + s.ns) / 4 * (d == 128 ? 8 : 5) / 8;
  };
  const auto by_segment = [&](long long n) {
    const long long ctas = s.segments * n, room = n == 1 ? resident : n <= 8 ? resident * 15 / 16 : resident * 3 / 4;
    return (ctas + room - 1) / room * (4000 + (per_segment + n - 1) / n * tile_ns(ctas)) + (n == 1 ? 0 : n <= 8 ? 1600 : 1900);
  };
  long long best = by_segment(1);
  if (cluster_enabled())
    for (int n = 2; n <= kMaxClusterCtas; ++n)
      if (by_segment(n) < best) best = by_segment(n), s.cluster = n;
  const long long cut = 4000 + 3500 * s.segments / resident + tiles * tile_ns(resident) / resident * 7 / 8 + 4500;
  if (cut >= best || s.groups > kMaxGroups || tiles > INT_MAX / 2 || static_cast<long long>(s.groups) * per_segment >= kMaxQuotient ||
      tiles / resident >= kMaxQuotient)
    return s;
  s.shares = static_cast<int>(std::min(resident, std::max(1ll, tiles / kWarps)));
  return s;
}
long long plan_bytes(const Int4Plan& s, int d) {
  return s.shares == 0 ? 0 : (s.shares + s.segments) * 4 * s.ns * (d + 2) * 4 + (s.groups + 2 + 3) / 4 * 16;
}

bool int4_shape_ok(int Hq, int Hk, int d, int per) {
  return (d == 64 || d == 128) && Hk > 0 && Hq > 0 && Hq % Hk == 0 && per > 0 && Hq / Hk <= kMaxColumns &&
         static_cast<long long>(per) * (Hq / Hk) <= kMaxColumns;
}

template <int D, int NS>
int launch_int4(const char* fn, const Int4AttnParams& p, const Int4Plan& s) {
  const cudaStream_t st = current_stream();
  if (s.segments > INT_MAX) return fail(fn, "too many rows");
  constexpr int smem = kWarps * kWarpBytes<D>;
  static_assert(smem <= 48 * 1024, "no opt-in needed");
  if (p.cluster > 1) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(s.segments * p.cluster)), cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem, cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = static_cast<unsigned>(p.cluster), attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr, cfg.numAttrs = 1;
    void (*const kernel)(const Int4AttnParams) = attn_int4_kernel<D, NS>;
    if (cluster_fits(reinterpret_cast<const void*>(kernel), cfg, p.cluster, kThreads)) {
      cfg.numAttrs = pdl_enabled() ? 2 : 1;
      G4_CUDA_TRY(fn, cudaLaunchKernelEx(&cfg, kernel, p));
      return 0;
    }
    Int4AttnParams one = p;  // a device that cannot place such a cluster
    one.cluster = 1;
    G4_LAUNCH_PDL(fn, kernel, dim3(static_cast<unsigned>(s.segments)), dim3(kThreads), smem, st, one);
    return 0;
  }
  G4_LAUNCH_PDL(fn, (attn_int4_kernel<D, NS>), dim3(static_cast<unsigned>(p.split ? s.shares : s.segments)), dim3(kThreads), smem, st, p);
  if (p.split) {
    const unsigned segments = static_cast<unsigned>(s.segments), columns = static_cast<unsigned>(std::min(4 * NS, p.per * p.G));
    if (s.segments * columns <= 2ll * sm_count())
      G4_LAUNCH_PDL(fn, (attn_int4_join_kernel<D, NS, 4>), dim3(segments, columns), dim3(kThreads), 0, st, p, s.shares);
    else
      G4_LAUNCH_PDL(fn, (attn_int4_join_kernel<D, NS, 1>), dim3(segments, (columns + kWarps - 1) / kWarps), dim3(kThreads), 0, st, p, s.shares);
  }
  return 0;
}

// Checked arguments in; without scratch every segment is one CTA's.
int attn_int4(const char* fn, Int4AttnParams p, int d, void* scratch, long long scratch_bytes, bool scratch_needed) {
  p.G = p.Hq / p.Hk;
  Int4Plan s = plan_int4(p.rows, p.per, p.Hq, p.Hk, d, p.max_len);
  if (p.window > 0 && p.window < p.max_len - kTile) {  // what a window leaves may want no cut
    const Int4Plan w = plan_int4(p.rows, p.per, p.Hq, p.Hk, d, p.window + kTile);
    if (w.shares == 0) s = w;
  }
  p.blocks = s.blocks, p.groups = s.groups;
  p.g_inv = (65536u + p.G - 1) / p.G;
  const bool have = scratch != nullptr && scratch_bytes >= plan_bytes(s, d) && aligned16(scratch);
  if (s.shares > 0 && !have) {
    if (scratch_needed) return fail(fn, "scratch missing, misaligned or smaller than the size the scratch query returns");
    s.shares = 0;
  }
  p.cluster = s.shares > 0 ? 1 : s.cluster;
  p.split = s.shares > 0;
  if (p.split) {
    p.part_o = static_cast<float*>(scratch);
    const long long slots = s.shares + s.segments;
    p.part_ml = p.part_o + slots * 4 * s.ns * d;
    p.prefix = reinterpret_cast<int*>(p.part_ml + slots * 4 * s.ns * 2);
  }
  switch (s.ns + (d == 128 ? 4 : 0)) {
    case 1: return launch_int4<64, 1>(fn, p, s);
    case 2: return launch_int4<64, 2>(fn, p, s);
    case 3: return launch_int4<64, 3>(fn, p, s);
    case 4: return launch_int4<64, 4>(fn, p, s);
    case 5: return launch_int4<128, 1>(fn, p, s);
    case 6: return launch_int4<128, 2>(fn, p, s);
    case 7: return launch_int4<128, 3>(fn, p, s);
    default: return launch_int4<128, 4>(fn, p, s);
  }
}

// Which chunks go through the kernels for an 8-bit pool. From 64 rows on the decode form pays for its tiles (every 16 / G rows
// unpack the prefix again), the widened one a start of some 20 us and a pass over the prefix, so the first is taken up to 1.4
// million rows x kv heads x positions, or until its segments no longer run at once. Measured, G 4, decode form and widened, us:
// 8 kv heads, 64 rows after 1203 positions 18 and 22, after 2500 27 and 26, after 16000 88 and 58; 77 after 1203 21 and 25;
// 192 after 0 10 and 19, after 1203 29 and 27; 256 after 0 26 and 20; 2 kv heads, 256 after 1203 19 and 23, 128 after 4000 21 and
// 28, 192 after 16000 71 and 42; 16 kv heads, 128 after 1203 46 and 30. Over 360 such calls (1 - 16 kv heads) the rule costs
// 1.4 % against the better of the two; worst are long prefixes of one kv head (64 rows after 60000: 48 and 98).
// Below 64 rows those kernels walk the cache in one piece: 48 rows after 0 positions 7 and 6, after 500 13 and 23, after 16000 70
// and 534.
bool widens(int rows, int base_pos, int Hq, int Hk, int d) {
  if (rows < 32 || d != 128 || Hq != 4 * Hk) return false;
  if (rows < 64) return base_pos <= 192 - rows;
  const long long segments = static_cast<long long>((rows + 3) / 4) * Hk;
  return segments > static_cast<long long>(ctas_per_sm(4)) * sm_count() ||
         (2ll * base_pos + rows) * rows * Hk >= 2800000;
}
int prefill_group(int Hq, int Hk) { return std::max(1, 16 / (Hq / Hk)); }
long long widened_bytes(long long n, int Hk) { return (2 * n * Hk * (128 + 4) + 4ll * Hk * widen_tops(n) + 63) / 16 * 16; }

}  // namespace
}  // namespace g4

extern "C" {

long long granite4_attn_decode_int4_scratch_bytes(int rows, int rows_per_group, int Hq, int Hk, int d, int max_len) {
  if (rows <= 0 || max_len <= 0 || !g4::int4_shape_ok(Hq, Hk, d, rows_per_group)) return -1;
  return g4::plan_bytes(g4::plan_int4(rows, rows_per_group, Hq, Hk, d, max_len), d);
}

int granite4_kernel_attn_decode_int4_paged(const uint16_t* d_q, const uint8_t* d_cache_k, const uint8_t* d_cache_v,
                                           const float* d_k_scale, const float* d_v_scale, const int* d_row_pos,
                                           const int* const* d_row_pt, const int* d_pt, int rows, int rows_per_group,
                                           int Hq, int Hk, int d, int stride, int max_len, int window, float scale,
                                           void* d_scratch, long long scratch_bytes, uint16_t* d_out) {
  const char* fn = "granite4_kernel_attn_decode_int4_paged";
  if (d_q == nullptr || d_cache_k == nullptr || d_cache_v == nullptr || d_k_scale == nullptr || d_v_scale == nullptr ||
      d_row_pos == nullptr || d_out == nullptr || rows <= 0 || stride <= 0 || max_len <= 0 ||
      (d_row_pt == nullptr && d_pt == nullptr && max_len > stride) || window < 0 || !std::isfinite(scale))
    return g4::fail(fn, "invalid arguments");
  if (!g4::int4_shape_ok(Hq, Hk, d, rows_per_group))
    return g4::fail(fn, "head dims of 64 and 128; Hq a multiple of Hk; at most 64 query rows x heads a kv head and group");
  if (!g4::aligned16(d_q) || !g4::aligned16(d_cache_k) || !g4::aligned16(d_cache_v))
    return g4::fail(fn, "q and the caches must be 16-byte aligned");
  g4::Int4AttnParams p{};
  p.q = d_q, p.ck = d_cache_k, p.cv = d_cache_v, p.ks = d_k_scale, p.vs = d_v_scale, p.out = d_out;
  p.row_pos = d_row_pos, p.row_pt = d_row_pt, p.pt = d_pt;
  p.rows = rows, p.per = rows_per_group, p.Hq = Hq, p.Hk = Hk, p.stride = stride, p.max_len = max_len, p.window = window;
  p.scale_log2 = scale * 1.4426950408889634f;
  return g4::attn_int4(fn, p, d, d_scratch, scratch_bytes, true);
}

long long granite4_prefill_attention_int4_scratch_bytes(int rows, int base_pos, int Hq, int Hk, int d) {
  if (rows <= 0 || base_pos < 0 || base_pos > INT_MAX - rows || !g4::int4_shape_ok(Hq, Hk, d, 1)) return -1;
  if (g4::widens(rows, base_pos, Hq, Hk, d)) return g4::widened_bytes(static_cast<long long>(base_pos) + rows, Hk);
  return g4::plan_bytes(g4::plan_int4(rows, g4::prefill_group(Hq, Hk), Hq, Hk, d, base_pos + rows), d);
}

int granite4_prefill_attention_int4(const uint16_t* d_q_rot, float scale, int Hq, int Hk, int d, int base_pos, int rows,
                                    int stride, uint16_t* d_out, const uint8_t* d_cache_k, const uint8_t* d_cache_v,
                                    const float* d_k_scale, const float* d_v_scale, const int* d_pt, void* d_scratch,
                                    long long scratch_bytes) {
  const char* fn = "granite4_prefill_attention_int4";
  if (d_q_rot == nullptr || d_cache_k == nullptr || d_cache_v == nullptr || d_k_scale == nullptr ||
      d_v_scale == nullptr || d_out == nullptr || base_pos < 0 || rows <= 0 || base_pos > INT_MAX - rows || stride <= 0 ||
      (d_pt == nullptr && base_pos + rows > stride) || !std::isfinite(scale))
    return g4::fail(fn, "invalid arguments");
  if (!g4::int4_shape_ok(Hq, Hk, d, 1))
    return g4::fail(fn, "head dims of 64 and 128; Hq a multiple of Hk; at most 64 query heads a kv head");
  if (!g4::aligned16(d_q_rot) || !g4::aligned16(d_cache_k) || !g4::aligned16(d_cache_v))
    return g4::fail(fn, "q and the caches must be 16-byte aligned");
  const int n = base_pos + rows;
  // (an output that those kernels cannot store to in their words takes the decode form)
  if (g4::widens(rows, base_pos, Hq, Hk, d) && reinterpret_cast<uintptr_t>(d_out) % (rows < 64 ? 4 : 16) == 0) {
    if (d_scratch == nullptr || !g4::aligned16(d_scratch) || scratch_bytes < g4::widened_bytes(n, Hk))
      return g4::fail(fn, "scratch missing, misaligned or smaller than the size the scratch query returns");
    const size_t codes = static_cast<size_t>(n) * Hk * 128, scales = static_cast<size_t>(n) * Hk;
    int8_t* ck = static_cast<int8_t*>(d_scratch);
    int8_t* cv = ck + codes;
    float* ks = reinterpret_cast<float*>(cv + codes);
    float* vs = ks + scales;
    float* tops = vs + scales;
    if (g4::widen_int4(fn, d_cache_k, d_cache_v, d_k_scale, d_v_scale, d_pt, Hk, stride, n, ck, cv, ks, vs, tops) != 0) return -1;
    const int rc = g4::attn_prefill_flash(fn, d_q_rot, scale, Hq, Hk, base_pos, rows, n, d_out, ck, cv, ks, vs, nullptr, tops,
                                          g4::widen_tops(n));
    if (rc <= 0) return rc;
  }
  g4::Int4AttnParams p{};
  p.q = d_q_rot, p.ck = d_cache_k, p.cv = d_cache_v, p.ks = d_k_scale, p.vs = d_v_scale, p.out = d_out;
  p.base_pos = base_pos, p.pt = d_pt;
  p.rows = rows, p.per = g4::prefill_group(Hq, Hk), p.Hq = Hq, p.Hk = Hk, p.stride = stride, p.max_len = n;
  p.scale_log2 = scale * 1.4426950408889634f;
  return g4::attn_int4(fn, p, d, d_scratch, scratch_bytes, false);
}

}  // extern "C"
