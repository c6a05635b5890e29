// Attention of one new token per sequence over a paged cache: any number of query heads per KV head, head
// sizes 64, 128 and 256, bf16 or fp16, caches of that type or e4m3 with a scale per slot and head, a block
// table, and a sliding window.
//
//   s_t = scale q.k_t,  p_t = exp(s_t - m),  o = sum p_t v_t / sum p_t,  lse = m + log sum p_t
//
// in one pass over the keys with the running maximum m, in fp32 from the products on.
//
// HBM-bound: a key and its value are read once and met by the few query heads that share them. A warp owns one KV
// head (eight of its query heads) and loads its keys straight into the operand registers of mma.m16n8k16, tokens as
// M: lane (g, t) has the 16-byte pieces t + 4 j of tokens g and g + 8, and the order of the reduction that this makes
// is given to q as well. V is turned by movmatrix, O^T = V^T P^T with features as M. The loop has no barrier; K of the
// next tile is requested when S is computed, V of a later one when O is.
//   * V in registers like K, or, for e4m3 and for 256 features, two tiles of it in shared memory by asynchronous copies that a
//     lane reads back itself (128 sequences in e4m3: all in registers 235 to 249 us, V in shared memory 218, K too 223;
//     three of up to 131 072 with 256 features, K and V there: 35, V alone 31).
//   * P goes in as two pieces, of bf16, which have the exponents of fp32: both hold what they should down to a weight (times its scale)
//     of 2^-110. Both are positive for a positive weight, so that an infinite value stays infinite: hi = P cut to its leading bits,
//     lo = the rest. One piece would put its own rounding beside the output's, and more of it the fewer keys there are.
//   * Groups of four query heads and fewer leave half of the eight columns free: the second piece of P goes there, and the
//     accumulators of the two halves are added at the end (64 sequences of up to 8 192 tokens 166 -> 161 us).
//   * fp16: the pieces of P are fp16, the largest weight at 2^15 (the sum too), as long as a tile's weights are 2^-23 of that
//     and more, which two pieces hold. Below, fp16's end at 2^-24 takes their bits, and where the key with the largest weight has
//     no value they are all there is: such a tile takes tf32 (mma.m16n8k8), which holds the pieces of bf16 and fp16 values
//     exactly. Three sequences of up to 131 072 tokens, seven heads over one of 256: 30.9 us, all on tf32 31.7; 64 of up to 8 192,
//     28 heads over 4 of 128: 84.5 and 87 to 90.
//   * e4m3 becomes fp16 exactly, NaN included (one conversion for a pair: 1.6 cycles of an SM for a word of each lane,
//     against 3.6 by shifts to bf16; mma.m16n8k32 on e4m3 itself, with q in pieces, takes more instructions in all), and V
//     goes on to bf16, exact too. The scale of a key multiplies its score, the scale of a value its weight: these products differ by as much
//     as scales do (a row of zeros is stored with the scale 1), and need the exponents. On tf32 the same is slower: 64
//     sequences with seven heads over each of four 64 against 61 us.
//   * Pages of whole blocks of 16 tokens need one look-up and one address for a block; others one for every token
//     (370 -> 300 instructions a block, e4m3 433 -> 390).
//
// Work split: flat_share.cuh over tiles of 16 tokens (32 in e4m3, whose chain from K to O is long). A CTA's warps take
// up to four (KV head, block of query heads) pairs; where there are fewer, or short sequences that fit the GPU at once,
// several warps take a pair's tiles in turn and put their parts together in shared memory. A share that ends inside a sequence leaves a partial (m, l, O)
// for the merge kernel.
//
// Measured, whole calls, over several GPUs of one kind: 64 sequences of up to 8 192 tokens, 32 heads over 8 of 128, bf16 (1.03 GB) 160 to
// 167 us, 6.2 to 6.5 TB/s, 0.945 to 0.99 of the copy rate. 128 of them in e4m3 (1.19 GB) 203 to 227, 0.80 to 0.90, 116 M instructions at 0.59 of
// the issue rate: it runs into the power limit on some (1.6 GHz), and fewer instructions are what helps there. Three of up to 131 072
// tokens, seven heads over one of 256, fp16 (98 MB) 31, half the rate: five tiles to a warp, which the start, the join and the merge (10)
// outlast; in e4m3 39 (50 MB). One of 41 tokens 5.3, 5.9 with a warp to a pair, 8.1 with shares and merge. More than eight heads to a KV head
// take K and V once for every eight of them: 64 x 8 192, 32 heads over 2 of 128 (252 MB) 70, in e4m3 (128 MB) 55.
#pragma once
#include <algorithm>
#include <cfloat>
#include <type_traits>

#include <cuda_fp16.h>

#include "flat_share.cuh"

namespace ako {
namespace paged {

constexpr int BLOCK = 16;   // tokens of a matrix product

constexpr int WARPS = 4, THREADS = WARPS * 32;

struct Cache {
  const uint4* data;
  const float* scale;
  uint32_t page, slot, head;              // strides in 16 bytes
  uint32_t scale_page, scale_slot, scale_head;   // in elements
};
struct Params {
  const void* q;
  Cache k, v;
  const int32_t* table;
  const int32_t* lens;
  void* o;
  float* lse;
  float* part_acc;   // [slot][q_heads][D]
  float* part_ml;    // [slot][q_heads][2]
  int2* cut;
  float scale_log2;
  int batch, q_heads, kv_heads, group, head_blocks;   // head_blocks: warps for the query heads of a KV head
  int per_cta, unit_ctas;   // (KV head, block) pairs of a CTA; CTAs of a share
  int num_pages, page_size, page_shift, max_pages, window;
  int shares;        // CTAs along the tiles
  bool same_strides; // of K and V
  bool whole_rows;   // a share is one sequence
};

// Entries for the merge, as in the split of the other decode kernels: {sequence, first share, shares}, one per
// sequence where there are no more sequences than shares (a partial lies in slot sequence + share), otherwise one per
// share, for the sequence that starts in it and goes on (slot 2 share, the first one of a sequence 2 share + 1).
__device__ __forceinline__ int2 cut_entry(int b, int first, int n) { return make_int2(b, first | n << 16); }

template <int TILE>
struct Span {          // visible tokens of a sequence
  int lo, hi;
  __device__ __forceinline__ int first_tile() const { return lo / TILE; }
  __device__ __forceinline__ int tiles() const { return hi > lo ? (hi + TILE - 1) / TILE - lo / TILE : 0; }
};
template <int TILE>
__device__ __forceinline__ Span<TILE> span_of(const Params& p, int b) {
  const int64_t most = min((int64_t)p.max_pages * p.page_size, (int64_t)0x7fffff00);   // tiles end in 32 bits
  Span<TILE> s;
  s.hi = p.num_pages > 0 ? (int)min((int64_t)max(0, p.lens[b]), most) : 0;
  s.lo = p.window > 0 ? max(0, s.hi - p.window) : 0;
  return s;
}

__device__ __forceinline__ uint4 ld16(const uint4* p) {
  uint4 r;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(p));
  return r;
}
__device__ __forceinline__ uint4 lds16(uint32_t a) {
  uint4 r;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(a) : "memory");
  return r;
}
__device__ __forceinline__ void sts16(uint32_t a, const uint4& v) {
  asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(a), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ uint32_t word(const uint4& v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }

template <class T>
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma<__nv_bfloat16>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  ako::mma_bf16_16816(d, a, b0, b1);
}
template <>
__device__ __forceinline__ void mma<__half>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// The four e4m3 values of a word as two pairs of fp16: exact, NaN included.
__device__ __forceinline__ void widen(uint32_t w, uint32_t& low, uint32_t& high) {
  asm("{\n.reg .b16 l, h;\nmov.b32 {l, h}, %2;\ncvt.rn.f16x2.e4m3x2 %0, l;\ncvt.rn.f16x2.e4m3x2 %1, h;\n}\n"
      : "=r"(low), "=r"(high)
      : "r"(w));
}
__device__ __forceinline__ float power_of_two(int e) { return __int_as_float((e + 127) << 23); }   // -126 .. 127
// e with 2^e <= x < 2^(e + 1), -112 at least
__device__ __forceinline__ int exponent(float x) { return min(max(((int)(__float_as_uint(x) >> 23) & 0xff) - 127, -112), 127); }

// A weight p >= 0 as hi + lo, both positive where p is: in bf16 p cut to its leading bits, and the rest with 2^-20 of p.
template <class T>
__device__ __forceinline__ void two_pieces(float p0, float p1, uint32_t& hi, uint32_t& lo);
template <>
__device__ __forceinline__ void two_pieces<__nv_bfloat16>(float p0, float p1, uint32_t& hi, uint32_t& lo) {
  hi = __byte_perm(__float_as_uint(p0), __float_as_uint(p1), 0x7632);
  lo = ako::pack_bf16x2(fmaf(p0, 1.f + 0x1p-20f, -ako::bf16_lo(hi)), fmaf(p1, 1.f + 0x1p-20f, -ako::bf16_hi(hi)));
}
// In fp16 0, or LEAST and more: the rest is 2^-24 at least, 2^-16 of that.
constexpr float LEAST = 0x1p-8f;
template <>
__device__ __forceinline__ void two_pieces<__half>(float p0, float p1, uint32_t& hi, uint32_t& lo) {
  __half2 h = __halves2half2(__float2half_rz(p0), __float2half_rz(p1));
  hi = *reinterpret_cast<uint32_t*>(&h);
  const float2 c = __half22float2(h);
  const float r0 = p0 > 0.f ? fmaxf(p0 - c.x, 0x1p-24f) : p0, r1 = p1 > 0.f ? fmaxf(p1 - c.y, 0x1p-24f) : p1;
  __half2 l = __floats2half2_rn(r0, r1);
  lo = *reinterpret_cast<uint32_t*>(&l);
}
// D (16 x 8) += A (16 x 8, row) B (8 x 8, column), both with eight bits of exponent and ten behind the point.
__device__ __forceinline__ void mma_tf32(float (&d)[4], const float (&a)[4], float b0, float b1) {
  asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(__float_as_uint(a[0])), "r"(__float_as_uint(a[1])), "r"(__float_as_uint(a[2])), "r"(__float_as_uint(a[3])),
        "r"(__float_as_uint(b0)), "r"(__float_as_uint(b1)));
}
__device__ __forceinline__ float2 unpack_half(uint32_t v) { return __half22float2(*reinterpret_cast<__half2*>(&v)); }

template <class T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) { return ako::pack_bf16x2(a, b); }
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
  __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&v);
}

template <class T, int D>
__device__ __forceinline__ void empty_head(const Params& p, int64_t row_head) {   // one thread
  uint4* op = reinterpret_cast<uint4*>((T*)p.o + row_head * D);
  for (int i = 0; i < D / 8; ++i) op[i] = make_uint4(0u, 0u, 0u, 0u);
  p.lse[row_head] = -INFINITY;
}

// Where the tiles under way are: K in registers; V too, or (e4m3, whose work on a tile is a long chain, and 256
// features, which are too many registers) two tiles of it in shared memory. Not K as well, which was slower (above).
__host__ __device__ constexpr bool ringed(int64_t d, bool fp8) { return fp8 || d == 256; }
__host__ __device__ constexpr int ctas_per_sm(int64_t d, bool fp8) { return d == 256 && !fp8 ? 2 : 3; }
// Blocks of a tile: two in e4m3 (64 and 128 features).
__host__ __device__ constexpr int blocks(int64_t d, bool fp8) { return fp8 && d <= 128 ? 2 : 1; }
// Shared memory of a warp: V of two tiles; and what it leaves for the others of its CTA, (m, l) of 8 heads, then O.
__host__ __device__ constexpr int ring_bytes(int64_t d, bool fp8) { return ringed(d, fp8) ? 2 * blocks(d, fp8) * BLOCK * (int)d * (fp8 ? 1 : 2) : 0; }
__host__ __device__ constexpr int part_bytes(int64_t d) { return (8 * (int)d + 16) * 4; }
__host__ __device__ constexpr int warp_bytes(int64_t d, bool fp8) { return ring_bytes(d, fp8) > part_bytes(d) ? ring_bytes(d, fp8) : part_bytes(d); }

template <class T, int D, bool FP8, bool ALIGNED, bool FOLD>
__global__ void __launch_bounds__(THREADS, ctas_per_sm(D, FP8)) paged_decode_kernel(const Params p) {
  constexpr int EB = FP8 ? 1 : 2;                  // bytes of a cache element
  constexpr int NJ = D * EB / 64;                  // pieces per lane and token
  constexpr int KS = D / 16;                       // steps of 16 features
  constexpr bool RINGED = ringed(D, FP8);
  constexpr int TT = blocks(D, FP8), TILE = BLOCK * TT, R = 2 * TT;   // R: tokens of a lane in a tile
  constexpr int SLOT = R * NJ * 512, PART = warp_bytes(D, FP8);      // V of a tile; what a warp has of shared memory
  using TM = typename std::conditional<FP8, __half, T>::type;   // operand type of Q K^T
  using TV = typename std::conditional<FP8, __nv_bfloat16, T>::type;   // and of P V
  constexpr bool HALF = std::is_same<TV, __half>::value;
  constexpr float LIFT = HALF ? 15.f : 0.f;
  __shared__ int s_scan[6];
  extern __shared__ __align__(16) unsigned char s_ring[];   // [warp]: its tiles, and then its part
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  ako::pdl_trigger();
  ako::pdl_wait();   // its launch is hidden behind the kernel before; no load here is of the read-only kind
  // per_cta neighbouring (KV head, block) pairs of the same tokens; along warps for each, every along-th tile
  const int share = blockIdx.x / p.unit_ctas, unit = (blockIdx.x % p.unit_ctas) * p.per_cta + warp % p.per_cta;
  const int along = WARPS / p.per_cta, my = warp / p.per_cta;
  const int kvh = unit / p.head_blocks, h0 = (unit % p.head_blocks) * 8;      // first head of the block in its group
  const int heads = min(8, p.group - h0), head0 = kvh * p.group + h0;
  const bool by_share = p.batch > p.shares;
  const bool keeper = unit == 0 && threadIdx.x == 0;
  const bool first_cta = blockIdx.x % p.unit_ctas == 0;
  ako::Share sh0;
  if (p.whole_rows) {
    sh0 = {share, 0, span_of<TILE>(p, share).tiles(), 1};
    if (sh0.left == 0 && first_cta && threadIdx.x < 32)
      for (int h = lane; h < p.q_heads; h += 32) empty_head<T, D>(p, (int64_t)share * p.q_heads + h);
  } else {
    sh0 = ako::find_share(p.batch, share, p.shares, s_scan, [&](int r) { return span_of<TILE>(p, r).tiles(); },
                                         [&](int r) {
                                           if (!first_cta) return;
                                           for (int h = 0; h < p.q_heads; ++h) empty_head<T, D>(p, (int64_t)r * p.q_heads + h);
                                           if (!by_share) p.cut[r] = cut_entry(r, 0, 0);
                                         });
  }
  int2 cut = cut_entry(0, 0, 0);
  int left = sh0.left, b = sh0.row, skip = sh0.skip;

  const uint32_t ring = ako::smem_u32(s_ring) + warp * PART + lane * 16;
  const uint4 *kbase[ALIGNED ? 2 : 1], *vbase[ALIGNED ? 2 : 1];       // ALIGNED: of tokens g and g + 8 of a tile
#pragma unroll
  for (int i = 0; i < (ALIGNED ? 2 : 1); ++i) {
    const uint32_t row = ALIGNED ? 8 * i + g : 0;
    kbase[i] = p.k.data + (uint64_t)kvh * p.k.head + t + row * p.k.slot;
    vbase[i] = p.v.data + (uint64_t)kvh * p.v.head + t + row * p.v.slot;
  }
  // The scale that this lane fetches for its quad: t = 0, 1: K of tokens g and g + 8, t = 2, 3: V.
  const Cache& sc = t < 2 ? p.k : p.v;
  const uint32_t sc_page = sc.scale_page, sc_slot = sc.scale_slot;
  const float* sc_base = sc.scale + kvh * sc.scale_head + (ALIGNED ? (8 * (t & 1) + g) * sc_slot : 0);
  while (left > 0) {
    const Span<TILE> sp = span_of<TILE>(p, b);
    const int tiles = sp.tiles(), tile0 = sp.first_tile();
    const int te = min(tiles, skip + left);
    if (te <= skip) {                               // an empty sequence
      ++b;
      skip = 0;
      continue;
    }
    left -= te - skip;
    const int32_t* pages = p.table + (int64_t)b * p.max_pages;

    // Where this lane's tokens of a tile are. ALIGNED: pages are whole blocks, so that one page id and one slot
    // do for all 16 tokens (what follows the last token of a page is still the page's). Past the end: the last
    // block, or token. Tokens of a page that does not exist, and those past the end, are masked below.
    constexpr int IDS = ALIGNED ? TT : R;
    int id[IDS] = {}, slot[IDS] = {};
    auto fetch_ids = [&](int tile) {
#pragma unroll
      for (int i = 0; i < IDS; ++i) {
        const int tok = ALIGNED ? min((tile0 + tile) * TILE + BLOCK * i, (sp.hi - 1) / BLOCK * BLOCK)
                                : min((tile0 + tile) * TILE + 8 * i + g, sp.hi - 1);
        const int page = p.page_shift >= 0 ? tok >> p.page_shift : (int)((unsigned)tok / (unsigned)p.page_size);
        slot[i] = tok - page * p.page_size;
        id[i] = pages[page];
      }
    };
    // A tile's offsets, and R bits that say which of this lane's tokens are visible
    uint64_t koff[IDS], voff[IDS], soff[TT];
    uint32_t bits = 0, seen = 0;
    auto locate = [&](int tile) {
      bool real[IDS];
#pragma unroll
      for (int i = 0; i < IDS; ++i) {
        real[i] = (unsigned)id[i] < (unsigned)p.num_pages;
        const uint32_t page = real[i] ? id[i] : 0, sl = slot[i];
        koff[i] = (uint64_t)page * p.k.page + sl * p.k.slot;
        voff[i] = p.same_strides ? koff[i] : (uint64_t)page * p.v.page + sl * p.v.slot;
        if (FP8 && (ALIGNED || (i & 1) == (t & 1))) soff[ALIGNED ? i : i / 2] = (uint64_t)page * sc_page + sl * sc_slot;
      }
      bits = 0;
#pragma unroll
      for (int i = 0; i < R; ++i) {
        const int tok = (tile0 + tile) * TILE + 8 * i + g;
        bits |= (uint32_t)(real[ALIGNED ? i / 2 : i] && tok >= sp.lo && tok < sp.hi) << i;
      }
    };
    uint4 kc[R][NJ], vc[RINGED ? 1 : R][RINGED ? 1 : NJ];
    float scales[TT];                               // of the quad's token that is this lane's
    auto request_k = [&] {
#pragma unroll
      for (int i = 0; i < R; ++i) {
        const uint4* from = kbase[ALIGNED ? i & 1 : 0] + koff[ALIGNED ? i / 2 : i];
#pragma unroll
        for (int j = 0; j < NJ; ++j) kc[i][j] = ld16(from + 4 * j);
      }
      if (FP8) {
#pragma unroll
        for (int u = 0; u < TT; ++u) scales[u] = sc_base[soff[u]];
      }
      seen = bits;
    };
    // A lane copies what it will read itself, so waiting for its own copies is all it takes.
    auto request_v = [&](uint32_t to) {
#pragma unroll
      for (int i = 0; i < R; ++i) {
        const uint4* from = vbase[ALIGNED ? i & 1 : 0] + voff[ALIGNED ? i / 2 : i];
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
          if (RINGED) ako::cp_async16(to + (i * NJ + j) * 512, from + 4 * j);
          else vc[RINGED ? 0 : i][RINGED ? 0 : j] = ld16(from + 4 * j);
        }
      }
    };

    // q of the block's heads as B fragments (n = head g), in the order of the K pieces. FOLD: the columns 4 to 7
    // have the same four heads again, for the second piece of P.
    const int qhead = FOLD ? g & 3 : g;
    uint32_t qb[KS][2];
#pragma unroll
    for (int i = 0; i < KS; ++i) qb[i][0] = qb[i][1] = 0u;
    if (qhead < heads) {
      const unsigned char* qp = (const unsigned char*)p.q + ((int64_t)b * p.q_heads + head0 + qhead) * D * 2;
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        if (FP8) {                                  // 16 features, a word of K has four
          const uint4 x = *reinterpret_cast<const uint4*>(qp + (64 * j + 16 * t) * 2);
          const uint4 y = *reinterpret_cast<const uint4*>(qp + (64 * j + 16 * t + 8) * 2);
          const uint32_t w[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            qb[4 * j + i][0] = w[2 * i];
            qb[4 * j + i][1] = w[2 * i + 1];
          }
        } else {
          const uint4 x = *reinterpret_cast<const uint4*>(qp + (32 * j + 8 * t) * 2);
          qb[2 * j][0] = x.x;
          qb[2 * j][1] = x.y;
          qb[2 * j + 1][0] = x.z;
          qb[2 * j + 1][1] = x.w;
        }
      }
    }
    float qs0 = p.scale_log2, qs1 = p.scale_log2;   // of heads 2t and 2t + 1
    if (FP8 && std::is_same<T, __nv_bfloat16>::value) {
      // bf16 to fp16: times the power of two that brings the head's largest element to [2^14, 2^15). Elements down to
      // 2^-31 of that are exact, what is below is off by 2^-39 of it at most.
      float top = 0.f;
#pragma unroll
      for (int i = 0; i < KS; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) top = fmaxf(top, fmaxf(fabsf(ako::bf16_lo(qb[i][j])), fabsf(ako::bf16_hi(qb[i][j]))));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const int e = exponent(top);
      const float down = power_of_two(14 - e), back = power_of_two(e - 14);
#pragma unroll
      for (int i = 0; i < KS; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) qb[i][j] = pack2<__half>(ako::bf16_lo(qb[i][j]) * down, ako::bf16_hi(qb[i][j]) * down);
      qs0 *= __shfl_sync(0xffffffffu, back, 8 * t);
      qs1 *= __shfl_sync(0xffffffffu, back, 8 * t + 4);
    }
    // acc[i]: rows g and g + 8 of O^T step i, heads 2t and 2t + 1
    float acc[KS][4];
#pragma unroll
    for (int i = 0; i < KS; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][j] = 0.f;
    // The maxima start at the lowest finite value, so that a score of -inf weighs 0 whatever else there is.
    float m0 = -FLT_MAX, m1 = -FLT_MAX, l0 = 0.f, l1 = 0.f;

    // K is asked for a tile ahead of the work, V one (registers) or two (shared memory), page ids one ahead of that. V in
    // shared memory is a group of copies for each tile, an empty one where there is none.
    const int begin = skip + my;
    uint32_t at_slot = ring;
    if (begin < te) {
      fetch_ids(begin);
      int id0[IDS], slot0[IDS];
#pragma unroll
      for (int i = 0; i < IDS; ++i) id0[i] = id[i], slot0[i] = slot[i];
      if (begin + along < te) fetch_ids(begin + along);   // under way with the first ones
#pragma unroll
      for (int i = 0; i < IDS; ++i) {
        const int a = id[i], b = slot[i];
        id[i] = id0[i], slot[i] = slot0[i];
        id0[i] = a, slot0[i] = b;
      }
      locate(begin);
      request_k();
      request_v(ring);
#pragma unroll
      for (int i = 0; i < IDS; ++i) id[i] = id0[i], slot[i] = slot0[i];
    }
    if (RINGED) {
      ako::cp_async_commit();
      if (begin + along < te) {
        locate(begin + along);
        request_v(ring + SLOT);
      }
      ako::cp_async_commit();
      if (begin + 2 * along < te) fetch_ids(begin + 2 * along);
    }
    for (int tile = begin; tile < te; tile += along) {
      float s[TT][2][4] = {};                        // two chains of products for a block, joined below
#pragma unroll
      for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int u = 0; u < TT; ++u) {
          const uint4 &x = kc[2 * u][j], &y = kc[2 * u + 1][j];
          if (FP8) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              uint32_t a[4];
              widen(word(x, i), a[0], a[2]);
              widen(word(y, i), a[1], a[3]);
              mma<TM>(s[u][i & 1], a, qb[4 * j + i][0], qb[4 * j + i][1]);
            }
          } else {
            const uint32_t a0[4] = {x.x, y.x, x.y, y.y}, a1[4] = {x.z, y.z, x.w, y.w};
            mma<TM>(s[u][0], a0, qb[2 * j][0], qb[2 * j][1]);
            mma<TM>(s[u][1], a1, qb[2 * j + 1][0], qb[2 * j + 1][1]);
          }
        }
      float ks[R], vs[R];
      if (FP8) {
#pragma unroll
        for (int u = 0; u < TT; ++u) {               // t = 0, 1: K's two, t = 2, 3: V's
          ks[2 * u] = __shfl_sync(0xffffffffu, scales[u], lane & ~3), ks[2 * u + 1] = __shfl_sync(0xffffffffu, scales[u], (lane & ~3) | 1);
          vs[2 * u] = __shfl_sync(0xffffffffu, scales[u], (lane & ~3) | 2), vs[2 * u + 1] = __shfl_sync(0xffffffffu, scales[u], lane | 3);
        }
      }
      bool now[R], all = true;
#pragma unroll
      for (int i = 0; i < R; ++i) {
        now[i] = (seen >> i & 1) != 0;
        all &= now[i];
      }
      const bool more = tile + along < te;
      if (more) {
        if (!RINGED) locate(tile + along);
        request_k();
      }
      // a lane's tokens, heads 2t and 2t + 1
      float e[R][2];
      float n0 = -INFINITY, n1 = -INFINITY;
#pragma unroll
      for (int i = 0; i < R; ++i) {
        const float x0 = s[i / 2][0][2 * (i & 1)] + s[i / 2][1][2 * (i & 1)], x1 = s[i / 2][0][2 * (i & 1) + 1] + s[i / 2][1][2 * (i & 1) + 1];
        e[i][0] = now[i] ? x0 * (FP8 ? qs0 * ks[i] : qs0) : -INFINITY;
        e[i][1] = now[i] ? x1 * (FP8 ? qs1 * ks[i] : qs1) : -INFINITY;
        n0 = fmaxf(n0, e[i][0]);
        n1 = fmaxf(n1, e[i][1]);
      }
#pragma unroll
      for (int o = 4; o <= 16; o <<= 1) {
        n0 = fmaxf(n0, __shfl_xor_sync(0xffffffffu, n0, o));
        n1 = fmaxf(n1, __shfl_xor_sync(0xffffffffu, n1, o));
      }
      if (__any_sync(0xffffffffu, n0 > m0 || n1 > m1)) {
        n0 = fmaxf(n0, m0);
        n1 = fmaxf(n1, m1);
        const float f0 = ako::fast_exp2(m0 - n0), f1 = ako::fast_exp2(m1 - n1);
        m0 = n0;
        m1 = n1;
        l0 *= f0;
        l1 *= f1;
#pragma unroll
        for (int i = 0; i < KS; ++i) {
          acc[i][0] *= f0; acc[i][1] *= f1; acc[i][2] *= f0; acc[i][3] *= f1;
        }
      }
#pragma unroll
      for (int i = 0; i < R; ++i) {
        e[i][0] = ako::fast_exp2(e[i][0] - m0 + LIFT);
        e[i][1] = ako::fast_exp2(e[i][1] - m1 + LIFT);
        l0 += e[i][0];
        l1 += e[i][1];
      }
      if (RINGED) ako::cp_async_wait<1>();
      if (!all) {   // weight 0, but what was read in its place may hold anything
#pragma unroll
        for (int i = 0; i < R; ++i)
#pragma unroll
          for (int j = 0; j < NJ; ++j)
            if (!now[i]) {
              if (RINGED) sts16(at_slot + (i * NJ + j) * 512, make_uint4(0u, 0u, 0u, 0u));
              else vc[RINGED ? 0 : i][RINGED ? 0 : j] = make_uint4(0u, 0u, 0u, 0u);
            }
      }
      if (FP8) {
#pragma unroll
        for (int i = 0; i < R; ++i) {
          const float f = now[i] ? vs[i] : 0.f;
          e[i][0] *= f;
          e[i][1] *= f;
        }
      }
      uint32_t bh[R], bl[R];
      auto pieces = [&](auto&& cut) {
#pragma unroll
        for (int i = 0; i < R; ++i) {
          cut(e[i][0], e[i][1], bh[i], bl[i]);
          if (FOLD) {
            bh[i] = ako::movmatrix_trans(t < 2 ? bh[i] : bl[i]);
          } else {
            bh[i] = ako::movmatrix_trans(bh[i]);
            bl[i] = ako::movmatrix_trans(bl[i]);
          }
        }
      };
      auto each_step = [&](auto&& put) {               // put(accumulators, V^T of 16 features and 16 tokens, which of the tile's)
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
          for (int u = 0; u < TT; ++u) {
            const uint4 x = RINGED ? lds16(at_slot + (2 * u * NJ + j) * 512) : vc[RINGED ? 0 : 2 * u][RINGED ? 0 : j];
            const uint4 y = RINGED ? lds16(at_slot + ((2 * u + 1) * NJ + j) * 512) : vc[RINGED ? 0 : 2 * u + 1][RINGED ? 0 : j];
#pragma unroll
            for (int i = 0; i < (FP8 ? 4 : 2); ++i) {
              uint32_t a[4];
#pragma unroll
              for (int c = 0; c < 2; ++c) {
                const uint4& z = c ? y : x;
                if (FP8) {                           // turned in pairs of features: (f, f + 1) of token 2t, then of token 2t + 1
                  uint32_t w0, w1;
                  widen(ako::movmatrix_trans(word(z, i)), w0, w1);
                  const float2 v0 = unpack_half(w0), v1 = unpack_half(w1);
                  a[2 * c] = ako::pack_bf16x2(v0.x, v1.x);
                  a[2 * c + 1] = ako::pack_bf16x2(v0.y, v1.y);
                } else {
                  a[2 * c] = ako::movmatrix_trans(word(z, 2 * i));
                  a[2 * c + 1] = ako::movmatrix_trans(word(z, 2 * i + 1));
                }
              }
              put(acc[(FP8 ? 4 : 2) * j + i], a, u);
            }
          }
      };
      auto multiply = [&](float (&d)[4], const uint32_t (&a)[4], int u) {
        if (!FOLD) mma<TV>(d, a, bl[2 * u], bl[2 * u + 1]);
        mma<TV>(d, a, bh[2 * u], bh[2 * u + 1]);
      };
      bool small = false;
      if (HALF) {
        float least = now[0] ? fminf(e[0][0], e[0][1]) : INFINITY;
#pragma unroll
        for (int i = 1; i < R; ++i) least = now[i] ? fminf(least, fminf(e[i][0], e[i][1])) : least;
        small = __any_sync(0xffffffffu, least < LEAST);
      }
      if (!HALF) {
        pieces(two_pieces<__nv_bfloat16>);
        each_step(multiply);
      } else if (!small) {
        pieces(two_pieces<__half>);
        each_step(multiply);
      } else {
        pieces(two_pieces<__nv_bfloat16>);
        each_step([&](float (&d)[4], const uint32_t (&a)[4], int u) {
#pragma unroll
          for (int c = 0; c < 2; ++c) {                // eight tokens at a time: as k = t and t + 4 the tokens 2t and 2t + 1
            const float2 v0 = unpack_half(a[2 * c]), v1 = unpack_half(a[2 * c + 1]);
            const float v[4] = {v0.x, v1.x, v0.y, v1.y};
            if (!FOLD) mma_tf32(d, v, ako::bf16_lo(bl[2 * u + c]), ako::bf16_hi(bl[2 * u + c]));
            mma_tf32(d, v, ako::bf16_lo(bh[2 * u + c]), ako::bf16_hi(bh[2 * u + c]));
          }
        });
      }
      if (RINGED) {
        if (tile + 2 * along < te) {
          locate(tile + 2 * along);
          request_v(at_slot);
        }
        ako::cp_async_commit();
        if (tile + 3 * along < te) fetch_ids(tile + 3 * along);
        at_slot = at_slot == ring ? ring + SLOT : ring;
      } else if (more) {
        request_v(0);
        if (tile + 2 * along < te) fetch_ids(tile + 2 * along);
      }
    }
#pragma unroll
    for (int o = 4; o <= 16; o <<= 1) {
      l0 += __shfl_xor_sync(0xffffffffu, l0, o);
      l1 += __shfl_xor_sync(0xffffffffu, l1, o);
    }

    if (FOLD) {
#pragma unroll
      for (int i = 0; i < KS; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] += __shfl_xor_sync(0xffffffffu, acc[i][j], 2);   // both pieces of P
    }
    const bool whole = te - skip == tiles;
    const int64_t at = by_share ? 2 * (int64_t)share + (skip == 0) : (int64_t)b + share;
    if (skip == 0 && !p.whole_rows) {
      cut = cut_entry(b, share, whole ? 1 : 1 + (tiles - te + sh0.per - 1) / sh0.per);
      if (!by_share && keeper) p.cut[b] = cut;
    }
    // Lanes g = 2 x and 2 x + 1 hold the even and the odd of eight neighbouring features (16 bits), or every other pair of
    // four and the next four (e4m3): swap, so that the even lane has the first four and the odd one the last four.
    const bool odd = g & 1;
    auto each_four = [&](auto&& put) {             // put(head of the block, feature, four values)
#pragma unroll
      for (int hh = 0; hh < 2; ++hh)
#pragma unroll
        for (int i = 0; i < KS; i += 2) {
          const float a = acc[i][hh], c = acc[i][2 + hh], e = acc[i + 1][hh], f = acc[i + 1][2 + hh];
          const float r0 = __shfl_xor_sync(0xffffffffu, odd ? a : e, 4), r1 = __shfl_xor_sync(0xffffffffu, odd ? c : f, 4);
          const int col = FP8 ? 64 * (i / 4) + 16 * (g >> 1) + 4 * (i % 4) : 32 * (i / 2) + 8 * (g >> 1);
          put(2 * t + hh, col + 4 * (g & 1), FP8 ? odd ? make_float4(r0, r1, e, f) : make_float4(a, c, r0, r1)
                                                 : odd ? make_float4(r0, e, r1, f) : make_float4(a, r0, c, r1));
        }
    };
    auto finish = [&](int h, int col, float4 x, float inv) {
      if (h >= heads) return;
      const int64_t head = head0 + h;
      if (whole)
        *reinterpret_cast<uint2*>((T*)p.o + ((int64_t)b * p.q_heads + head) * D + col) =
            make_uint2(pack2<T>(x.x * inv, x.y * inv), pack2<T>(x.z * inv, x.w * inv));
      else
        *reinterpret_cast<float4*>(p.part_acc + (at * p.q_heads + head) * D + col) = x;
    };
    auto finish_ml = [&](int h, float m, float l) {
      if (h >= heads) return;
      const int64_t head = head0 + h;
      if (whole) p.lse[(int64_t)b * p.q_heads + head] = l == 0.f ? -INFINITY : (m - LIFT) + log2f(l);
      else *reinterpret_cast<float2*>(p.part_ml + (at * p.q_heads + head) * 2) = make_float2(m - LIFT, l);
    };
    if (along == 1) {
      const float i0 = l0 == 0.f ? 0.f : 1.f / l0, i1 = l1 == 0.f ? 0.f : 1.f / l1;
      each_four([&](int h, int col, float4 x) { finish(h, col, x, h & 1 ? i1 : i0); });
      if (g == 0) {
        finish_ml(2 * t, m0, l0);
        finish_ml(2 * t + 1, m1, l1);
      }
    } else {
      // the warps of a pair put theirs together, in order
      auto part = [&](int w) { return reinterpret_cast<float*>(s_ring + w * PART); };
      float* mine = part(warp);
      __syncwarp();                                // every lane is through with the tiles
      if (g == 0) {
        mine[2 * t] = m0, mine[2 * t + 1] = m1;
        mine[8 + 2 * t] = l0, mine[8 + 2 * t + 1] = l1;
      }
      each_four([&](int h, int col, float4 x) { *reinterpret_cast<float4*>(mine + 16 + h * D + col) = x; });
      __syncthreads();
      // this warp: heads my, my + along, ... of its pair
      for (int h = my; h < heads; h += along) {
        float M = -FLT_MAX, L = 0.f;
        for (int i = 0; i < along; ++i) M = fmaxf(M, part(i * p.per_cta + warp % p.per_cta)[h]);
        for (int i = 0; i < along; ++i) {
          const float* x = part(i * p.per_cta + warp % p.per_cta);
          L = fmaf(x[8 + h], exp2f(x[h] - M), L);
        }
        const float inv = L == 0.f ? 0.f : 1.f / L;
        for (int col = 4 * lane; col < D; col += 128) {
          float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
          for (int i = 0; i < along; ++i) {
            const float* x = part(i * p.per_cta + warp % p.per_cta);
            const float f = exp2f(x[h] - M);
            const float4 y = *reinterpret_cast<const float4*>(x + 16 + h * D + col);
            o = make_float4(fmaf(y.x, f, o.x), fmaf(y.y, f, o.y), fmaf(y.z, f, o.z), fmaf(y.w, f, o.w));
          }
          finish(h, col, o, inv);
        }
        if (lane == 0) finish_ml(h, M, L);
      }
      __syncthreads();                             // before the next segment's
    }
    ++b;
    skip = 0;
  }
  if (by_share && keeper && !p.whole_rows) p.cut[share] = cut;
}

// Merge. Few partials of a sequence: a warp per (sequence, head), lanes hold columns.
constexpr int MERGE_MAX = 1024;                     // shares of a call never exceed this
struct Cut {
  int64_t row, slot0;
  int n;
  bool by_share;
  __device__ __forceinline__ Cut(const Params& p, int64_t entry) {
    const int2 c = p.cut[entry];
    by_share = p.batch > p.shares;
    row = c.x;
    n = (unsigned)c.y >> 16;
    slot0 = by_share ? 2 * (int64_t)(c.y & 0xffff) : row + (c.y & 0xffff);
  }
  __device__ __forceinline__ int64_t slot(int i) const { return slot0 + (by_share ? 2 * i + (i == 0) : i); }
};
template <class T, int D>
__global__ void __launch_bounds__(128) paged_merge_few_kernel(const Params p) {
  constexpr int C = D / 32;                         // columns per lane
  const int lane = threadIdx.x & 31;
  const int64_t job = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  ako::pdl_wait();
  if (job >= (int64_t)min(p.batch, p.shares) * p.q_heads) return;
  const int head = (int)(job % p.q_heads);
  const Cut cut(p, job / p.q_heads);
  if (cut.n <= 1) return;
  float M = -FLT_MAX, L = 0.f, acc[C];
#pragma unroll
  for (int c = 0; c < C; ++c) acc[c] = 0.f;
  for (int i0 = 0; i0 < cut.n; i0 += 32) {          // 32 partials at once, with their own maximum
    float2 x = make_float2(-FLT_MAX, 0.f);
    if (i0 + lane < cut.n) x = *reinterpret_cast<const float2*>(p.part_ml + (cut.slot(i0 + lane) * p.q_heads + head) * 2);
    float top = fmaxf(M, x.x);
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float back = exp2f(M - top), f = exp2f(x.x - top);
    M = top;
    L = fmaf(L, back, x.y * f);
#pragma unroll
    for (int c = 0; c < C; ++c) acc[c] *= back;
    const int k1 = min(32, cut.n - i0);
#pragma unroll 4
    for (int k = 0; k < k1; ++k) {
      const float w = __shfl_sync(0xffffffffu, f, k);
      const float* from = p.part_acc + (cut.slot(i0 + k) * p.q_heads + head) * D + lane * C;
      float y[C];
      if (C == 2) *reinterpret_cast<float2*>(y) = *reinterpret_cast<const float2*>(from);
      else
#pragma unroll
        for (int c = 0; c < C; c += 4) *reinterpret_cast<float4*>(y + c) = *reinterpret_cast<const float4*>(from + c);
#pragma unroll
      for (int c = 0; c < C; ++c) acc[c] = fmaf(y[c], w, acc[c]);
    }
  }
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) L += __shfl_xor_sync(0xffffffffu, L, o);
  const float inv = L == 0.f ? 0.f : 1.f / L;
  const int64_t oi = cut.row * p.q_heads + head;
  uint32_t* op = reinterpret_cast<uint32_t*>((T*)p.o + oi * D + lane * C);
#pragma unroll
  for (int c = 0; c < C; c += 2) op[c / 2] = pack2<T>(acc[c] * inv, acc[c + 1] * inv);
  if (lane == 0) p.lse[oi] = L == 0.f ? -INFINITY : M + log2f(L);
}
// Many: a CTA per (sequence, head, 64 columns), a thread per partial for the weights, then 16 warps for every 16th one.
constexpr int MERGE_WARPS = 16;
template <class T, int D>
__global__ void __launch_bounds__(MERGE_WARPS * 32) paged_merge_many_kernel(const Params p) {
  constexpr int PER = MERGE_MAX / (MERGE_WARPS * 32);
  __shared__ float s_w[MERGE_MAX], s_red[2][MERGE_WARPS];
  __shared__ float2 s_acc[MERGE_WARPS][32];
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
  const int block = blockIdx.x % (D / 64);
  const int64_t job = blockIdx.x / (D / 64);
  ako::pdl_wait();
  const int head = (int)(job % p.q_heads);
  const Cut cut(p, job / p.q_heads);
  if (cut.n <= 1) return;
  float2 x[PER];
  float M = -FLT_MAX, L = 0.f;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int k = i * MERGE_WARPS * 32 + tid;
    x[i] = make_float2(-FLT_MAX, 0.f);
    if (k < cut.n) x[i] = *reinterpret_cast<const float2*>(p.part_ml + (cut.slot(k) * p.q_heads + head) * 2);
    M = fmaxf(M, x[i].x);
  }
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
  if (lane == 0) s_red[0][w] = M;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < MERGE_WARPS; ++i) M = fmaxf(M, s_red[0][i]);
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const float f = exp2f(x[i].x - M);
    s_w[i * MERGE_WARPS * 32 + tid] = f;
    L = fmaf(x[i].y, f, L);
  }
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) L += __shfl_xor_sync(0xffffffffu, L, o);
  if (lane == 0) s_red[1][w] = L;
  __syncthreads();
  float2 acc = make_float2(0.f, 0.f);
#pragma unroll 8
  for (int i = w; i < cut.n; i += MERGE_WARPS) {
    const float f = s_w[i];
    const float2 y = *reinterpret_cast<const float2*>(p.part_acc + (cut.slot(i) * p.q_heads + head) * D + block * 64 + lane * 2);
    acc.x = fmaf(y.x, f, acc.x);
    acc.y = fmaf(y.y, f, acc.y);
  }
  s_acc[w][lane] = acc;
  __syncthreads();
  if (w != 0) return;
  L = s_red[1][0];
#pragma unroll
  for (int i = 1; i < MERGE_WARPS; ++i) {
    acc.x += s_acc[i][lane].x;
    acc.y += s_acc[i][lane].y;
    L += s_red[1][i];
  }
  const float inv = L == 0.f ? 0.f : 1.f / L;
  const int64_t oi = cut.row * p.q_heads + head;
  *reinterpret_cast<uint32_t*>((T*)p.o + oi * D + block * 64 + lane * 2) = pack2<T>(acc.x * inv, acc.y * inv);
  if (lane == 0 && block == 0) p.lse[oi] = L == 0.f ? -INFINITY : M + log2f(L);
}

struct Plan {
  int head_blocks, per_cta, unit_ctas;
  int shares;
  bool whole_rows;
  size_t ml, acc, total;   // offsets in the workspace; the entries are first
};
inline Plan plan_for(int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t dim, int64_t max_pages, int64_t page_size, int64_t window,
              bool fp8) {
  Plan pl;
  pl.head_blocks = (int)ako::cdiv(q_heads / kv_heads, (int64_t)8);
  const int64_t units = kv_heads * pl.head_blocks;
  pl.per_cta = units % 4 == 0 ? 4 : units % 2 == 0 ? 2 : 1;
  pl.unit_ctas = (int)(units / pl.per_cta);
  // All CTAs resident at once, and a tile at least for a warp. What the lengths are is known on the device only.
  const int64_t resident = (int64_t)ako::sm_count() * ctas_per_sm(dim, fp8);
  const int64_t TILE = BLOCK * blocks(dim, fp8);
  int64_t tokens = std::min<int64_t>(max_pages * page_size, 0x7fffff00);   // more are not read
  if (window > 0 && tokens - TILE > window) tokens = window + TILE;
  const int64_t each = ako::cdiv(tokens, TILE), tiles = batch * each;
  // Sequences that can only be short (by the table's width, or the window) get a CTA each (for its KV heads), and nothing
  // is left to merge: up to 4 tiles for a warp, 8 where there are CTAs enough. 32 heads over 8 of 128 in bf16, shares and
  // merge against this: 1 x 64 tokens 7.4 -> 6.3 us, 20 x 16 5.8 -> 4.0, 200 x 64 13.7 -> 10.3, 200 x 128 21.4 -> 19.2; past
  // that 1 x 128 7.1 -> 9.5. Eight heads over one: 20 x 16 16.0 -> 4.7.
  // While the GPU holds a CTA for every pair, the four warps of a CTA share one pair's tiles: 1 x 64 tokens 6.3 -> 4.2 us,
  // 1 x 128 7.2 -> 5.0, 40 x 256 14.6 -> 10.0; with twice the pairs 60 x 64 8.2 -> 8.9 and 120 x 64 9.1 -> 13.6. 512 tokens, 8 tiles
  // for a warp: 24 x 8 pairs 18.9 -> 15.4, 8 x 8 10.9 -> 10.5, but 1 x 8 7.5 -> 10.1 and 24 x 1 9.9 -> 11.8.
  const bool spread = batch * units <= resident && each > 1 && each <= (8 * batch * units >= resident ? 8 : 4) * WARPS;
  if (spread) {
    pl.per_cta = 1;
    pl.unit_ctas = (int)units;
  }
  const int64_t along = WARPS / pl.per_cta;
  pl.whole_rows = spread || each <= (batch * pl.unit_ctas >= resident ? 8 : 4) * along;
  if (pl.whole_rows) {
    pl.shares = (int)batch;
    pl.ml = pl.acc = pl.total = 0;
    return pl;
  }
  int64_t shares = std::min(resident / pl.unit_ctas, ako::cdiv(tiles, along));
  pl.shares = (int)std::max<int64_t>(1, std::min<int64_t>(shares, MERGE_MAX));
  const int64_t entries = std::min<int64_t>(batch, pl.shares), slots = entries + pl.shares;
  pl.ml = (entries * sizeof(int2) + 255) / 256 * 256;
  pl.acc = pl.ml + ((size_t)slots * q_heads * 8 + 255) / 256 * 256;
  pl.total = pl.acc + (size_t)slots * q_heads * dim * 4;
  return pl;
}
template <class T, int D, bool FP8, bool ALIGNED, bool FOLD>
int launch(const Params& p, const Plan& pl, cudaStream_t st) {
  constexpr int most = WARPS * warp_bytes(D, FP8);
  if (!ako::ensure_dynamic_smem<paged_decode_kernel<T, D, FP8, ALIGNED, FOLD>>(most)) return AKO4X_ELAUNCH;
  const int smem = ringed(D, FP8) || pl.per_cta < WARPS ? most : 0;
  if (ako::launch_pdl(true, paged_decode_kernel<T, D, FP8, ALIGNED, FOLD>, dim3((unsigned)(pl.shares * pl.unit_ctas)), dim3(THREADS), smem, st, p) !=
      cudaSuccess)
    return AKO4X_ELAUNCH;
  if (pl.shares == 1 || pl.whole_rows) return AKO4X_OK;
  const int64_t jobs = (int64_t)std::min(p.batch, p.shares) * p.q_heads;
  // Partials of a sequence: a warp for all of them, or 16. 32 heads over 8 of 128: 1 x 2 048 tokens 34.0 and 10.6 us, 16 x 4 096 49.0
  // and 48.0, 64 x 2 048 86 and 98; seven heads over one of 256: 1 x 65 536 79 and 23, 32 x 4 096 31.9 and 31.2.
  const bool many = p.shares >= 8LL * p.batch;
  const cudaError_t e = many ? ako::launch_pdl(true, paged_merge_many_kernel<T, D>, dim3((unsigned)jobs * (D / 64)), dim3(MERGE_WARPS * 32), 0, st, p)
                             : ako::launch_pdl(true, paged_merge_few_kernel<T, D>, dim3((unsigned)ako::cdiv(jobs, (int64_t)4)), dim3(128), 0, st, p);
  return e == cudaSuccess ? AKO4X_OK : AKO4X_ELAUNCH;
}
template <class T, int D, bool FP8>
int launch(const Params& p, const Plan& pl, cudaStream_t st) {
  const bool fold = p.group <= 4;
  if (p.page_size % BLOCK == 0) return fold ? launch<T, D, FP8, true, true>(p, pl, st) : launch<T, D, FP8, true, false>(p, pl, st);
  return fold ? launch<T, D, FP8, false, true>(p, pl, st) : launch<T, D, FP8, false, false>(p, pl, st);
}
template <class T, bool FP8>
int launch_dim(const Params& p, const Plan& pl, int64_t dim, cudaStream_t st) {
  if (dim == 64) return launch<T, 64, FP8>(p, pl, st);
  if (dim == 128) return launch<T, 128, FP8>(p, pl, st);
  return launch<T, 256, FP8>(p, pl, st);
}

// One type of query to a source file.
int run_bf16(const Params& p, const Plan& pl, int64_t dim, bool fp8, cudaStream_t st);
int run_fp16(const Params& p, const Plan& pl, int64_t dim, bool fp8, cudaStream_t st);

}  // namespace paged
}  // namespace ako
