// Attention of one new token per sequence over a paged cache: any number of query heads per KV head, head
// sizes 64, 128 and 256, bf16 or fp16, caches of that type or e4m3 with a scale per slot and head, a block
// table, and a sliding window.
//
//   s_t = scale q.k_t,  p_t = exp(s_t - m),  o = sum p_t v_t / sum p_t,  lse = m + log sum p_t
//
// in one pass over the keys with the running maximum m, in fp32 from the products on.
//
// HBM-bound: a key and its value are read once and met by the few query heads that share them, so nothing is
// staged: a warp owns one KV head (eight of its query heads) and loads its keys straight into the operand
// registers of mma.m16n8k16, tokens as M. Lane (g, t) has the 16-byte pieces t + 4 j of tokens g and g + 8;
// the order of the reduction that this makes is given to q as well. V is loaded the same way and turned by
// movmatrix, O^T = V^T P^T with features as M. There is no barrier and no shared memory in the loop; the
// next tile's K is requested when S is computed, its V when O is.
//   * P goes in as two pieces of 16 bits, both of them positive for a positive weight, so that an infinite
//     value stays infinite: hi = P cut to its leading bits, lo = the rest. One piece would put its own rounding
//     beside the output's, and more of it the fewer keys there are.
//   * fp16: P is scaled by 2^15 on its way in (the sum too). A weight of 2^-24 of the largest is the
//     smallest fp16 value otherwise, and a long tail of keys below it would vanish from o but not from lse.
//   * e4m3 becomes fp16 exactly (one conversion for a pair: 1.6 cycles of an SM for the 128 values of a warp's word,
//     against 3.6 by shifts to bf16). The scale of a key multiplies its score. The scale of a value multiplies
//     its weight, over a power of two above all scales met so far, for fp16's range again.
//
// Work split: the 16-token tiles of all sequences form one sequence of tiles, cut into equal shares, one per
// warp; a share that ends inside a sequence leaves a partial (m, l, O) for the merge kernel.
#include <algorithm>
#include <cfloat>

#include <cuda_fp16.h>

#include "common.cuh"

namespace {

constexpr int TILE = 16;
constexpr int WARPS = 4, THREADS = WARPS * 32;

struct Cache {
  const unsigned char* data;
  const float* scale;
  int64_t page, slot, head;               // strides in bytes
  int64_t scale_page, scale_slot, scale_head;   // in elements
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
  int shares;        // warps along the tiles
};

// Entries for the merge, as in the split of the other decode kernels: {sequence, first share, shares}, one per
// sequence where there are no more sequences than shares (a partial lies in slot sequence + share), otherwise one per
// share, for the sequence that starts in it and goes on (slot 2 share, the first one of a sequence 2 share + 1).
__device__ __forceinline__ int2 cut_entry(int b, int first, int n) { return make_int2(b, first | n << 16); }

struct Span {          // visible tokens of a sequence
  int lo, hi;
  __device__ __forceinline__ int first_tile() const { return lo / TILE; }
  __device__ __forceinline__ int tiles() const { return hi > lo ? (hi + TILE - 1) / TILE - lo / TILE : 0; }
};
__device__ __forceinline__ Span span_of(const Params& p, int b) {
  const int64_t most = min((int64_t)p.max_pages * p.page_size, (int64_t)0x7fffff00);   // tiles end in 32 bits
  Span s;
  s.hi = p.num_pages > 0 ? (int)min((int64_t)max(0, p.lens[b]), most) : 0;
  s.lo = p.window > 0 ? max(0, s.hi - p.window) : 0;
  return s;
}

struct Share {
  int row, skip, left, per;
};
// Every warp finds its own share; called by the whole CTA. s: WARPS + 2 WARPS ints. `empty(r)` is called by one
// thread of the CTA with r % ctas == cta for a row without tiles.
template <class Tiles, class Empty>
__device__ __forceinline__ Share find_share(int nrows, int index, int shares, int cta, int ctas, int* s, Tiles tiles, Empty empty) {
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
  int* s_row = s + WARPS;
  int* s_skip = s_row + WARPS;
  int first = 0, mine = 0;
  for (int r = tid; r < nrows; r += THREADS) {
    const int n = tiles(r);
    if (r == tid) first = n;
    if (n == 0 && r % ctas == cta) empty(r);
    mine += n;
  }
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, off);
  if (lane == 0) s[w] = mine;
  if (lane == 0) s_row[w] = -1;
  __syncthreads();
  int total = 0;
#pragma unroll
  for (int i = 0; i < WARPS; ++i) total += s[i];
  Share sh = {0, 0, 0, max(1, (total + shares - 1) / shares)};
  // `begin` of the four warps: index is that of this warp, the CTA's lowest is warp 0's
  __shared__ int s_begin[WARPS];
  if (lane == 0) s_begin[w] = (int64_t)index * sh.per < total ? index * sh.per : -1;
  __syncthreads();
  int begin[WARPS], last = -1;
#pragma unroll
  for (int i = 0; i < WARPS; ++i) {
    begin[i] = s_begin[i];
    last = max(last, begin[i]);
  }
  if (last < 0) return sh;
  int base = 0;
  for (int r0 = 0; r0 < nrows && base <= last; r0 += THREADS) {
    const int r = r0 + tid;
    const int n = (r0 == 0) ? first : (r < nrows) ? tiles(r) : 0;
    int x = n;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, x, off);
      if (lane >= off) x += up;
    }
    __syncthreads();
    if (lane == 31) s[w] = x;
    __syncthreads();
    x += base;
#pragma unroll
    for (int i = 0; i < WARPS; ++i) {
      if (i < w) x += s[i];
      base += s[i];
    }
#pragma unroll
    for (int i = 0; i < WARPS; ++i)
      if (x - n <= begin[i] && begin[i] < x) {
        s_row[i] = r;
        s_skip[i] = begin[i] - (x - n);
      }
  }
  __syncthreads();
  if (begin[w] >= 0 && s_row[w] >= 0) {
    sh.row = s_row[w];
    sh.skip = s_skip[w];
    sh.left = min(sh.per, total - begin[w]);
  }
  return sh;
}

__device__ __forceinline__ uint4 ld16(const unsigned char* p) {
  uint4 r;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(p));
  return r;
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
// e with 2^e <= x < 2^(e + 1), within [-120, 120]
__device__ __forceinline__ int exponent(float x) { return min(max(((int)(__float_as_uint(x) >> 23) & 0xff) - 127, -120), 120); }

// A weight as hi + lo, both of its sign and neither zero where it is not.
template <class T>
__device__ __forceinline__ void two_pieces(float p0, float p1, uint32_t& hi, uint32_t& lo);
template <>
__device__ __forceinline__ void two_pieces<__nv_bfloat16>(float p0, float p1, uint32_t& hi, uint32_t& lo) {
  hi = __byte_perm(__float_as_uint(p0), __float_as_uint(p1), 0x7632);   // cut
  const float r0 = p0 - ako::bf16_lo(hi), r1 = p1 - ako::bf16_hi(hi);
  lo = ako::pack_bf16x2(r0 == 0.f ? p0 * 0x1p-16f : r0, r1 == 0.f ? p1 * 0x1p-16f : r1);
}
template <>
__device__ __forceinline__ void two_pieces<__half>(float p0, float p1, uint32_t& hi, uint32_t& lo) {
  __half2 h = __halves2half2(__float2half_rz(p0), __float2half_rz(p1));
  hi = *reinterpret_cast<uint32_t*>(&h);
  const float2 c = __half22float2(h);
  const float r0 = p0 == 0.f ? 0.f : copysignf(fmaxf(fabsf(p0 - c.x), 0x1p-24f), p0);
  const float r1 = p1 == 0.f ? 0.f : copysignf(fmaxf(fabsf(p1 - c.y), 0x1p-24f), p1);
  __half2 l = __floats2half2_rn(r0, r1);
  lo = *reinterpret_cast<uint32_t*>(&l);
}

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

template <int D, bool FP8>
constexpr int ctas_per_sm() { return D == 256 ? 2 : 3; }

template <class T, int D, bool FP8>
__global__ void __launch_bounds__(THREADS, (ctas_per_sm<D, FP8>())) paged_decode_kernel(const Params p) {
  constexpr int EB = FP8 ? 1 : 2;                  // bytes of a cache element
  constexpr int NJ = D * EB / 64;                  // pieces per lane and token
  constexpr int KS = D / 16;                       // steps of 16 features
  using TM = typename std::conditional<FP8, __half, T>::type;   // operand type
  constexpr float LIFT = std::is_same<TM, __half>::value ? 15.f : 0.f;
  __shared__ int s_scan[3 * WARPS];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  ako::pdl_trigger();
  // per_cta neighbouring (KV head, block) pairs of the same tokens, and WARPS / per_cta neighbouring shares
  const int cta = blockIdx.x / p.unit_ctas, unit = (blockIdx.x % p.unit_ctas) * p.per_cta + warp % p.per_cta;
  const int along = WARPS / p.per_cta;
  const int share = cta * along + warp / p.per_cta;
  const int kvh = unit / p.head_blocks, h0 = (unit % p.head_blocks) * 8;      // first head of the block in its group
  const int heads = min(8, p.group - h0), head0 = kvh * p.group + h0;
  const bool by_share = p.batch > p.shares;
  const bool keeper = unit == 0 && lane == 0;
  const Share sh0 = find_share(p.batch, share, p.shares, blockIdx.x, gridDim.x, s_scan, [&](int r) { return span_of(p, r).tiles(); },
                               [&](int r) {
                                 for (int h = 0; h < p.q_heads; ++h) empty_head<T, D>(p, (int64_t)r * p.q_heads + h);
                                 if (!by_share) p.cut[r] = cut_entry(r, 0, 0);
                               });
  int2 cut = cut_entry(0, 0, 0);
  int left = sh0.left, b = sh0.row, skip = sh0.skip;

  const unsigned char* kbase = p.k.data + kvh * p.k.head + t * 16;
  const unsigned char* vbase = p.v.data + kvh * p.v.head + t * 16;
  while (left > 0) {
    const Span sp = span_of(p, b);
    const int tiles = sp.tiles(), tile0 = sp.first_tile();
    const int te = min(tiles, skip + left);
    if (te <= skip) {                               // an empty sequence
      ++b;
      skip = 0;
      continue;
    }
    left -= te - skip;
    const int32_t* pages = p.table + (int64_t)b * p.max_pages;

    // this lane's two tokens of a tile (past the end: the last one, masked below); page -1: not visible
    int id[2], slot[2];
    auto fetch_ids = [&](int tile) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int tok = min((tile0 + tile) * TILE + 8 * i + g, sp.hi - 1);
        const int page = p.page_shift >= 0 ? tok >> p.page_shift : (int)((unsigned)tok / (unsigned)p.page_size);
        slot[i] = tok - page * p.page_size;
        id[i] = __ldg(pages + page);
      }
    };
    int64_t koff[2], voff[2];
    float ks[2] = {1.f, 1.f}, vs[2] = {1.f, 1.f};
    bool seen[2];
    auto locate = [&](int tile) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int tok = (tile0 + tile) * TILE + 8 * i + g;
        const bool real = (unsigned)id[i] < (unsigned)p.num_pages;
        const int64_t page = real ? id[i] : 0;
        seen[i] = real && tok >= sp.lo && tok < sp.hi;
        koff[i] = page * p.k.page + slot[i] * p.k.slot;
        voff[i] = page * p.v.page + slot[i] * p.v.slot;
        if (FP8) {
          ks[i] = __ldg(p.k.scale + page * p.k.scale_page + slot[i] * p.k.scale_slot + kvh * p.k.scale_head);
          vs[i] = __ldg(p.v.scale + page * p.v.scale_page + slot[i] * p.v.scale_slot + kvh * p.v.scale_head);
        }
      }
    };
    uint4 kc[2][NJ], vc[2][NJ];
    auto load = [&](uint4 (&x)[2][NJ], const unsigned char* base, const int64_t (&off)[2]) {
#pragma unroll
      for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int i = 0; i < 2; ++i) x[i][j] = ld16(base + off[i] + 64 * j);
    };

    // q of the block's heads as B fragments (n = head g), in the order of the K pieces
    uint32_t qb[KS][2];
#pragma unroll
    for (int i = 0; i < KS; ++i) qb[i][0] = qb[i][1] = 0u;
    if (g < heads) {
      const unsigned char* qp = (const unsigned char*)p.q + ((int64_t)b * p.q_heads + head0 + g) * D * 2;
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        if (FP8) {                                  // 16 features, a word of K has four
          const uint4 x = __ldg(reinterpret_cast<const uint4*>(qp + (64 * j + 16 * t) * 2));
          const uint4 y = __ldg(reinterpret_cast<const uint4*>(qp + (64 * j + 16 * t + 8) * 2));
          const uint32_t w[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            qb[4 * j + i][0] = w[2 * i];
            qb[4 * j + i][1] = w[2 * i + 1];
          }
        } else {
          const uint4 x = __ldg(reinterpret_cast<const uint4*>(qp + (32 * j + 8 * t) * 2));
          qb[2 * j][0] = x.x;
          qb[2 * j][1] = x.y;
          qb[2 * j + 1][0] = x.z;
          qb[2 * j + 1][1] = x.w;
        }
      }
    }
    float qs0 = p.scale_log2, qs1 = p.scale_log2;   // of heads 2t and 2t + 1
    if (FP8 && std::is_same<T, __nv_bfloat16>::value) {
      // bf16 to fp16: times the power of two that brings the head's largest element to [1, 2). What falls below
      // the fp16 range is off by 2^-25 of that.
      float top = 0.f;
#pragma unroll
      for (int i = 0; i < KS; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) top = fmaxf(top, fmaxf(fabsf(ako::bf16_lo(qb[i][j])), fabsf(ako::bf16_hi(qb[i][j]))));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const int e = exponent(top);
      const float down = power_of_two(-e), back = power_of_two(e);
#pragma unroll
      for (int i = 0; i < KS; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) qb[i][j] = pack2<__half>(ako::bf16_lo(qb[i][j]) * down, ako::bf16_hi(qb[i][j]) * down);
      qs0 *= __shfl_sync(0xffffffffu, back, 8 * t);
      qs1 *= __shfl_sync(0xffffffffu, back, 8 * t + 4);
    }
    // e4m3: the weights of P times their scales, over 2^unit > all scales met so far, are what goes into the product
    int unit_v = -121;
    float over = 0.f, under = 0.f;                  // 2^unit, 2^-unit
    // acc[i]: rows g and g + 8 of O^T step i, heads 2t and 2t + 1
    float acc[KS][4];
#pragma unroll
    for (int i = 0; i < KS; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][j] = 0.f;
    // The maxima start at the lowest finite value, so that a score of -inf weighs 0 whatever else there is.
    float m0 = -FLT_MAX, m1 = -FLT_MAX, l0 = 0.f, l1 = 0.f;

    fetch_ids(skip);
    locate(skip);
    load(kc, kbase, koff);
    load(vc, vbase, voff);
    fetch_ids(skip + 1);
    for (int tile = skip; tile < te; ++tile) {
      float s[2][4] = {};
      float s2[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        if (FP8) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint32_t a[4];
            widen(word(kc[0][j], i), a[0], a[2]);
            widen(word(kc[1][j], i), a[1], a[3]);
            mma<TM>(s[i & 1], a, qb[4 * j + i][0], qb[4 * j + i][1]);
          }
        } else {
          const uint32_t a0[4] = {kc[0][j].x, kc[1][j].x, kc[0][j].y, kc[1][j].y};
          const uint32_t a1[4] = {kc[0][j].z, kc[1][j].z, kc[0][j].w, kc[1][j].w};
          mma<TM>(s[0], a0, qb[2 * j][0], qb[2 * j][1]);
          mma<TM>(s[1], a1, qb[2 * j + 1][0], qb[2 * j + 1][1]);
        }
      }
      const bool v0 = seen[0], v1 = seen[1];
      const float k0 = ks[0], k1 = ks[1], w0 = vs[0], w1 = vs[1];
      const bool more = tile + 1 < te;
      if (more) {
        locate(tile + 1);
        load(kc, kbase, koff);
      }
      // rows g and g + 8, columns 2t and 2t + 1
      s2[0] = v0 ? (s[0][0] + s[1][0]) * (FP8 ? qs0 * k0 : qs0) : -INFINITY;
      s2[1] = v0 ? (s[0][1] + s[1][1]) * (FP8 ? qs1 * k0 : qs1) : -INFINITY;
      s2[2] = v1 ? (s[0][2] + s[1][2]) * (FP8 ? qs0 * k1 : qs0) : -INFINITY;
      s2[3] = v1 ? (s[0][3] + s[1][3]) * (FP8 ? qs1 * k1 : qs1) : -INFINITY;
      float n0 = fmaxf(s2[0], s2[2]), n1 = fmaxf(s2[1], s2[3]);
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
      float e[4];
      e[0] = ako::fast_exp2(s2[0] - m0 + LIFT);
      e[1] = ako::fast_exp2(s2[1] - m1 + LIFT);
      e[2] = ako::fast_exp2(s2[2] - m0 + LIFT);
      e[3] = ako::fast_exp2(s2[3] - m1 + LIFT);
      l0 += e[0] + e[2];
      l1 += e[1] + e[3];
      if (!(v0 && v1)) {   // weight 0, but what is read in its place may hold anything
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
          if (!v0) vc[0][j] = make_uint4(0u, 0u, 0u, 0u);
          if (!v1) vc[1][j] = make_uint4(0u, 0u, 0u, 0u);
        }
      }
      if (FP8) {
        const float a0 = v0 ? w0 : 0.f, a1 = v1 ? w1 : 0.f;
        if (__any_sync(0xffffffffu, fabsf(a0) >= over || fabsf(a1) >= over)) {
          float top = fmaxf(fabsf(a0), fabsf(a1));
#pragma unroll
          for (int o = 4; o <= 16; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
          const int u = max(unit_v, exponent(top) + 1);
          if (u != unit_v) {
            const float f = unit_v == -121 ? 0.f : power_of_two(max(unit_v - u, -126));
#pragma unroll
            for (int i = 0; i < KS; ++i)
#pragma unroll
              for (int j = 0; j < 4; ++j) acc[i][j] *= f;
            unit_v = u;
            over = power_of_two(u);
            under = power_of_two(-u);
          }
        }
        e[0] *= a0 * under;
        e[1] *= a0 * under;
        e[2] *= a1 * under;
        e[3] *= a1 * under;
      }
      uint32_t h0p, h1p, l0p, l1p;
      two_pieces<TM>(e[0], e[1], h0p, l0p);
      two_pieces<TM>(e[2], e[3], h1p, l1p);
      const uint32_t b0 = ako::movmatrix_trans(h0p), b1 = ako::movmatrix_trans(h1p);
      const uint32_t c0 = ako::movmatrix_trans(l0p), c1 = ako::movmatrix_trans(l1p);
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        if (FP8) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint32_t x0, y0, x1, y1;
            widen(word(vc[0][j], i), x0, y0);
            widen(word(vc[1][j], i), x1, y1);
            const uint32_t a[4] = {ako::movmatrix_trans(x0), ako::movmatrix_trans(y0), ako::movmatrix_trans(x1), ako::movmatrix_trans(y1)};
            mma<TM>(acc[4 * j + i], a, c0, c1);
            mma<TM>(acc[4 * j + i], a, b0, b1);
          }
        } else {
          const uint32_t a0[4] = {ako::movmatrix_trans(vc[0][j].x), ako::movmatrix_trans(vc[0][j].y), ako::movmatrix_trans(vc[1][j].x), ako::movmatrix_trans(vc[1][j].y)};
          const uint32_t a1[4] = {ako::movmatrix_trans(vc[0][j].z), ako::movmatrix_trans(vc[0][j].w), ako::movmatrix_trans(vc[1][j].z), ako::movmatrix_trans(vc[1][j].w)};
          mma<TM>(acc[2 * j], a0, c0, c1);
          mma<TM>(acc[2 * j], a0, b0, b1);
          mma<TM>(acc[2 * j + 1], a1, c0, c1);
          mma<TM>(acc[2 * j + 1], a1, b0, b1);
        }
      }
      if (more) {
        load(vc, vbase, voff);
        fetch_ids(tile + 2);
      }
    }
#pragma unroll
    for (int o = 4; o <= 16; o <<= 1) {
      l0 += __shfl_xor_sync(0xffffffffu, l0, o);
      l1 += __shfl_xor_sync(0xffffffffu, l1, o);
    }

    if (FP8) {
#pragma unroll
      for (int i = 0; i < KS; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] *= over;
    }
    const bool whole = te - skip == tiles;
    const float i0 = !whole ? 1.f : l0 == 0.f ? 0.f : 1.f / l0, i1 = !whole ? 1.f : l1 == 0.f ? 0.f : 1.f / l1;
    const int64_t at = by_share ? 2 * (int64_t)share + (skip == 0) : (int64_t)b + share;
    if (skip == 0) {
      cut = cut_entry(b, share, whole ? 1 : 1 + (tiles - te + sh0.per - 1) / sh0.per);
      if (!by_share && keeper) p.cut[b] = cut;
    }
#pragma unroll
    for (int hh = 0; hh < 2; ++hh) {
      if (2 * t + hh < heads) {
        const int head = head0 + 2 * t + hh;
        const float inv = hh ? i1 : i0;
        // an operand register has two neighbouring features, the next one the two behind them
#pragma unroll
        for (int i = 0; i < KS; ++i) {
          const float a = acc[i][hh] * inv, c = acc[i][2 + hh] * inv;
          const int col = FP8 ? 64 * (i / 4) + 16 * (g >> 1) + 4 * (i % 4) + (g & 1)
                              : 32 * (i / 2) + 8 * (g >> 1) + 4 * (i % 2) + (g & 1);
          if (whole) {
            T* op = (T*)p.o + ((int64_t)b * p.q_heads + head) * D + col;
            op[0] = (T)a;
            op[2] = (T)c;
          } else {
            float* op = p.part_acc + (at * p.q_heads + head) * D + col;
            op[0] = a;
            op[2] = c;
          }
        }
        if (g == 0) {
          const float m = hh ? m1 : m0, l = hh ? l1 : l0;
          if (whole)
            p.lse[(int64_t)b * p.q_heads + head] = l == 0.f ? -INFINITY : (m - LIFT) + log2f(l);
          else
            *reinterpret_cast<float2*>(p.part_ml + (at * p.q_heads + head) * 2) = make_float2(m - LIFT, l);
        }
      }
    }
    ++b;
    skip = 0;
  }
  if (by_share && keeper) p.cut[share] = cut;
}

// Merge: WARPS_PER warps per (sequence, head), each of them every WARPS_PER-th run of 32 partials; lanes hold columns.
template <class T, int D, int WARPS_PER>
__global__ void __launch_bounds__(WARPS_PER == 1 ? 128 : WARPS_PER * 32) paged_merge_kernel(const Params p) {
  constexpr int C = D / 32;                         // columns per lane
  __shared__ float s_acc[WARPS_PER][D];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int64_t job = WARPS_PER == 1 ? (int64_t)blockIdx.x * 4 + w : blockIdx.x;
  const int entries = min(p.batch, p.shares);
  ako::pdl_wait();
  if (job >= (int64_t)entries * p.q_heads) return;
  const int head = (int)(job % p.q_heads), part = WARPS_PER == 1 ? 0 : w;
  const int2 cut = p.cut[job / p.q_heads];
  const int c0 = cut.y & 0xffff, n = (unsigned)cut.y >> 16;
  if (n <= 1) return;
  const bool by_share = p.batch > p.shares;
  const int64_t slot0 = by_share ? 2 * (int64_t)c0 : (int64_t)cut.x + c0;
  auto slot = [&](int i) { return slot0 + (by_share ? 2 * i + (i == 0) : i); };
  auto ml = [&](int i) { return *reinterpret_cast<const float2*>(p.part_ml + (slot(i) * p.q_heads + head) * 2); };
  // every warp finds the maximum and the sum over all partials
  float M = -FLT_MAX;
  for (int i = lane; i < n; i += 32) M = fmaxf(M, ml(i).x);
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
  float L = 0.f, acc[C];
#pragma unroll
  for (int c = 0; c < C; ++c) acc[c] = 0.f;
  for (int i0 = 0; i0 < n; i0 += 32) {
    float wgt = 0.f;
    if (i0 + lane < n) {
      const float2 x = ml(i0 + lane);
      wgt = exp2f(x.x - M);
      L = fmaf(x.y, wgt, L);
    }
    if ((i0 / 32) % WARPS_PER != part) continue;
    const int k1 = min(32, n - i0);
#pragma unroll 4
    for (int k = 0; k < k1; ++k) {
      const float f = __shfl_sync(0xffffffffu, wgt, k);
      const float* x = p.part_acc + (slot(i0 + k) * p.q_heads + head) * D + lane * C;
      float y[C];
      if (C == 2) *reinterpret_cast<float2*>(y) = *reinterpret_cast<const float2*>(x);
      else
#pragma unroll
        for (int c = 0; c < C; c += 4) *reinterpret_cast<float4*>(y + c) = *reinterpret_cast<const float4*>(x + c);
#pragma unroll
      for (int c = 0; c < C; ++c) acc[c] = fmaf(y[c], f, acc[c]);
    }
  }
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) L += __shfl_xor_sync(0xffffffffu, L, o);
  if (WARPS_PER > 1) {
#pragma unroll
    for (int c = 0; c < C; ++c) s_acc[w][lane * C + c] = acc[c];
    __syncthreads();
    if (w != 0) return;
#pragma unroll
    for (int i = 1; i < WARPS_PER; ++i)
#pragma unroll
      for (int c = 0; c < C; ++c) acc[c] += s_acc[i][lane * C + c];
  }
  const float inv = L == 0.f ? 0.f : 1.f / L;
  const int64_t oi = (int64_t)cut.x * p.q_heads + head;
  uint32_t* op = reinterpret_cast<uint32_t*>((T*)p.o + oi * D + lane * C);
#pragma unroll
  for (int c = 0; c < C; c += 2) op[c / 2] = pack2<T>(acc[c] * inv, acc[c + 1] * inv);
  if (lane == 0) p.lse[oi] = L == 0.f ? -INFINITY : M + log2f(L);
}

struct Plan {
  int head_blocks, per_cta, unit_ctas, along;
  int shares, ctas;
  size_t ml, acc, total;   // offsets in the workspace; the entries are first
};
Plan plan_for(int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t dim, int64_t max_pages, int64_t page_size, int64_t window) {
  Plan pl;
  pl.head_blocks = (int)ako::cdiv(q_heads / kv_heads, (int64_t)8);
  const int64_t units = kv_heads * pl.head_blocks;
  pl.per_cta = units % 4 == 0 ? 4 : units % 2 == 0 ? 2 : 1;
  pl.unit_ctas = (int)(units / pl.per_cta);
  pl.along = WARPS / pl.per_cta;
  // All CTAs resident at once, and a tile at least for a warp. What the lengths are is known on the device only.
  const int64_t resident = (int64_t)ako::sm_count() * (dim == 256 ? 2 : 3);
  int64_t tokens = max_pages * page_size;
  if (window > 0 && tokens > window + TILE) tokens = window + TILE;
  const int64_t tiles = batch * ako::cdiv(tokens, (int64_t)TILE);
  int64_t ctas = std::max<int64_t>(1, resident / pl.unit_ctas);
  ctas = std::min(ctas, std::max<int64_t>(1, ako::cdiv(tiles, (int64_t)pl.along)));
  ctas = std::min<int64_t>(ctas, 32767 / pl.along);   // a merge entry has 15 bits for it
  pl.ctas = (int)ctas;
  pl.shares = pl.ctas * pl.along;
  const int64_t entries = std::min<int64_t>(batch, pl.shares), slots = entries + pl.shares;
  pl.ml = (entries * sizeof(int2) + 255) / 256 * 256;
  pl.acc = pl.ml + ((size_t)slots * q_heads * 8 + 255) / 256 * 256;
  pl.total = pl.acc + (size_t)slots * q_heads * dim * 4;
  return pl;
}
bool sizes_ok(int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t dim, int64_t max_pages, int64_t page_size, int64_t window) {
  const int64_t most = 0x7fffffffLL;
  return batch >= 0 && batch < most && q_heads > 0 && kv_heads > 0 && q_heads <= (1 << 16) && q_heads % kv_heads == 0 && page_size >= 1 &&
         page_size < most && max_pages >= 0 && max_pages < most && window >= 0 && (dim == 64 || dim == 128 || dim == 256);
}

template <class T, int D, bool FP8>
int launch(const Params& p, const Plan& pl, cudaStream_t st) {
  paged_decode_kernel<T, D, FP8><<<(unsigned)(pl.ctas * pl.unit_ctas), THREADS, 0, st>>>(p);
  AKO_CHECK_LAUNCH();
  if (pl.shares == 1) return AKO4X_OK;
  const int64_t jobs = (int64_t)std::min(p.batch, p.shares) * p.q_heads;
  const bool many = p.shares >= 64LL * p.batch;     // partials of a sequence
  const cudaError_t e = many ? ako::launch_pdl(true, paged_merge_kernel<T, D, 8>, dim3((unsigned)jobs), dim3(256), 0, st, p)
                             : ako::launch_pdl(true, paged_merge_kernel<T, D, 1>, dim3((unsigned)ako::cdiv(jobs, (int64_t)4)), dim3(128), 0, st, p);
  return e == cudaSuccess ? AKO4X_OK : AKO4X_ELAUNCH;
}
template <class T, bool FP8>
int launch(const Params& p, const Plan& pl, int64_t dim, cudaStream_t st) {
  if (dim == 64) return launch<T, 64, FP8>(p, pl, st);
  if (dim == 128) return launch<T, 128, FP8>(p, pl, st);
  return launch<T, 256, FP8>(p, pl, st);
}

bool set_cache(Cache& c, const ako4x_kv_cache* in, bool fp8) {
  const int size = fp8 ? 1 : 2;
  c.data = (const unsigned char*)in->data;
  c.page = in->page_stride * size;
  c.slot = in->slot_stride * size;
  c.head = in->head_stride * size;
  c.scale = in->scale;
  c.scale_page = in->scale_page_stride;
  c.scale_slot = in->scale_slot_stride;
  c.scale_head = in->scale_head_stride;
  if (!in->data || (((uintptr_t)in->data | (uint64_t)c.page | (uint64_t)c.slot | (uint64_t)c.head) & 15)) return false;
  return !fp8 || (in->scale && ((uintptr_t)in->scale & 3) == 0);
}

}  // namespace

extern "C" size_t ako4x_paged_decode_workspace_bytes(int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t dim,
                                                     int64_t max_pages, int64_t page_size, int64_t window) {
  if (batch == 0 || !sizes_ok(batch, q_heads, kv_heads, dim, max_pages, page_size, window)) return 0;
  return plan_for(batch, q_heads, kv_heads, dim, max_pages, page_size, window).total;
}

extern "C" int ako4x_paged_decode(const void* q, const ako4x_kv_cache* k_cache, const ako4x_kv_cache* v_cache,
                                  const int32_t* block_table, const int32_t* seq_lens, float sm_scale, int64_t window, void* o,
                                  float* lse, int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t dim, int64_t num_pages,
                                  int64_t page_size, int64_t max_pages, int dtype, int cache_dtype, void* workspace,
                                  size_t workspace_bytes, void* stream) {
  if (batch < 0 || num_pages < 0 || num_pages > 0x7fffffffLL) return AKO4X_EINVAL;
  if (dtype != AKO4X_BF16 && dtype != AKO4X_FP16) return AKO4X_EUNSUPPORTED_SHAPE;
  if (cache_dtype != dtype && cache_dtype != AKO4X_E4M3) return AKO4X_EUNSUPPORTED_SHAPE;
  if (!sizes_ok(batch, q_heads, kv_heads, dim, max_pages, page_size, window)) return AKO4X_EUNSUPPORTED_SHAPE;
  if (batch == 0) return AKO4X_OK;
  if (!q || !k_cache || !v_cache || !seq_lens || !o || !lse || (max_pages > 0 && !block_table)) return AKO4X_EINVAL;
  if (((uintptr_t)q | (uintptr_t)o) & 15) return AKO4X_EINVAL;
  const bool fp8 = cache_dtype == AKO4X_E4M3;
  Params p = {};
  if ((!set_cache(p.k, k_cache, fp8) || !set_cache(p.v, v_cache, fp8)) && num_pages > 0) return AKO4X_EINVAL;
  const Plan pl = plan_for(batch, q_heads, kv_heads, dim, max_pages, page_size, window);
  if (!workspace || workspace_bytes < pl.total) return AKO4X_EWORKSPACE;
  if ((uintptr_t)workspace & 15) return AKO4X_EINVAL;
  unsigned char* ws = (unsigned char*)workspace;
  p.q = q;
  p.table = block_table;
  p.lens = seq_lens;
  p.o = o;
  p.lse = lse;
  p.cut = (int2*)ws;
  p.part_ml = (float*)(ws + pl.ml);
  p.part_acc = (float*)(ws + pl.acc);
  p.scale_log2 = sm_scale * AKO_LOG2E;
  p.batch = (int)batch;
  p.q_heads = (int)q_heads;
  p.kv_heads = (int)kv_heads;
  p.group = (int)(q_heads / kv_heads);
  p.head_blocks = pl.head_blocks;
  p.per_cta = pl.per_cta;
  p.unit_ctas = pl.unit_ctas;
  p.num_pages = (int)num_pages;
  p.page_size = (int)page_size;
  p.page_shift = (page_size & (page_size - 1)) == 0 ? __builtin_ctzll((unsigned long long)page_size) : -1;
  p.max_pages = (int)max_pages;
  p.window = (int)std::min<int64_t>(window, 0x7fffffff);
  p.shares = pl.shares;
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == AKO4X_BF16) return fp8 ? launch<__nv_bfloat16, true>(p, pl, dim, st) : launch<__nv_bfloat16, false>(p, pl, dim, st);
  return fp8 ? launch<__half, true>(p, pl, dim, st) : launch<__half, false>(p, pl, dim, st);
}
