// Rotary positions, and the RMS norm of every query and key head with the rotation in the same pass, the
// keys and values of the call stored into a paged cache if one is given.
//
//   y = x * rsqrt(mean(x^2) + eps) * w              (norm, optional)
//   z_a = y_a c - y_b s,  z_b = y_b c + y_a s       (a, b) = (i, i + R/2) or (2i, 2i + 1), i < R/2
//   c, s = m cos(pos f_i), m sin(pos f_i)
//
// Everything between the load and the one rounding of the result is fp32, but the angles: pos f_i has as
// many digits in front of the point as the position, so the product is taken in fp64, in turns
// (f_i / 2 pi), and its whole quarter turns are taken off there; what is left fits an fp32 sincospi to
// its last bits, for any position. In the norm the factors of a token are the same for all its heads: z = inv (x A + x' B)
// with x' the partner and A = w c, B = -+ w' s kept in registers.
//
// HBM-bound: every element is read and written once. 4, 8 or 16 lanes own a row, two pieces of 16 bytes each,
// and a lane's second piece holds the partners of its first: nothing is exchanged but the sum of the squares, and
// nothing is unpacked twice. A warp takes row groups of one token (all of them, or a share where there are few
// tokens), the loads two groups ahead; the token's R/2 angles are shared out over the lanes once.
// Interleaved pairs lie in one piece. Where R/2 is an odd multiple of 4, pieces of 8 bytes and twice the lanes put the
// partners into one lane; where it is no multiple of 4 the rotated elements go through shared memory, a pair to a lane
// (8 192 tokens of 40 rows of 64, 40 of them rotated: 60 us so, 18 with the smaller pieces; 5 007 tokens of 96 rows of 80,
// 40 rotated: 86 and 54. For all sizes the smaller pieces are not better: 48 us for the next paragraph's 45).
// Measured, 8 192 tokens with 32 + 8 + 8 heads of 128 into a bf16 cache (201 MB): one piece per lane and partners by
// shuffle 72 us; two pieces 61; grid without divisions, tables from whole vectors 51; loads ahead across the kinds of
// rows, 20 warps to an SM 43 to 45 (4.5 to 4.7 TB/s). The same without arithmetic 31. What is left is neither HBM (0.69 of the copy
// rate) nor issue slots (257 instructions for a row group, 0.58 of the rate): it is latency, of the loads first, that 20 warps do
// not cover, and five CTAs to an SM leave 96 registers a thread, of which the forms with pieces of 16 bytes spill 74 bytes (half
// pairs) or 98 (interleaved). Into an e4m3 cache (185 MB) 52, with 338 instructions a row group, sixteen divisions of a lane and row
// among them; without norms 44 and 49; rotation alone 36 (168 MB). Angles in shared memory for a CTA's tokens instead of tables in
// registers: 49 to 63; the next row's norm beside this row's rotation: 46; packed fp32 pairs (fma.rn.f32x2): the moves outweigh them.
#include <algorithm>

#include "common.cuh"

#include <cuda_fp16.h>

namespace {

constexpr int WARPS = 4;
constexpr int WARPS_TO_FILL = 20;   // of an SM
constexpr int MAX_DIM = 256;
constexpr int MAX_ANGLES = 256;   // of a warp: 256 / dim tokens at most, half of dim each, and room for odd numbers

struct Rows {                 // heads of one kind
  const unsigned char* in;
  int64_t token_stride, head_stride;   // bytes
  int heads;
  int groups;                 // warp instructions for a token
};
struct Cache {
  unsigned char* data;
  float* scale;
  int64_t page_stride, slot_stride, head_stride;              // bytes
  int64_t scale_page_stride, scale_slot_stride, scale_head_stride;   // elements
};
struct Params {
  Rows q, k, v;
  unsigned char* q_out;
  unsigned char* k_out;       // null: the cache
  const void* q_weight;       // null: no norm
  const void* k_weight;
  const void* positions;
  const void* slots;          // null: no cache
  const float* inv_freq;
  Cache kc, vc;
  int64_t tokens, num_slots;
  int dim, rotary, page_size;
  int per_share;              // groups of a warp
  int log_tokens;             // tokens of a warp, side by side
  float eps, inv_dim, factor;
  bool interleaved, positions64, slots64, weights32, quant, ragged;   // ragged: some lanes are behind the row's end
};

template <class T>
struct Pair;
template <>
struct Pair<__nv_bfloat16> {
  static __device__ __forceinline__ float2 get(uint32_t v) { return make_float2(ako::bf16_lo(v), ako::bf16_hi(v)); }
  static __device__ __forceinline__ uint32_t put(float a, float b) { return ako::pack_bf16x2(a, b); }
  static __device__ __forceinline__ float one(const void* p) { return __bfloat162float(*(const __nv_bfloat16*)p); }
};
template <>
struct Pair<__half> {
  static __device__ __forceinline__ float2 get(uint32_t v) { return __half22float2(*reinterpret_cast<__half2*>(&v)); }
  static __device__ __forceinline__ uint32_t put(float a, float b) {
    __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&v);
  }
  static __device__ __forceinline__ float one(const void* p) { return __half2float(*(const __half*)p); }
};

__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) { return make_float2(fmaf(a.x, b.x, c.x), fmaf(a.y, b.y, c.y)); }
__device__ __forceinline__ float2 mul2(float2 a, float2 b) { return make_float2(a.x * b.x, a.y * b.y); }

__device__ __forceinline__ float max_nan(float a, float b) {   // a NaN stays
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ uint32_t word(const uint4& v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }
__device__ __forceinline__ uint32_t word(const uint2& v, int i) { return i == 0 ? v.x : v.y; }

template <int ELEMENTS>   // of two bytes each
struct Words;
template <>
struct Words<8> {
  using Piece = uint4;
  static __device__ __forceinline__ void put_once(void* to, const uint32_t (&w)[4]) { __stcs((uint4*)to, make_uint4(w[0], w[1], w[2], w[3])); }
};
template <>
struct Words<4> {
  using Piece = uint2;
  static __device__ __forceinline__ void put(void* to, const uint32_t (&w)[2]) { *(uint2*)to = make_uint2(w[0], w[1]); }
  static __device__ __forceinline__ void put_once(void* to, const uint32_t (&w)[2]) { __stcs((uint2*)to, make_uint2(w[0], w[1])); }
};
template <>
struct Words<2> {
  static __device__ __forceinline__ void put(void* to, const uint32_t (&w)[1]) { *(uint32_t*)to = w[0]; }
};

// Where the partner of a rotated element is.
enum Partner { OTHER_PIECE, SAME_PIECE, STAGED };   // STAGED: anywhere, by way of shared memory

// PE: elements of a piece. CTAs to an SM: with the smaller pieces 5, 6, 7 take 64.9, 54.4, 66.4 us for 96 rows of 80.
template <class T, int LANES, Partner PARTNER, int PE>
__global__ void __launch_bounds__(WARPS * 32, PARTNER == STAGED ? 4 : PE == 8 ? 5 : 6) qk_norm_rope_kernel(const Params p) {
  using Piece = typename Words<PE>::Piece;
  constexpr int GROUP = 32 / LANES;   // rows of a warp instruction
  __shared__ __align__(16) float2 s_cs[WARPS][MAX_ANGLES];
  __shared__ __align__(16) float s_row[PARTNER == STAGED ? WARPS : 1][32 / LANES][PARTNER == STAGED ? LANES * 2 * PE : 1];
  ako::pdl_trigger();
  ako::pdl_wait();   // nothing before this reads what a kernel wrote, and no load below is of the read-only kind
  const int warp = threadIdx.x >> 5, lane32 = threadIdx.x & 31;
  const int lane = lane32 % LANES, slots = GROUP >> p.log_tokens;   // slots: rows of a token at once
  const int sub = lane32 / LANES & (slots - 1), mine = lane32 / LANES / slots;
  const int64_t first = ((int64_t)blockIdx.x * WARPS + warp) << p.log_tokens;
  if (first >= p.tokens) return;      // whole warps; there is no block barrier
  const int64_t token = min(first + mine, p.tokens - 1);
  const bool real = first + mine < p.tokens;
  const int end_q = p.q.groups, end_k = end_q + p.k.groups, end_v = end_k + p.v.groups;
  const int g0 = blockIdx.y * p.per_share, g1 = min(g0 + p.per_share, end_v);

  // this lane's two pieces of a row: the partners of each other in front; behind, the lanes' first pieces and then their
  // second ones, so that an instruction's bytes are one stretch (8 192 tokens of 17 rows of 64, pairs: 11.4 -> 11.0 us)
  const int half = p.rotary / 2, pitch = (half + 1) & ~1, paired = PARTNER == OTHER_PIECE ? p.rotary / (2 * PE) : 0;
  const int e0 = PE * (lane < paired ? lane : lane + paired), e1 = PE * (lane < paired ? lane + paired : lane + LANES);
  const bool in0 = e0 < p.dim, in1 = e1 < p.dim;

  // The loads run two row groups ahead, from one kind into the next. A lane past the last row, or past the row's
  // end, reads what another one does.
  int at = g0, at_kind = g0 < end_q ? 0 : g0 < end_k ? 1 : 2, at_stop, at_head, at_heads;
  const unsigned char *from0, *from1;
  int64_t step;
  Piece raw[2][2];
  auto aim = [&] {
    const Rows& r = at_kind == 0 ? p.q : at_kind == 1 ? p.k : p.v;
    const int start = at_kind == 0 ? 0 : at_kind == 1 ? end_q : end_k;
    at_stop = min(g1, start + r.groups);
    at_head = (at - start) * slots + sub;
    at_heads = r.heads;
    from0 = r.in + token * r.token_stride + min(at_head, at_heads - 1) * r.head_stride;
    from1 = from0 + (in1 ? e1 * 2 : 0);
    from0 += in0 ? e0 * 2 : 0;
    step = slots * r.head_stride;
  };
  auto fetch = [&](Piece (&x)[2]) {
    if (at >= g1) return;
    x[0] = *reinterpret_cast<const Piece*>(from0);
    x[1] = *reinterpret_cast<const Piece*>(from1);
    if (++at == at_stop) {
      if (at < g1) {
        at_kind = at < end_k ? 1 : 2;
        aim();
      }
    } else {
      at_head += slots;
      if (at_head < at_heads) {
        from0 += step;
        from1 += step;
      }
    }
  };
  aim();
  fetch(raw[0]);                      // under way while the angles are made
  fetch(raw[1]);
  auto next = [&] {                   // called when raw[0] has been taken
    raw[0][0] = raw[1][0], raw[0][1] = raw[1][1];
    fetch(raw[1]);
  };

  if (g0 < end_k) {
    for (int t = 0; t < 1 << p.log_tokens && first + t < p.tokens; ++t) {
      const double pos = p.positions64 ? (double)((const int64_t*)p.positions)[first + t] : (double)((const int32_t*)p.positions)[first + t];
      for (int i = lane32; i < half; i += 32) {
        double turn = pos * ((double)p.inv_freq[i] * 0.15915494309189533577);   // f / 2 pi
        turn -= rint(turn);
        // and the nearest quarter: sine and cosine are then both good to their last bits, next to their zeros too
        const double quarters = rint(turn * 4.0);
        float s, c;
        sincospif(2.0f * (float)(turn - quarters * 0.25), &s, &c);
        const int quadrant = (int)quarters & 3;
        const float x = quadrant & 1 ? -s : c, y = quadrant & 1 ? c : s;
        s_cs[warp][t * pitch + i] = make_float2((quadrant & 2 ? -x : x) * p.factor, (quadrant & 2 ? -y : y) * p.factor);
      }
    }
    __syncwarp();
  }
  int64_t page = 0;
  int slot = 0;
  bool stored = false;
  if (p.slots) {
    const int64_t at = p.slots64 ? ((const int64_t*)p.slots)[token] : (int64_t)((const int32_t*)p.slots)[token];
    stored = at >= 0 && at < p.num_slots;   // anything else: a padding token, its keys and values go nowhere
    if (stored) {
      page = p.num_slots <= 0xffffffffLL ? (int64_t)((unsigned)at / (unsigned)p.page_size) : at / p.page_size;
      slot = (int)(at - page * p.page_size);
    }
  }

  const float2* cs_of = s_cs[warp] + (real ? mine : 0) * pitch;
  // Pairs (2i, 2i + 1) of the pieces' elements: z = inv (x A + x' B), where `mask` says so; inv x A elsewhere.
  float2 A[2][PE / 2], B[2][PE / 2];
  unsigned mask = 0;
  auto tables = [&](const void* weight) {
    float w[2][PE];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int e = h ? e1 : e0;
#pragma unroll
      for (int j = 0; j < PE; ++j) w[h][j] = 1.f;
      if (weight && (h ? in1 : in0)) {
        if (p.weights32) {
#pragma unroll
          for (int j = 0; j < PE; j += 4) {
            const float4 y = *reinterpret_cast<const float4*>((const float*)weight + e + j);
            w[h][j] = y.x, w[h][j + 1] = y.y, w[h][j + 2] = y.z, w[h][j + 3] = y.w;
          }
        } else {
          const Piece x = *reinterpret_cast<const Piece*>((const T*)weight + e);
#pragma unroll
          for (int j = 0; j < PE / 2; ++j) {
            const float2 y = Pair<T>::get(word(x, j));
            w[h][2 * j] = y.x;
            w[h][2 * j + 1] = y.y;
          }
        }
      }
#pragma unroll
      for (int j = 0; j < PE / 2; ++j) {
        A[h][j] = make_float2(w[h][2 * j], w[h][2 * j + 1]);
        B[h][j] = make_float2(0.f, 0.f);
      }
    }
    mask = 0;
    if (PARTNER == OTHER_PIECE) {
      if (lane < paired) {            // the angles of both pieces
        mask = (1u << PE) - 1;
#pragma unroll
        for (int j = 0; j < PE / 2; ++j) {
          const float4 cs = *reinterpret_cast<const float4*>(cs_of + e0 + 2 * j);
          A[0][j] = make_float2(w[0][2 * j] * cs.x, w[0][2 * j + 1] * cs.z);
          A[1][j] = make_float2(w[1][2 * j] * cs.x, w[1][2 * j + 1] * cs.z);
          B[0][j] = make_float2(-w[1][2 * j] * cs.y, -w[1][2 * j + 1] * cs.w);
          B[1][j] = make_float2(w[0][2 * j] * cs.y, w[0][2 * j + 1] * cs.w);
        }
      }
    } else if (PARTNER == SAME_PIECE) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int j = 0; j < PE / 2; ++j) {
          const int e = (h ? e1 : e0) + 2 * j;
          if (e < p.rotary) {
            const float2 cs = cs_of[e / 2];
            mask |= 1u << (PE / 2 * h + j);
            A[h][j] = make_float2(w[h][2 * j] * cs.x, w[h][2 * j + 1] * cs.x);
            B[h][j] = make_float2(-w[h][2 * j + 1] * cs.y, w[h][2 * j] * cs.y);
          }
        }
    }
  };

  const bool all = PARTNER != STAGED && p.rotary == p.dim;   // every element is rotated
  bool ready = false;
#pragma unroll 1
  for (int it = g0; it < g1;) {       // a kind
    const int kind = it < end_q ? 0 : it < end_k ? 1 : 2, start = kind == 0 ? 0 : kind == 1 ? end_q : end_k;
    const Rows& r = kind == 0 ? p.q : kind == 1 ? p.k : p.v;
    const int heads = r.heads, stop = min(g1, start + r.groups);
    int head = (it - start) * slots + sub;
    const bool to_cache = kind == 2 || (kind == 1 && !p.k_out), turn = kind != 2;
    const void* weight = kind == 0 ? p.q_weight : kind == 1 ? p.k_weight : nullptr;
    if (turn && (weight || !ready)) {
      tables(weight);
      ready = weight == nullptr;
    }
    unsigned char* out;
    int64_t out_step;
    float* scale_out = nullptr;
    int64_t scale_step = 0;
    const bool quant = to_cache && p.quant;
    if (!to_cache) {
      out = (kind == 0 ? p.q_out : p.k_out) + (token * heads + head) * p.dim * 2;
      out_step = (int64_t)slots * p.dim * 2;
    } else {
      const Cache& c = kind == 1 ? p.kc : p.vc;
      out = c.data + page * c.page_stride + slot * c.slot_stride + head * c.head_stride;
      out_step = slots * c.head_stride;
      if (quant) {
        scale_out = c.scale + page * c.scale_page_stride + slot * c.scale_slot_stride + head * c.scale_head_stride;
        scale_step = slots * c.scale_head_stride;
      }
    }
    unsigned char *to0 = out + (quant ? e0 : e0 * 2), *to1 = out + (quant ? e1 : e1 * 2);
    const bool store = real && (!to_cache || stored);
    if (!turn && !quant) {            // values as they are
#pragma unroll 1
      for (; it < stop; ++it, head += slots, to0 += out_step, to1 += out_step) {
        const Piece x0 = raw[0][0], x1 = raw[0][1];
        next();
        if (store && head < heads && in0) __stcs(reinterpret_cast<Piece*>(to0), x0);
        if (store && head < heads && in1) __stcs(reinterpret_cast<Piece*>(to1), x1);
      }
    }
#pragma unroll 1
    for (; it < stop; ++it, head += slots, to0 += out_step, to1 += out_step) {
      const bool live = store && head < heads;
      float2 y[2][PE / 2];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int j = 0; j < PE / 2; ++j) y[h][j] = Pair<T>::get(word(raw[0][h], j));
      next();
      if (p.ragged) {                 // pieces behind the row's end
#pragma unroll
        for (int h = 0; h < 2; ++h)
          if (!(h ? in1 : in0)) {
#pragma unroll
            for (int j = 0; j < PE / 2; ++j) y[h][j] = make_float2(0.f, 0.f);
          }
      }
      if (turn) {
        float2 o[2][PE / 2];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int j = 0; j < PE / 2; ++j) {
            if (PARTNER == OTHER_PIECE) o[h][j] = y[1 - h][j];
            if (PARTNER == SAME_PIECE) o[h][j] = make_float2(y[h][j].y, y[h][j].x);
          }
        float inv = 1.f;
        if (weight) {
          float2 ss = mul2(y[0][0], y[0][0]), st = mul2(y[1][0], y[1][0]);
#pragma unroll
          for (int j = 1; j < PE / 2; ++j) {
            ss = fma2(y[0][j], y[0][j], ss);
            st = fma2(y[1][j], y[1][j], st);
          }
          float sum = (ss.x + ss.y) + (st.x + st.y);
#pragma unroll
          for (int m = LANES / 2; m >= 1; m >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, m);
          inv = rsqrtf(fmaf(sum, p.inv_dim, p.eps));
        }
        float2 z[2][PE / 2];
        if (PARTNER == STAGED) {            // a pair to a lane, and back
          float* staged = s_row[warp][lane32 / LANES];
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int j = 0; j < PE / 2; ++j) {
              z[h][j] = mul2(y[h][j], A[h][j]);
              const int e = (h ? e1 : e0) + 2 * j;
              if (e < p.rotary) *reinterpret_cast<float2*>(staged + e) = z[h][j];
            }
          __syncwarp();
          for (int i = lane; i < half; i += LANES) {
            const float2 cs = cs_of[i];
            const float a = staged[i], b = staged[i + half];
            staged[i] = fmaf(a, cs.x, -b * cs.y);
            staged[i + half] = fmaf(b, cs.x, a * cs.y);
          }
          __syncwarp();
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int j = 0; j < PE / 2; ++j) {
              const int e = (h ? e1 : e0) + 2 * j;
              if (e < p.rotary) z[h][j] = *reinterpret_cast<const float2*>(staged + e);
            }
          __syncwarp();                     // read before the next row is put there
        } else if (all) {
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int j = 0; j < PE / 2; ++j) z[h][j] = fma2(o[h][j], B[h][j], mul2(y[h][j], A[h][j]));
        } else {                            // an element that is not rotated takes nothing from another one
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int j = 0; j < PE / 2; ++j) {
              z[h][j] = mul2(y[h][j], A[h][j]);
              if (mask >> (PE / 2 * h + j) & 1) z[h][j] = fma2(o[h][j], B[h][j], z[h][j]);
            }
        }
        const float2 by = make_float2(inv, inv);
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int j = 0; j < PE / 2; ++j) y[h][j] = weight ? mul2(z[h][j], by) : z[h][j];
      }
      if (quant) {
        // e4m3 with the row's own scale: amax / 448, 1 for a row of (nearly) zeros
        float top = 0.f;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int j = 0; j < PE / 2; ++j) {
            const float2 x = y[h][j];
            top = max_nan(top, max_nan(fabsf(x.x), fabsf(x.y)));
          }
#pragma unroll
        for (int m = LANES / 2; m >= 1; m >>= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, m));
        const float sc = top <= 1e-10f ? 1.0f : __fdiv_rn(top, 448.0f);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t w[PE / 4] = {};
#pragma unroll
          for (int j = 0; j < PE / 2; ++j) {
            const float2 x = y[h][j];
            const uint32_t pair = __nv_cvt_float2_to_fp8x2(make_float2(__fdiv_rn(x.x, sc), __fdiv_rn(x.y, sc)), __NV_SATFINITE, __NV_E4M3);
            w[j >> 1] |= pair << (16 * (j & 1));
          }
          if (live && (h ? in1 : in0)) Words<PE / 2>::put(h ? to1 : to0, w);
        }
        if (live && lane == 0) *scale_out = sc;
        scale_out += scale_step;
      } else {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t w[PE / 2];
#pragma unroll
          for (int j = 0; j < PE / 2; ++j) {
            const float2 x = y[h][j];
            w[j] = Pair<T>::put(x.x, x.y);
          }
          if (live && (h ? in1 : in0)) Words<PE>::put_once(h ? to1 : to0, w);
        }
      }
    }
  }
}

// Elements of a piece: 8, or 4 where that puts the partners into one lane and 8 does not.
int piece_of(bool interleaved, int rotary) { return !interleaved && rotary % 16 == 8 ? 4 : 8; }

template <class T, int LANES>   // LANES: of a row, with pieces of 8
cudaError_t launch(const Params& p, dim3 blocks, cudaStream_t st) {
  const auto kernel = p.interleaved         ? qk_norm_rope_kernel<T, LANES, SAME_PIECE, 8>
                      : p.rotary % 16 == 0 ? qk_norm_rope_kernel<T, LANES, OTHER_PIECE, 8>
                      : p.rotary % 16 == 8 ? qk_norm_rope_kernel<T, 2 * LANES, OTHER_PIECE, 4>
                                           : qk_norm_rope_kernel<T, LANES, STAGED, 8>;
  return ako::launch_pdl(true, kernel, blocks, dim3(WARPS * 32), 0, st, p);
}
template <class T>
cudaError_t launch(const Params& p, dim3 blocks, cudaStream_t st) {
  return p.dim <= 64 ? launch<T, 4>(p, blocks, st) : p.dim <= 128 ? launch<T, 8>(p, blocks, st) : launch<T, 16>(p, blocks, st);
}

bool aligned(const void* ptr, int64_t a, int64_t b, int64_t c, int64_t to) {
  return ptr && (((uintptr_t)ptr | (uintptr_t)a | (uintptr_t)b | (uintptr_t)c) & (to - 1)) == 0;
}

int run(Params& p, const ako4x_head_rows* q, const ako4x_head_rows* k, const ako4x_head_rows* v, int64_t tokens, int64_t dim,
        int64_t rotary, int dtype, void* stream) {
  if (tokens < 0 || dim < 0 || rotary < 0) return AKO4X_EINVAL;
  if (dim < 8 || dim > MAX_DIM || dim % 8 || rotary > dim || rotary % 2) return AKO4X_EUNSUPPORTED_SHAPE;
  if (dtype != AKO4X_BF16 && dtype != AKO4X_FP16) return AKO4X_EUNSUPPORTED_SHAPE;
  const int padded = dim <= 64 ? 64 : dim <= 128 ? 128 : 256;   // elements of a row with those behind its end
  const int group = 32 * 2 * piece_of(p.interleaved, (int)rotary) / padded;
  const ako4x_head_rows* in[3] = {q, k, v};
  Rows* to[3] = {&p.q, &p.k, &p.v};
  bool any = false;
  for (int i = 0; i < 3; ++i) {
    *to[i] = Rows{};
    if (!in[i]) continue;
    if (in[i]->heads < 0 || in[i]->heads > (1 << 20)) return AKO4X_EINVAL;
    if (tokens == 0 || in[i]->heads == 0) continue;
    if (!aligned(in[i]->data, in[i]->token_stride * 2, in[i]->head_stride * 2, 0, 16)) return AKO4X_EINVAL;
    to[i]->in = (const unsigned char*)in[i]->data;
    to[i]->token_stride = in[i]->token_stride * 2;
    to[i]->head_stride = in[i]->head_stride * 2;
    to[i]->heads = (int)in[i]->heads;
    any = true;
  }
  if (!any) return AKO4X_OK;
  if (!p.positions || (rotary && !p.inv_freq)) return AKO4X_EINVAL;
  if (p.q.heads && !aligned(p.q_out, 0, 0, 0, 16)) return AKO4X_EINVAL;
  if (((uintptr_t)p.q_weight | (uintptr_t)p.k_weight) & 15) return AKO4X_EINVAL;
  if (((uintptr_t)p.inv_freq & 3) || ((uintptr_t)p.positions & (p.positions64 ? 7 : 3)) || ((uintptr_t)p.slots & (p.slots64 ? 7 : 3)))
    return AKO4X_EINVAL;
  p.tokens = tokens;
  p.dim = (int)dim;
  p.rotary = (int)rotary;
  p.inv_dim = 1.0f / (float)dim;
  p.ragged = dim != padded;
  // A warp takes a token's rows; several tokens side by side, as long as there are warps for the GPU, where a token has few
  // (what is done once for a token weighs more then: 8 192 tokens of 17 rows of 64 12.8 -> 11.3 us; with 48 rows of 128
  // 44.7 -> 51.6, the warps are fewer and longer); or a share of the rows while there are fewer warps than the GPU holds.
  int64_t row_groups = 0;
  for (const Rows* r : to) row_groups += ako::cdiv(r->heads, group);
  while (row_groups <= 4 && (group >> p.log_tokens) > 1 && (tokens >> (p.log_tokens + 1)) >= ako::sm_count() * WARPS_TO_FILL) ++p.log_tokens;
  int64_t groups = 0;
  for (Rows* r : to) {
    r->groups = (int)ako::cdiv(r->heads, group >> p.log_tokens);
    groups += r->groups;
  }
  const int64_t wanted = (int64_t)ako::sm_count() * 48;   // more than fit, so that the shares are small: 969 tokens 9.4 -> 8.1 us
  int64_t shares = std::min(ako::cdiv(wanted, tokens), groups);
  p.per_share = (int)ako::cdiv(groups, shares);
  shares = ako::cdiv(groups, (int64_t)p.per_share);
  const int64_t blocks = ako::cdiv(tokens, (int64_t)WARPS << p.log_tokens);
  if (blocks > 0x7fffffffLL || shares > 65535 || groups > 0x3fffffffLL) return AKO4X_ETOOLARGE;
  const dim3 grid((unsigned)blocks, (unsigned)shares);
  cudaStream_t st = (cudaStream_t)stream;
  const cudaError_t e = dtype == AKO4X_BF16 ? launch<__nv_bfloat16>(p, grid, st) : launch<__half>(p, grid, st);
  return e == cudaSuccess ? AKO4X_OK : AKO4X_ELAUNCH;
}

Params common(const void* positions, int positions_int64, const float* inv_freq, int interleaved, float factor, void* q_out,
              void* k_out) {
  Params p = {};
  p.positions = positions;
  p.positions64 = positions_int64 != 0;
  p.inv_freq = inv_freq;
  p.interleaved = interleaved != 0;
  p.factor = factor;
  p.q_out = (unsigned char*)q_out;
  p.k_out = (unsigned char*)k_out;
  return p;
}

bool set_cache(Cache& c, const ako4x_kv_cache* in, int cache_dtype) {
  const int size = cache_dtype == AKO4X_E4M3 ? 1 : 2;
  c.data = (unsigned char*)in->data;
  c.page_stride = in->page_stride * size;
  c.slot_stride = in->slot_stride * size;
  c.head_stride = in->head_stride * size;
  c.scale = in->scale;
  c.scale_page_stride = in->scale_page_stride;
  c.scale_slot_stride = in->scale_slot_stride;
  c.scale_head_stride = in->scale_head_stride;
  if (size == 1 && (!in->scale || ((uintptr_t)in->scale & 3))) return false;
  return aligned(c.data, c.page_stride, c.slot_stride, c.head_stride, 8 * size);
}

}  // namespace

extern "C" int ako4x_rope(const ako4x_head_rows* q, const ako4x_head_rows* k, const void* positions, int positions_int64,
                          const float* inv_freq, int64_t rotary_dim, int interleaved, float attention_factor, void* q_out,
                          void* k_out, int64_t tokens, int64_t dim, int dtype, void* stream) {
  if (!q) return AKO4X_EINVAL;
  Params p = common(positions, positions_int64, inv_freq, interleaved, attention_factor, q_out, k_out);
  if (k && k->heads > 0 && tokens > 0 && !aligned(k_out, 0, 0, 0, 16)) return AKO4X_EINVAL;
  return run(p, q, k, nullptr, tokens, dim, rotary_dim, dtype, stream);
}

extern "C" int ako4x_qk_norm_rope(const ako4x_head_rows* q, const ako4x_head_rows* k, const void* q_weight,
                                  const void* k_weight, int weights_fp32, float eps, const void* positions,
                                  int positions_int64, const float* inv_freq, int64_t rotary_dim, int interleaved,
                                  float attention_factor, void* q_out, void* k_out, int64_t tokens, int64_t dim, int dtype,
                                  void* stream) {
  if (!q || !k) return AKO4X_EINVAL;
  if (tokens > 0 && (!q_weight || !k_weight || (k->heads > 0 && !aligned(k_out, 0, 0, 0, 16)))) return AKO4X_EINVAL;
  Params p = common(positions, positions_int64, inv_freq, interleaved, attention_factor, q_out, k_out);
  p.q_weight = q_weight;
  p.k_weight = k_weight;
  p.weights32 = weights_fp32 != 0;
  p.eps = eps;
  return run(p, q, k, nullptr, tokens, dim, rotary_dim, dtype, stream);
}

extern "C" int ako4x_qk_norm_rope_cache(const ako4x_head_rows* q, const ako4x_head_rows* k, const ako4x_head_rows* v,
                                        const void* q_weight, const void* k_weight, int weights_fp32, float eps,
                                        const void* positions, int positions_int64, const float* inv_freq,
                                        int64_t rotary_dim, int interleaved, float attention_factor, void* q_out,
                                        const void* slot_mapping, int slots_int64, const ako4x_kv_cache* k_cache,
                                        const ako4x_kv_cache* v_cache, int cache_dtype, int64_t num_pages, int64_t page_size,
                                        int64_t tokens, int64_t dim, int dtype, void* stream) {
  if (!q || !k || !v || !k_cache || !v_cache) return AKO4X_EINVAL;
  if (num_pages < 0 || page_size < 1 || page_size > 0x7fffffffLL || k->heads != v->heads) return AKO4X_EINVAL;
  if (cache_dtype != dtype && cache_dtype != AKO4X_E4M3) return AKO4X_EUNSUPPORTED_SHAPE;
  Params p = common(positions, positions_int64, inv_freq, interleaved, attention_factor, q_out, nullptr);
  if (tokens > 0 && k->heads > 0) {
    if (!slot_mapping || !set_cache(p.kc, k_cache, cache_dtype) || !set_cache(p.vc, v_cache, cache_dtype)) {
      if (!slot_mapping || num_pages > 0) return AKO4X_EINVAL;
    }
  }
  p.q_weight = q_weight;
  p.k_weight = k_weight;
  p.weights32 = weights_fp32 != 0;
  p.eps = eps;
  p.slots = slot_mapping;
  p.slots64 = slots_int64 != 0;
  p.num_slots = num_pages * page_size;
  p.page_size = (int)page_size;
  p.quant = cache_dtype == AKO4X_E4M3;
  return run(p, q, k, v, tokens, dim, rotary_dim, dtype, stream);
}
