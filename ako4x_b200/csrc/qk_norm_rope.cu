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
// its last bits, for any position. In the norm the factors of a token are the same for all its heads: z = (inv x) A + (inv x') B
// with x' the partner and A = w c, B = -+ w' s kept in registers, 16 per lane.
//
// HBM-bound: every element is read and written once. 8, 16 or 32 lanes own a row (16 bytes each), a warp
// takes row groups of one token (all of them, or a share where there are few tokens), four loads in flight
// per lane; the token's R/2 angles are shared out over the lanes once. The partner is R/16 lanes away (one
// shuffle per word), in the same lane (interleaved), or, where R/2 is no multiple of 8, read again.
#include "common.cuh"

#include <cuda_fp16.h>

namespace {

constexpr int WARPS = 4;
constexpr int MAX_DIM = 256;
constexpr int UNROLL = 4;

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
  int shares;                 // warps per token
  float eps, inv_dim, factor;
  bool interleaved, positions64, slots64, weights32, quant;
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

template <class T>
__device__ __forceinline__ void unpack(const uint4& v, float (&x)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 p = Pair<T>::get(w[i]);
    x[2 * i] = p.x;
    x[2 * i + 1] = p.y;
  }
}
template <class T>
__device__ __forceinline__ uint4 packed(const float (&x)[8]) {
  return make_uint4(Pair<T>::put(x[0], x[1]), Pair<T>::put(x[2], x[3]), Pair<T>::put(x[4], x[5]), Pair<T>::put(x[6], x[7]));
}
__device__ __forceinline__ float max_nan(float a, float b) {   // a NaN stays
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// 8 values of a row, quantised with the row's own scale: amax / 448, 1 for a row of (nearly) zeros.
template <int LANES>
__device__ __forceinline__ void store_e4m3(const float (&x)[8], unsigned char* to, float* scale, int lane, bool live) {
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max_nan(top, fabsf(x[i]));
#pragma unroll
  for (int o = LANES / 2; o >= 1; o >>= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
  const float s = top <= 1e-10f ? 1.0f : __fdiv_rn(top, 448.0f);
  if (!live) return;
  uint32_t out[2] = {0u, 0u};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t pair = __nv_cvt_float2_to_fp8x2(make_float2(__fdiv_rn(x[2 * i], s), __fdiv_rn(x[2 * i + 1], s)), __NV_SATFINITE, __NV_E4M3);
    out[i >> 1] |= pair << (16 * (i & 1));
  }
  *(reinterpret_cast<uint2*>(to) + lane) = make_uint2(out[0], out[1]);
  if (lane == 0) *scale = s;
}

// Where the partner of a rotated element is.
enum Partner { OTHER_LANE, SAME_LANE, MEMORY };

template <class T, int LANES, Partner PARTNER>
__global__ void __launch_bounds__(WARPS * 32) qk_norm_rope_kernel(const Params p) {
  constexpr int GROUP = 32 / LANES;   // rows of a warp instruction
  __shared__ float2 s_cs[WARPS][MAX_DIM / 2];
  const int warp = threadIdx.x >> 5, lane32 = threadIdx.x & 31;
  const int lane = lane32 % LANES, sub = lane32 / LANES;
  const int64_t unit = (int64_t)blockIdx.x * WARPS + warp;
  const int64_t token = unit / p.shares;
  if (token >= p.tokens) return;      // whole warps; there is no block barrier
  const int share = (int)(unit - token * p.shares);
  const int groups = p.q.groups + p.k.groups + p.v.groups;
  const int g0 = (int)((int64_t)groups * share / p.shares), g1 = (int)((int64_t)groups * (share + 1) / p.shares);

  const int half = p.rotary / 2;
  if (g0 < p.q.groups + p.k.groups) {
    const double pos = p.positions64 ? (double)((const int64_t*)p.positions)[token] : (double)((const int32_t*)p.positions)[token];
    for (int i = lane32; i < half; i += 32) {
      double turn = pos * ((double)__ldg(p.inv_freq + i) * 0.15915494309189533577);   // f / 2 pi
      turn -= rint(turn);
      // and the nearest quarter: sine and cosine are then both good to their last bits, next to their zeros too
      const double quarters = rint(turn * 4.0);
      float s, c;
      sincospif(2.0f * (float)(turn - quarters * 0.25), &s, &c);
      const int quadrant = (int)quarters & 3;
      const float x = quadrant & 1 ? -s : c, y = quadrant & 1 ? c : s;
      s_cs[warp][i] = make_float2((quadrant & 2 ? -x : x) * p.factor, (quadrant & 2 ? -y : y) * p.factor);
    }
    __syncwarp();
  }
  int64_t page = 0, slot = 0;
  bool stored = false;
  if (p.slots) {
    const int64_t at = p.slots64 ? ((const int64_t*)p.slots)[token] : (int64_t)((const int32_t*)p.slots)[token];
    stored = at >= 0 && at < p.num_slots;   // anything else: a padding token, its keys and values go nowhere
    page = stored ? at / p.page_size : 0;
    slot = stored ? at - page * p.page_size : 0;
  }
  const int e0 = lane * 8;
  const bool in_row = e0 < p.dim;

  int first = 0;                       // groups in front of this kind
#pragma unroll 1
  for (int kind = 0; kind < 3; ++kind) {
    const Rows& r = kind == 0 ? p.q : kind == 1 ? p.k : p.v;
    const int lo = max(g0, first) - first, hi = min(g1, first + r.groups) - first;
    first += r.groups;
    if (lo >= hi) continue;
    const bool to_cache = kind == 2 || (kind == 1 && !p.k_out);
    if (to_cache && !stored) continue;
    const void* weight = kind == 0 ? p.q_weight : kind == 1 ? p.k_weight : nullptr;
    const bool turn = kind != 2;

    // z = (inv x) A + (inv x') B
    float A[8], B[8];
    bool whole = turn;                 // all eight elements have a partner
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      A[j] = 1.f;
      B[j] = 0.f;
      const int e = e0 + j;
      const bool rot = turn && e < p.rotary;
      whole &= rot;
      int other = e, i = 0;
      bool second = false;
      if (rot) {
        second = PARTNER == SAME_LANE ? (e & 1) : e >= half;
        i = PARTNER == SAME_LANE ? e >> 1 : second ? e - half : e;
        other = PARTNER == SAME_LANE ? e ^ 1 : second ? e - half : e + half;
        const float2 cs = s_cs[warp][i];
        A[j] = cs.x;
        B[j] = second ? cs.y : -cs.y;
      }
      if (weight && in_row) {
        A[j] *= p.weights32 ? __ldg((const float*)weight + e) : Pair<T>::one((const T*)weight + e);
        if (rot) B[j] *= p.weights32 ? __ldg((const float*)weight + other) : Pair<T>::one((const T*)weight + other);
      }
    }
    const int away = e0 < half ? half / 8 : -(half / 8);   // lanes to the partner

    const unsigned char* base = r.in + token * r.token_stride + e0 * 2;
#pragma unroll 1
    for (int g = lo; g < hi; g += UNROLL) {
      uint4 raw[UNROLL];
#pragma unroll
      for (int u = 0; u < UNROLL; ++u) {
        const int head = (g + u) * GROUP + sub;
        raw[u] = make_uint4(0u, 0u, 0u, 0u);
        if (g + u < hi && head < r.heads && in_row) raw[u] = __ldg(reinterpret_cast<const uint4*>(base + head * r.head_stride));
      }
#pragma unroll
      for (int u = 0; u < UNROLL; ++u) {
        if (g + u >= hi) break;        // the whole warp
        const int head = (g + u) * GROUP + sub;
        const bool live = head < r.heads && in_row;
        float x[8], y[8];
        unpack<T>(raw[u], x);
        if (turn) {
          float o[8];                  // the partners
          if (PARTNER == OTHER_LANE) {
            const int from = lane32 + away;
            const uint4 w = make_uint4(__shfl_sync(0xffffffffu, raw[u].x, from), __shfl_sync(0xffffffffu, raw[u].y, from),
                                       __shfl_sync(0xffffffffu, raw[u].z, from), __shfl_sync(0xffffffffu, raw[u].w, from));
            unpack<T>(w, o);
          } else if (PARTNER == SAME_LANE) {
#pragma unroll
            for (int j = 0; j < 8; ++j) o[j] = x[j ^ 1];
          } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const int e = e0 + j;
              o[j] = 0.f;
              if (live && e < p.rotary)
                o[j] = Pair<T>::one(base + head * r.head_stride + (j + (e < half ? half : -half)) * 2);
            }
          }
          if (!whole) {                // an element that is not rotated takes nothing from another one
#pragma unroll
            for (int j = 0; j < 8; ++j)
              if (e0 + j >= p.rotary) o[j] = 0.f;
          }
          float inv = 1.f;
          if (weight) {
            float ss = 0.f;
#pragma unroll
            for (int j = 0; j < 8; ++j) ss = fmaf(x[j], x[j], ss);
#pragma unroll
            for (int m = LANES / 2; m >= 1; m >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, m);
            inv = rsqrtf(fmaf(ss, p.inv_dim, p.eps));
          }
#pragma unroll
          for (int j = 0; j < 8; ++j) y[j] = fmaf(x[j] * inv, A[j], (o[j] * inv) * B[j]);
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) y[j] = x[j];
        }
        if (!to_cache) {
          unsigned char* out = kind == 0 ? p.q_out : p.k_out;
          if (live) __stcs(reinterpret_cast<uint4*>(out + ((token * r.heads + head) * p.dim + e0) * 2), packed<T>(y));
        } else {
          const Cache& c = kind == 1 ? p.kc : p.vc;
          unsigned char* to = c.data + page * c.page_stride + slot * c.slot_stride + head * c.head_stride;
          if (p.quant)
            store_e4m3<LANES>(y, to, c.scale + page * c.scale_page_stride + slot * c.scale_slot_stride + head * c.scale_head_stride,
                              lane, live);
          else if (live)
            *(reinterpret_cast<uint4*>(to) + lane) = packed<T>(y);
        }
      }
    }
  }
}

template <class T, int LANES>
void launch(const Params& p, unsigned blocks, cudaStream_t st) {
  if (p.interleaved)
    qk_norm_rope_kernel<T, LANES, SAME_LANE><<<blocks, WARPS * 32, 0, st>>>(p);
  else if (p.rotary % 16 == 0)
    qk_norm_rope_kernel<T, LANES, OTHER_LANE><<<blocks, WARPS * 32, 0, st>>>(p);
  else
    qk_norm_rope_kernel<T, LANES, MEMORY><<<blocks, WARPS * 32, 0, st>>>(p);
}
template <class T>
void launch(const Params& p, int lanes, unsigned blocks, cudaStream_t st) {
  if (lanes == 8) launch<T, 8>(p, blocks, st);
  else if (lanes == 16) launch<T, 16>(p, blocks, st);
  else launch<T, 32>(p, blocks, st);
}

bool aligned(const void* ptr, int64_t a, int64_t b, int64_t c, int64_t to) {
  return ptr && (((uintptr_t)ptr | (uintptr_t)a | (uintptr_t)b | (uintptr_t)c) & (to - 1)) == 0;
}

int run(Params& p, const ako4x_head_rows* q, const ako4x_head_rows* k, const ako4x_head_rows* v, int64_t tokens, int64_t dim,
        int64_t rotary, int dtype, void* stream) {
  if (tokens < 0 || dim < 0 || rotary < 0) return AKO4X_EINVAL;
  if (dim < 8 || dim > MAX_DIM || dim % 8 || rotary > dim || rotary % 2) return AKO4X_EUNSUPPORTED_SHAPE;
  if (dtype != AKO4X_BF16 && dtype != AKO4X_FP16) return AKO4X_EUNSUPPORTED_SHAPE;
  const int lanes = dim <= 64 ? 8 : dim <= 128 ? 16 : 32;
  const int group = 32 / lanes;
  const ako4x_head_rows* in[3] = {q, k, v};
  Rows* to[3] = {&p.q, &p.k, &p.v};
  int64_t groups = 0;
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
    to[i]->groups = (int)ako::cdiv(in[i]->heads, group);
    groups += to[i]->groups;
  }
  if (tokens == 0 || groups == 0) return AKO4X_OK;
  if (!p.positions || (rotary && !p.inv_freq)) return AKO4X_EINVAL;
  if (p.q.heads && !aligned(p.q_out, 0, 0, 0, 16)) return AKO4X_EINVAL;
  p.tokens = tokens;
  p.dim = (int)dim;
  p.rotary = (int)rotary;
  p.inv_dim = 1.0f / (float)dim;
  // A warp takes a token's rows, or a share of them while there are fewer warps than the GPU holds.
  const int64_t wanted = (int64_t)ako::sm_count() * 32;
  int64_t shares = ako::cdiv(wanted, tokens);
  if (shares > groups) shares = groups;
  p.shares = (int)shares;
  const int64_t blocks = ako::cdiv(tokens * shares, WARPS);
  if (blocks > 0x7fffffffLL) return AKO4X_ETOOLARGE;
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == AKO4X_BF16) launch<__nv_bfloat16>(p, lanes, (unsigned)blocks, st);
  else launch<__half>(p, lanes, (unsigned)blocks, st);
  AKO_CHECK_LAUNCH();
  return AKO4X_OK;
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
