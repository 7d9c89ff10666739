// Rotary positions, the 4-bit append of keys and values, and the read-back of cached tokens.
//
// out = x cos - x' sin over rotation pairs (x, x'), in fp32 with each product rounded by itself:
// pairs (d, d + R/2) in the half layout, (2i, 2i + 1) in the interleaved one; dimensions from R
// on pass through. cos and sin come from a table with one row a position, so a scaled rotation
// is a scaled table. Queries are rounded to bf16 once; rotated keys go to 4 bits from fp32.
//
// The work is a few operations a byte, so memory bounds it (and launch latency at decode sizes). A warp
// takes queries, or keys and values, of one token and loads them all before it computes, so the
// rotation row is read once for them. A query vector is owned by D/8 lanes with both halves of their
// rotation pairs. A key or value vector is owned by D/4 lanes, four contiguous dimensions each:
// rotation partners are a shuffle away in the half layout and in the lane itself in the interleaved
// one, a group of 32 dimensions is 8 lanes, and a lane's four codes are one 16-bit store. 8191 tokens x
// 28 + 8 heads of 128, 139 MB: 36 us, 3.8 TB/s (with queries laid out as keys and a division a value:
// 64); the scattered 16-bit stores of codes hold up the rest. The read of them, 21 MB: 7 us.
#include "kv4.cuh"
#include "qrow_common.cuh"

namespace mrb {

constexpr int KA_WARPS = 4;  // warps a CTA
constexpr int KA_ITERS = 4;  // vectors a lane group takes in one go

struct Kv4AppendArgs {
  const __nv_bfloat16 *q, *k, *v;
  int64_t q_stride, k_stride, v_stride;
  const int32_t *positions, *slots;
  const float *cos, *sin;
  const __nv_bfloat16 *q_norm, *k_norm;
  __nv_bfloat16* q_out;
  int32_t* error_flag;
  Kv4Pool pool;
  int64_t tokens, rope_len;
  int hq, hkv, half, q_chunks, chunks;  // half: R / 2; warps a token: of queries, in all
  float eps;
};

__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float4 unpack_bf16x4(uint2 u) {
  return make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u), __uint_as_float(u.y << 16),
                     __uint_as_float(u.y & 0xffff0000u));
}
__device__ __forceinline__ uint2 pack_bf16x4(float4 f) {
  const __nv_bfloat162 a = __floats2bfloat162_rn(f.x, f.y), b = __floats2bfloat162_rn(f.z, f.w);
  uint2 u;
  u.x = *reinterpret_cast<const uint32_t*>(&a);
  u.y = *reinterpret_cast<const uint32_t*>(&b);
  return u;
}

// Four dimensions of one vector to 4 bits; the lanes of a group of G dimensions agree on its
// scale and minimum (min and max keep NaN, so a group that holds one, or an infinity, stands
// for NaN throughout).
template <int G>
__device__ __forceinline__ void quantise4(float4 x, uint16_t* codes, uint32_t* param) {
  float lo = min_nan(min_nan(x.x, x.y), min_nan(x.z, x.w)), hi = max_nan(max_nan(x.x, x.y), max_nan(x.z, x.w));
  if constexpr (G == 128) {  // the whole warp: one instruction each
    asm volatile("redux.sync.min.NaN.f32 %0, %0, 0xffffffff;" : "+f"(lo));
    asm volatile("redux.sync.max.NaN.f32 %0, %0, 0xffffffff;" : "+f"(hi));
  } else {
#pragma unroll
    for (int o = 1; o < G / 4; o <<= 1) {
      lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, o));
      hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    }
  }
  const __nv_bfloat16 mb = __float2bfloat16_rn(lo);
  const float m = __bfloat162float(mb);
  float s = max_nan(__fdiv_rn(__fsub_rn(hi, m), 15.f), 0.f);
  // of an infinite range: NaN, so that readers meet finite scales or NaN
  if (s > 3e38f) s = __int_as_float(0x7fffffff);
  const __nv_bfloat16 sb = __float2bfloat16_rn(s);
  s = __bfloat162float(sb);
  // (v - m) / s to the nearest integer, by a product with 1 / s whose remainder tells whether it is: what
  // is further than 0.49999 s from its integer (a tie, nearly), and a range out of the ordinary, is
  // divided (all of them by division: 45 us instead of 35 for 8191 tokens x 28 + 8 heads)
  const float inv = __frcp_rn(s), v[4] = {__fsub_rn(x.x, m), __fsub_rn(x.y, m), __fsub_rn(x.z, m), __fsub_rn(x.w, m)};
  float far = 0.f;
  int c[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float t = fmaf(v[e], inv, 12582912.f);  // 1.5 x 2^23: the integer in the low bits
    c[e] = min(max(__float_as_int(t) - 0x4b400000, 0), 15);
    far = fmaxf(far, fabsf(fmaf(12582912.f - t, s, v[e])));
  }
  if (!(far <= 0.49999f * s && s > 1e-30f && s < 1e30f))
#pragma unroll
    for (int e = 0; e < 4; ++e)  // fmaxf takes the number of a number and a NaN: 0 / 0 of a constant group is code 0
      c[e] = (int)fminf(fmaxf(rintf(__fdiv_rn(v[e], s)), 0.f), 15.f);
  *codes = (uint16_t)(c[0] | c[1] << 4 | c[2] << 8 | c[3] << 12);
  *param = (uint32_t)__bfloat16_as_ushort(sb) | (uint32_t)__bfloat16_as_ushort(mb) << 16;
}

__device__ __forceinline__ float4 turn(float4 x, float4 y, float4 c, float4 n) {  // x c + y n
  return make_float4(__fadd_rn(__fmul_rn(x.x, c.x), __fmul_rn(y.x, n.x)), __fadd_rn(__fmul_rn(x.y, c.y), __fmul_rn(y.y, n.y)),
                     __fadd_rn(__fmul_rn(x.z, c.z), __fmul_rn(y.z, n.z)), __fadd_rn(__fmul_rn(x.w, c.w), __fmul_rn(y.w, n.w)));
}
__device__ __forceinline__ float4 negated(float4 x) { return make_float4(-x.x, -x.y, -x.z, -x.w); }
__device__ __forceinline__ float squares(float4 x) { return x.x * x.x + x.y * x.y + x.z * x.z + x.w * x.w; }
__device__ __forceinline__ float4 scaled(float4 x, float r, float4 w) {
  return make_float4(x.x * r * w.x, x.y * r * w.y, x.z * r * w.z, x.w * r * w.w);
}

// Queries: a head vector is owned by D/8 lanes, each with two fours of dimensions that turn together, so
// that no rotation leaves its lane; KA_ITERS x 256 / D vectors of one token a warp.
template <int D, bool INTERLEAVED>
__device__ __forceinline__ void append_queries(const Kv4AppendArgs& a, int64_t t, int chunk, int lane) {
  constexpr int SUB = D / 8, PER = 32 / SUB;
  const int l = lane % SUB, first = chunk * KA_ITERS * PER + lane / SUB;
  const int pairs = a.half / 4;  // lanes with two halves of pairs; the others' dimensions stay
  const int da = INTERLEAVED ? 8 * l : l < pairs ? 4 * l : 2 * a.half + 8 * (l - pairs);
  const int db = INTERLEAVED || l >= pairs ? da + 4 : da + a.half;
  uint2 in[KA_ITERS][2];
#pragma unroll
  for (int i = 0; i < KA_ITERS; ++i) {
    const int h = first + i * PER;
    in[i][0] = in[i][1] = make_uint2(0u, 0u);
    if (h >= a.hq) continue;
    const __nv_bfloat16* src = a.q + t * a.q_stride + (int64_t)h * D;
    in[i][0] = __ldg(reinterpret_cast<const uint2*>(src + da));
    in[i][1] = __ldg(reinterpret_cast<const uint2*>(src + db));
  }
  const int pos = a.half ? a.positions[t] : 0;
  const bool pos_ok = !a.half || (pos >= 0 && pos < a.rope_len);
  if (chunk == 0 && lane == 0 && a.error_flag && !pos_ok) atomicOr(a.error_flag, MRB_KV_BAD_SLOT);
  const bool turns = l < pairs && pos_ok;
  float4 c = make_float4(1.f, 1.f, 1.f, 1.f), n = make_float4(0.f, 0.f, 0.f, 0.f);
  if (turns) {
    c = *reinterpret_cast<const float4*>(a.cos + (int64_t)pos * a.half + 4 * l);
    n = *reinterpret_cast<const float4*>(a.sin + (int64_t)pos * a.half + 4 * l);
  }
#pragma unroll
  for (int i = 0; i < KA_ITERS; ++i) {
    const int h = first + i * PER;
    float4 x = unpack_bf16x4(in[i][0]), y = unpack_bf16x4(in[i][1]);
    if (a.q_norm != nullptr) {
      float ss = squares(x) + squares(y);
#pragma unroll
      for (int o = 1; o < SUB; o <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      const float r = rsqrtf(ss / D + a.eps);
      x = scaled(x, r, unpack_bf16x4(*reinterpret_cast<const uint2*>(a.q_norm + da)));
      y = scaled(y, r, unpack_bf16x4(*reinterpret_cast<const uint2*>(a.q_norm + db)));
    }
    if (turns) {
      if (INTERLEAVED) {
        const float4 u = x, v = y;
        x = turn(u, make_float4(u.y, u.x, u.w, u.z), make_float4(c.x, c.x, c.y, c.y), make_float4(-n.x, n.x, -n.y, n.y));
        y = turn(v, make_float4(v.y, v.x, v.w, v.z), make_float4(c.z, c.z, c.w, c.w), make_float4(-n.z, n.z, -n.w, n.w));
      } else {
        const float4 u = x;
        x = turn(u, y, c, negated(n));
        y = turn(y, u, c, n);
      }
    }
    if (!pos_ok) x = y = make_float4(0.f, 0.f, 0.f, 0.f);
    if (h < a.hq) {
      __nv_bfloat16* dst = a.q_out + (t * a.hq + h) * D;
      *reinterpret_cast<uint2*>(dst + da) = pack_bf16x4(x);
      *reinterpret_cast<uint2*>(dst + db) = pack_bf16x4(y);
    }
  }
}

template <int D, int G, bool INTERLEAVED>
__global__ void __launch_bounds__(KA_WARPS * 32) rope_kv4_append_kernel(const __grid_constant__ Kv4AppendArgs a) {
  constexpr int SUB = D / 4, PER = 32 / SUB, VECS = KA_ITERS * PER;  // lanes a vector, vectors a warp
  constexpr int BLOCK = kv4_block_bytes(D, G), CODES = kv4_codes_bytes(D), PARAMS = kv4_params_bytes(D, G);
  const int lane = threadIdx.x & 31, sub = lane / SUB, l = lane % SUB, d0 = 4 * l;
  const unsigned item = blockIdx.x * KA_WARPS + (threadIdx.x >> 5);  // at most 2^31
  pdl_launch_dependents();
  const int64_t t = item / (unsigned)a.chunks;
  if (t >= a.tokens) return;
  const int chunk = (int)(item - (unsigned)t * a.chunks);
  pdl_wait();
  if (chunk < a.q_chunks) {
    append_queries<D, INTERLEAVED>(a, t, chunk, lane);
    return;
  }
  const int first = (chunk - a.q_chunks) * VECS, heads = 2 * a.hkv;
  // every vector of this warp, in flight together: heads in the order k, v
  uint2 in[KA_ITERS];
#pragma unroll
  for (int i = 0; i < KA_ITERS; ++i) {
    const int h = first + i * PER + sub;
    in[i] = make_uint2(0u, 0u);
    if (h >= heads) continue;
    const __nv_bfloat16* src = h < a.hkv ? a.k + t * a.k_stride + (int64_t)h * D
                                         : a.v + t * a.v_stride + (int64_t)(h - a.hkv) * D;
    in[i] = __ldg(reinterpret_cast<const uint2*>(src + d0));
  }
  const int slot = a.slots[t];
  const int pos = a.half ? a.positions[t] : 0;
  const bool pos_ok = !a.half || (pos >= 0 && pos < a.rope_len);
  const bool slot_ok = slot >= 0 && slot < a.pool.num_pages * a.pool.page_size;
  if (lane == 0 && a.error_flag && ((slot != -1 && !slot_ok) || !pos_ok)) atomicOr(a.error_flag, MRB_KV_BAD_SLOT);
  float4 c = make_float4(1.f, 1.f, 1.f, 1.f), n = make_float4(0.f, 0.f, 0.f, 0.f);
  const bool turns = a.half && d0 < 2 * a.half && pos_ok;
  if (turns) {
    const int64_t row = (int64_t)pos * a.half;
    if (INTERLEAVED) {
      const float2 cc = *reinterpret_cast<const float2*>(a.cos + row + 2 * l);
      const float2 nn = *reinterpret_cast<const float2*>(a.sin + row + 2 * l);
      c = make_float4(cc.x, cc.x, cc.y, cc.y);
      n = make_float4(-nn.x, nn.x, -nn.y, nn.y);
    } else {
      const int f = d0 < a.half ? d0 : d0 - a.half;
      c = *reinterpret_cast<const float4*>(a.cos + row + f);
      n = *reinterpret_cast<const float4*>(a.sin + row + f);
      if (d0 < a.half) n = make_float4(-n.x, -n.y, -n.z, -n.w);
    }
  }
  const int hop = a.half / 4;  // lanes between the halves of a pair
  const int partner = lane - l + (l < hop ? l + hop : l < 2 * hop ? l - hop : l);
  const int64_t page = slot_ok ? slot / a.pool.page_size : 0;
  const int tok = slot_ok ? slot - (int)page * a.pool.page_size : 0, row = tok % KV4_TILE;

#pragma unroll
  for (int i = 0; i < KA_ITERS; ++i) {
    const int h = first + i * PER + sub;
    float4 x = unpack_bf16x4(in[i]);
    if (a.k_norm != nullptr) {
      float ss = squares(x);
#pragma unroll
      for (int o = 1; o < SUB; o <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      if (h < a.hkv) x = scaled(x, rsqrtf(ss / D + a.eps), unpack_bf16x4(*reinterpret_cast<const uint2*>(a.k_norm + d0)));
    }
    float4 y;
    if (INTERLEAVED) {
      y = make_float4(x.y, x.x, x.w, x.z);
    } else {
      y.x = __shfl_sync(0xffffffffu, x.x, partner);
      y.y = __shfl_sync(0xffffffffu, x.y, partner);
      y.z = __shfl_sync(0xffffffffu, x.z, partner);
      y.w = __shfl_sync(0xffffffffu, x.w, partner);
    }
    if (turns && h < a.hkv) x = turn(x, y, c, n);
    uint16_t codes;
    uint32_t param;
    quantise4<G>(x, &codes, &param);
    if (h < heads && slot_ok && pos_ok) {
      const bool is_v = h >= a.hkv;
      unsigned char* b = a.pool.block(page, h - (is_v ? a.hkv : 0), tok, BLOCK);
      *reinterpret_cast<uint16_t*>(b + (is_v ? CODES : 0) + row * (D / 2) + 2 * l) = codes;
      if (l % (G / 4) == 0)
        *reinterpret_cast<uint32_t*>(b + 2 * CODES + (is_v ? PARAMS : 0) + (row * (D / G) + l / (G / 4)) * 4) = param;
    }
  }
}

struct Kv4ReadArgs {
  Kv4Pool pool;
  const int32_t* slots;
  void *k_out, *v_out;
  int32_t* error_flag;
  int64_t tokens;
};

// What the given slots stand for: one fp32 fused multiply-add a value (code times scale is
// exact), rounded once to the output's type. A lane takes eight dimensions of one head's K or V.
template <int D, int G, typename T>
__global__ void __launch_bounds__(256) kv4_read_kernel(const __grid_constant__ Kv4ReadArgs a) {
  constexpr unsigned SUB = D / 8;
  constexpr int BLOCK = kv4_block_bytes(D, G), CODES = kv4_codes_bytes(D), PARAMS = kv4_params_bytes(D, G);
  pdl_launch_dependents();
  pdl_wait();
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  const int l = (int)(i % SUB);
  const unsigned vec = (unsigned)(i / SUB), t = vec / (unsigned)(2 * a.pool.hkv);  // vec is below 2^31 and a CTA
  if (t >= a.tokens) return;
  const int hv = (int)(vec - t * 2 * a.pool.hkv);
  const bool is_v = hv >= a.pool.hkv;
  const int h = hv - (is_v ? a.pool.hkv : 0);
  const int slot = a.slots[t];
  const bool ok = slot >= 0 && slot < a.pool.num_pages * a.pool.page_size;
  float x[8] = {};
  if (ok) {
    const int64_t page = slot / a.pool.page_size;
    const int tok = slot - (int)page * a.pool.page_size, row = tok % KV4_TILE;
    const unsigned char* b = a.pool.block(page, h, tok, BLOCK);
    const uint32_t c = *reinterpret_cast<const uint32_t*>(b + (is_v ? CODES : 0) + row * (D / 2) + 4 * l);
    const uint32_t p = *reinterpret_cast<const uint32_t*>(b + 2 * CODES + (is_v ? PARAMS : 0) +
                                                          (row * (D / G) + l / (G / 8)) * 4);
    const float s = __uint_as_float(p << 16), m = __uint_as_float(p & 0xffff0000u);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = fmaf(s, (float)(c >> (4 * e) & 15u), m);
  } else if (slot != -1 && l == 0 && a.error_flag) {
    atomicOr(a.error_flag, MRB_KV_BAD_SLOT);
  }
  T* out = reinterpret_cast<T*>(is_v ? a.v_out : a.k_out) + ((int64_t)t * a.pool.hkv + h) * D + 8 * l;
  const float4 lo = make_float4(x[0], x[1], x[2], x[3]), hi = make_float4(x[4], x[5], x[6], x[7]);
  if constexpr (sizeof(T) == 4) {
    reinterpret_cast<float4*>(out)[0] = lo;
    reinterpret_cast<float4*>(out)[1] = hi;
  } else {
    const uint2 u = pack_bf16x4(lo), v = pack_bf16x4(hi);
    *reinterpret_cast<uint4*>(out) = make_uint4(u.x, u.y, v.x, v.y);
  }
}

template <int D, int G>
static int launch_append(const Kv4AppendArgs& a, bool interleaved, cudaStream_t s) {
  const int64_t ctas = (a.tokens * a.chunks + KA_WARPS - 1) / KA_WARPS;
  launch_kernel(interleaved ? rope_kv4_append_kernel<D, G, true> : rope_kv4_append_kernel<D, G, false>,
                dim3((unsigned)ctas), dim3(KA_WARPS * 32), 0, s, true, a);
  return launch_status("rope_kv4_append");
}

template <int D, int G>
static int launch_read(const Kv4ReadArgs& a, int dtype, cudaStream_t s) {
  const int64_t threads = a.tokens * 2 * a.pool.hkv * (D / 8);
  launch_kernel(dtype == MRB_F32 ? kv4_read_kernel<D, G, float> : kv4_read_kernel<D, G, __nv_bfloat16>,
                dim3((unsigned)((threads + 255) / 256)), dim3(256), 0, s, true, a);
  return launch_status("kv4_read");
}

}  // namespace mrb

extern "C" int mrb_rope_kv4_append_strided(const void* q_in, const void* k_in, const void* v_in, int64_t q_row_stride,
                                           int64_t k_row_stride, int64_t v_row_stride, int64_t tokens, int64_t hq,
                                           int64_t hkv, int64_t head_dim, int64_t group, const int32_t* positions,
                                           const int32_t* slots, const float* rope_cos, const float* rope_sin,
                                           int64_t rope_len, int64_t rotary_dim, int interleaved, const void* q_norm,
                                           const void* k_norm, float norm_eps, void* q_out, void* pool,
                                           int64_t num_pages, int64_t page_size, int64_t stride_page,
                                           int64_t stride_head, int32_t* error_flag, void* stream) {
  using namespace mrb;
  const char* what = "rope_kv4_append";
  Kv4AppendArgs a = {};
  const int rc = kv4_check_pool(what, pool, num_pages, hkv, page_size, stride_page, stride_head, head_dim, group, &a.pool);
  if (rc != MRB_OK) return rc;
  if (tokens < 0 || hq < 0) return fail(MRB_ERR_ARG, "%s: bad sizes", what);
  if (hq > 65535 || hkv > 65535) return fail(MRB_ERR_UNSUPPORTED, "%s: at most 65535 heads", what);
  if (!rope_cos != !rope_sin) return fail(MRB_ERR_ARG, "%s: give both rotary tables or neither", what);
  if (rope_cos) {
    if (rotary_dim < 1 || rotary_dim > head_dim || rotary_dim % 8)
      return fail(MRB_ERR_ARG, "%s: rotary_dim must be a multiple of 8 up to head_dim", what);
    if (rope_len < 1) return fail(MRB_ERR_ARG, "%s: empty rotary tables", what);
  }
  if (!q_norm != !k_norm) return fail(MRB_ERR_ARG, "%s: give both norm weights or neither", what);
  if (tokens == 0) {
    clear_error();
    return MRB_OK;
  }
  if (!k_in || !v_in || !slots || (hq > 0 && (!q_in || !q_out)) || (rope_cos && !positions))
    return fail(MRB_ERR_ARG, "%s: null pointer", what);
  if (!aligned(q_in, 8) || !aligned(k_in, 8) || !aligned(v_in, 8) || !aligned(q_out, 8) || q_row_stride % 4 || k_row_stride % 4 ||
      v_row_stride % 4 || !aligned(rope_cos, 16) || !aligned(rope_sin, 16) || !aligned(q_norm, 8) ||
      !aligned(k_norm, 8))
    return fail(MRB_ERR_ARG, "%s: rows must be 8-byte aligned and rotary tables 16-byte aligned", what);
  a.q = (const __nv_bfloat16*)q_in;
  a.k = (const __nv_bfloat16*)k_in;
  a.v = (const __nv_bfloat16*)v_in;
  a.q_stride = q_row_stride;
  a.k_stride = k_row_stride;
  a.v_stride = v_row_stride;
  a.positions = positions;
  a.slots = slots;
  a.cos = rope_cos;
  a.sin = rope_sin;
  a.q_norm = (const __nv_bfloat16*)q_norm;
  a.k_norm = (const __nv_bfloat16*)k_norm;
  a.q_out = (__nv_bfloat16*)q_out;
  a.error_flag = error_flag;
  a.tokens = tokens;
  a.rope_len = rope_len;
  a.hq = (int)hq;
  a.hkv = (int)hkv;
  a.half = rope_cos ? (int)rotary_dim / 2 : 0;
  const int vecs = KA_ITERS * (head_dim == 128 ? 1 : 2);  // keys or values a warp; of queries twice as many
  a.q_chunks = (int)((hq + 2 * vecs - 1) / (2 * vecs));
  a.chunks = a.q_chunks + (int)((2 * hkv + vecs - 1) / vecs);
  a.eps = norm_eps;
  if (tokens > ((int64_t)INT32_MAX - KA_WARPS) / a.chunks) return fail(MRB_ERR_UNSUPPORTED, "%s: too many tokens", what);
  cudaStream_t s = (cudaStream_t)stream;
  if (head_dim == 64) return group == 32 ? launch_append<64, 32>(a, interleaved, s) : launch_append<64, 64>(a, interleaved, s);
  if (group == 32) return launch_append<128, 32>(a, interleaved, s);
  if (group == 64) return launch_append<128, 64>(a, interleaved, s);
  return launch_append<128, 128>(a, interleaved, s);
}

extern "C" int mrb_rope_kv4_append(const void* q_in, const void* k_in, const void* v_in, int64_t in_row_stride,
                                   int64_t v_row_stride, int64_t tokens, int64_t hq, int64_t hkv, int64_t head_dim,
                                   int64_t group, const int32_t* positions, const int32_t* slots,
                                   const float* rope_cos, const float* rope_sin, int64_t rope_len, int64_t rotary_dim,
                                   int interleaved, const void* q_norm, const void* k_norm, float norm_eps,
                                   void* q_out, void* pool, int64_t num_pages, int64_t page_size, int64_t stride_page,
                                   int64_t stride_head, int32_t* error_flag, void* stream) {
  return mrb_rope_kv4_append_strided(q_in, k_in, v_in, in_row_stride, in_row_stride, v_row_stride, tokens, hq, hkv,
                                     head_dim, group, positions, slots, rope_cos, rope_sin, rope_len, rotary_dim,
                                     interleaved, q_norm, k_norm, norm_eps, q_out, pool, num_pages, page_size,
                                     stride_page, stride_head, error_flag, stream);
}

extern "C" int mrb_kv4_read(const void* pool, int64_t num_pages, int64_t hkv, int64_t head_dim, int64_t group,
                            int64_t page_size, int64_t stride_page, int64_t stride_head, const int32_t* slots,
                            int64_t tokens, void* k_out, void* v_out, int out_dtype, int32_t* error_flag,
                            void* stream) {
  using namespace mrb;
  const char* what = "kv4_read";
  Kv4ReadArgs a = {};
  const int rc = kv4_check_pool(what, pool, num_pages, hkv, page_size, stride_page, stride_head, head_dim, group, &a.pool);
  if (rc != MRB_OK) return rc;
  if (tokens < 0) return fail(MRB_ERR_ARG, "%s: bad sizes", what);
  if (out_dtype != MRB_F32 && out_dtype != MRB_BF16) return fail(MRB_ERR_ARG, "%s: output must be fp32 or bf16", what);
  if (tokens == 0) {
    clear_error();
    return MRB_OK;
  }
  if (!slots || !k_out || !v_out) return fail(MRB_ERR_ARG, "%s: null pointer", what);
  if (!aligned(k_out, 16) || !aligned(v_out, 16)) return fail(MRB_ERR_ARG, "%s: outputs must be 16-byte aligned", what);
  if (hkv > 65535 || tokens > (int64_t)INT32_MAX / (2 * hkv))
    return fail(MRB_ERR_UNSUPPORTED, "%s: too many tokens", what);
  a.slots = slots;
  a.k_out = k_out;
  a.v_out = v_out;
  a.error_flag = error_flag;
  a.tokens = tokens;
  cudaStream_t s = (cudaStream_t)stream;
  if (head_dim == 64) return group == 32 ? launch_read<64, 32>(a, out_dtype, s) : launch_read<64, 64>(a, out_dtype, s);
  if (group == 32) return launch_read<128, 32>(a, out_dtype, s);
  if (group == 64) return launch_read<128, 64>(a, out_dtype, s);
  return launch_read<128, 128>(a, out_dtype, s);
}
