// Attention of one query token per row over the 4-bit paged K/V pool.
//
// Codes go to the tensor pipe as they are and the scales stay outside: with c the codes of a
// token's group, q . k = s (q . c) + m sum(q), and sum_t p_t v_t = sum_t (p_t s_t) c_t + sum_t p_t m_t.
// The four bits of a code, put at the low end of an fp16 pattern, are the (subnormal) number
// c 2^-24, and one nibble higher 16 c 2^-24, both exact: a mask makes two codes an operand pair,
// and the factors go elsewhere -- 2^-24 into the softmax scale and the final division, 16 into
// the queries (K) or the output dimension (V). Queries are scaled by a power of two to at most
// 2^14, so that fp16 holds bf16 ones exactly. Weights p s are rounded to fp16 (11 bits), relative
// to a running maximum of their own, over all groups of dimensions, which goes to 2^7 and which they
// may pass by 2^8 before the accumulators are rescaled; from 2^-21 below it fp16 rounds them to
// multiples of 2^-31 of it, so groups whose scales lie 2^21 below another's lose their codes. Sums,
// maxima and the p m term are fp32.
//
// Memory and the instructions that unpack it bound it (calls in a row: 256 rows of 4096 tokens at most x 32/8 heads, 680
// MB: 194 us, 3.5 TB/s, with 860 instructions a warp and unit, half of the issue slots used by three
// warps a scheduler, of 168 registers and 40 to 64 bytes spilled in the instances of <128, 32>; copies of
// this size alone reach 6 TB/s) and, where the cache is short, latency (32 rows x 32/4 heads, 35 MB: 22 us;
// one row of 131071 tokens, 71 MB: 31 us: the first loads of each warp and the join of the parts). A 16-token tile of one KV head is one contiguous block,
// fetched by one bulk copy into the warp's ring. Tokens fill the 16 rows of mma.sync m16n8k16 and the group's
// queries its 8 columns (NT of them): S^T = K Q^T, O^T += V^T P^T. A lane reads whole words of
// codes: eight dimensions of a token are four register pairs of a K fragment (the order of
// dimensions inside a product is free, so the queries take the same order), and for V two tokens'
// half words are put side by side first. The maxima move only when a vote finds them passed by
// 2^8, so most tiles rescale nothing.
//
// Work split, in units of two tiles: with few groups, each is cut into equal parts, one a CTA.
// With many, the groups' units, laid end to end with an allowance for each group's start and end,
// are cut into equal ranges, one a CTA, whose warps take its units in turn, their rings running on
// over group boundaries. At a group's end the warps' states are summed in shared memory, in warp
// order. A group of several CTAs leaves partials, and the last CTA to leave one sums them in CTA
// order, so results do not depend on timing.
#include "kv4.cuh"
#include "qrow_common.cuh"
#include "tc_common.cuh"

#include <math.h>

#include <algorithm>

namespace mrb {

constexpr int KD_MAX_ROWS = 512;   // rows a launch
constexpr int KD_MAX_STAGES = 6;
constexpr int KD_TILES = 2;  // tiles a unit: what a warp fetches, waits for and weighs in one go
constexpr int KD_UNIT = KD_TILES * KV4_TILE;
constexpr float KD_ROOM = 0x1p-7f;  // of fp16's range, kept for small weights: its largest are 2^15
constexpr int KD_CHUNK = 64;       // parts of a group summed at a time
constexpr int KD_COUNTERS = MRB_KV4_COUNTER_BYTES;  // of the workspace, one a CTA

__device__ unsigned g_kv4_timeouts = 0;

struct Kv4DecodeArgs {
  const __nv_bfloat16* q;
  __nv_bfloat16* out;
  Kv4Pool pool;
  const int32_t *block_table, *row_seq, *row_len;
  int32_t* error_flag;
  unsigned* counters;
  float* part;
  int64_t bt_stride, num_seqs;
  int row0, rows, hq, cap, stages, merge_bytes, by_group;  // cap: most tokens of a row
  uint32_t q_and, q_xor;            // applied to query pairs: a negative or zero scale
  float scale2;                     // |softmax scale| log2(e)
};

// warps an SM, by the registers that one needs
template <int NT>
constexpr int KD_SM_WARPS = NT == 2 ? 8 : 12;
static int kd_sm_warps(int nt) { return nt == 2 ? 8 : 12; }

// floats of one partial state: fragments, then (max, sum) of each column
template <int D, int NT>
constexpr int KD_PART = NT * (D / 16) * 128 + NT * 8 * 2;

__device__ __forceinline__ float fast_exp2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float fast_log2(float x) {
  float r;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ uint32_t max_bf16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ void mma_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                          uint32_t b0, uint32_t b1, const float* c) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
               : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ float low_half(uint32_t u) { return __uint_as_float(u << 16); }  // of a bf16 pair
__device__ __forceinline__ float high_half(uint32_t u) { return __uint_as_float(u & 0xffff0000u); }
template <int N>
__device__ __forceinline__ void load_words(uint32_t (&w)[N], const unsigned char* p) {
  if constexpr (N == 1) {
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  } else if constexpr (N == 2) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    w[0] = v.x, w[1] = v.y;
  } else {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
  }
}
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
               ::"r"(smem_u32(dst)), "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

// Units before each row, over all KV heads, in pre[0..rows]; returns their sum. Whole CTA. A
// group with tokens takes a unit for each 32 of them and an allowance of `extra`.
__device__ __forceinline__ int kd_prefix(const Kv4DecodeArgs& a, int extra, int* pre, int* wsum) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, threads = blockDim.x;
  const int per = (a.rows + threads - 1) / threads, r0 = min(tid * per, a.rows), r1 = min(r0 + per, a.rows);
  int mine = 0;
  for (int r = r0; r < r1; ++r) {
    const int all = a.row_len[a.row0 + r], len = min(all, a.cap);
    if (all > a.cap && blockIdx.x == 0 && a.error_flag) atomicOr(a.error_flag, MRB_KV_TOO_LONG);
    pre[r] = len > 0 ? ((len + KD_UNIT - 1) / KD_UNIT + extra) * a.pool.hkv : 0;
    mine += pre[r];
  }
  int incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += u;
  }
  if (lane == 31) wsum[warp] = incl;
  __syncthreads();
  int at = incl - mine, all = 0;
  for (int w = 0; w < threads / 32; ++w) {
    if (w < warp) at += wsum[w];
    all += wsum[w];
  }
  for (int r = r0; r < r1; ++r) {
    const int n = pre[r];
    pre[r] = at;
    at += n;
  }
  if (tid == 0) pre[a.rows] = all;
  __syncthreads();
  return all;
}
// the row that holds unit x
__device__ __forceinline__ int kd_row(const int* pre, int rows, int x) {
  int lo = 0, hi = rows;
  while (hi - lo > 1) {
    const int m = (lo + hi) >> 1;
    if (pre[m] <= x) lo = m; else hi = m;
  }
  return lo;
}

// What a state's (max, sum) weighs under the common maximum m. A state without a finite score is
// empty, or holds a NaN that has to stay.
__device__ __forceinline__ float kd_factor(float2 state, float m) {
  return state.x == -INFINITY ? (state.y == 0.f ? 0.f : 1.f) : fast_exp2(state.x - m);
}

template <int D, int G, int NT, int W>
__global__ void __launch_bounds__(W * 32, KD_SM_WARPS<NT> / W)
kv4_decode_kernel(const __grid_constant__ Kv4DecodeArgs a) {
  constexpr int NG = D / G, KW = G / 32, GI = G / 16, MI = D / 16, COLS = NT * 8;
  constexpr int BLOCK = kv4_block_bytes(D, G), CODES = kv4_codes_bytes(D), PARAMS = kv4_params_bytes(D, G);
  constexpr int STAGE = KD_TILES * BLOCK, FULL = KV4_TILE | KV4_TILE << 8;
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ __align__(8) uint64_t bars[W * KD_MAX_STAGES];
  __shared__ int lims[W * KD_MAX_STAGES];
  __shared__ __align__(8) float stat[W][COLS][2], qsum[NG][COLS], qscale[COLS], total[COLS], most[COLS];
  __shared__ int wsum[W], tally;
  __shared__ bool is_last;
  const int tid = threadIdx.x, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);  // the same for all lanes, and known to be
  const int group = a.hq / a.pool.hkv, S = a.stages;
  unsigned char* ring = smem + warp * S * STAGE;
  float4* merge = reinterpret_cast<float4*>(smem + W * S * STAGE);  // [W][NT * MI][32]: the warps' fragments
  uint4* qfrag = reinterpret_cast<uint4*>(smem + W * S * STAGE + a.merge_bytes);  // [NT][D / 32][32]
  int* pre = reinterpret_cast<int*>(qfrag + NT * (D / 32) * 32);
  uint64_t* bar = bars + warp * KD_MAX_STAGES;
  int* lim_of = lims + warp * KD_MAX_STAGES;
  if (lane == 0) {
    for (int i = 0; i < S; ++i) mbar_init(bar + i, 1);
    fence_proxy_async_smem();
  }
  if (tid == 0) tally = 0;
  pdl_launch_dependents();
  pdl_wait();
  const int extra = a.by_group ? 0 : W;
  const int T = kd_prefix(a, extra, pre, wsum);
  // rows without tokens
  for (int r = blockIdx.x; r < a.rows; r += gridDim.x)
    if (pre[r + 1] == pre[r])
      for (int i = tid; i < a.hq * D / 8; i += W * 32)
        reinterpret_cast<uint4*>(a.out + (int64_t)(a.row0 + r) * a.hq * D)[i] = make_uint4(0, 0, 0, 0);
  if (T == 0) return;
  // ---- this CTA's range of units [lo, hi); of the group that holds unit x (units [gs, gs + size)):
  // its parts, the first one's place in the workspace, and this CTA's part
  const int c = blockIdx.x;
  int lo, hi, row, head, size;
  int base = 0, more = 0, parts = 1, first = 0;
  if (a.by_group) {
    // every group is cut into equal parts of at most `target` units, one part a CTA: with G groups and
    // P CTAs, sum ceil(u / target) <= T / target + G <= P
    const int P = gridDim.x, target = max((T + P - a.rows * a.pool.hkv - 1) / (P - a.rows * a.pool.hkv), 4 * W);
    // the rows before this CTA's part are those whose parts end at or before it
    int seen = 0;
    row = 0;
    if (warp == 0) {
      int at = 0, found = -1;
      for (int r0 = 0; r0 < a.rows && found < 0; r0 += 32) {
        const int r = r0 + lane;
        const int mine = r < a.rows ? ((pre[r + 1] - pre[r]) / a.pool.hkv + target - 1) / target * a.pool.hkv : 0;
        int incl = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int u = __shfl_up_sync(0xffffffffu, incl, o);
          if (lane >= o) incl += u;
        }
        const unsigned has = __ballot_sync(0xffffffffu, mine > 0 && at + incl > c);
        if (has) {
          const int l = __ffs(has) - 1;
          found = r0 + l;
          at += __shfl_sync(0xffffffffu, incl - mine, l);
        } else {
          at += __shfl_sync(0xffffffffu, incl, 31);
        }
      }
      if (lane == 0) wsum[0] = found, tally = at;
    }
    __syncthreads();
    row = wsum[0];
    seen = tally;
    if (row < 0) return;  // fewer parts than CTAs
    size = (pre[row + 1] - pre[row]) / a.pool.hkv;
    parts = (size + target - 1) / target;
    head = (c - seen) / parts;
    first = seen + head * parts;
    const int j = c - first, gs = pre[row] + head * size;
    lo = gs + j * (size / parts) + min(j, size % parts);
    hi = lo + size / parts + (j < size % parts ? 1 : 0);
  } else {
    // equal ranges; the first `more` CTAs take one unit more than the others
    const int P = max(1, min((int)gridDim.x, T / (2 * W)));
    if (c >= P) return;
    base = T / P, more = T - base * P;
    lo = c * base + min(c, more), hi = lo + base + (c < more ? 1 : 0);
    row = kd_row(pre, a.rows, lo);
    size = (pre[row + 1] - pre[row]) / a.pool.hkv, head = (lo - pre[row]) / size;
  }
  auto cta_of = [&](int x) { return x < more * (base + 1) ? x / (base + 1) : more + (x - more * (base + 1)) / base; };
  const int n = hi - lo > warp ? (hi - lo - warp + W - 1) / W : 0;  // this warp's units

  // ---- requests: lane i holds the blocks of unit k0 + i of this warp, and how many of each one's
  // tokens count (0: an allowance unit, a tile past the row's end, or an unmapped one)
  uint32_t src[KD_TILES];  // in steps of 128 bytes
  int src_lim = 0, in_stage = 0;
  auto request = [&](int k) {  // unit k of this warp (whole warp)
    if (k >= n) return;
    if ((k & 31) == 0) {
      src_lim = 0;
      if (k + lane < n) {
        const int x = lo + warp + (k + lane) * W, r = kd_row(pre, a.rows, x);
        const int size = (pre[r + 1] - pre[r]) / a.pool.hkv, head = (x - pre[r]) / size;
        const int unit = x - pre[r] - head * size - extra;
        if (unit >= 0) {
          const int64_t seq = a.row_seq ? a.row_seq[a.row0 + r] : a.row0 + r;
          const int len = min(a.row_len[a.row0 + r], a.cap);
#pragma unroll
          for (int j = 0; j < KD_TILES; ++j) {
            const int tok = (unit * KD_TILES + j) * KV4_TILE, at = tok / a.pool.page_size;
            if (tok >= len) continue;
            const int page = seq >= 0 && seq < a.num_seqs ? a.block_table[seq * a.bt_stride + at] : -1;
            if (page >= 0 && page < a.pool.num_pages) {
              src[j] = (uint32_t)((a.pool.block(page, head, tok - at * a.pool.page_size, BLOCK) - a.pool.base) >> 7);
              src_lim |= min(KV4_TILE, len - tok) << (8 * j);
            } else if (a.error_flag) {
              atomicOr(a.error_flag, MRB_KV_UNMAPPED);
            }
          }
        }
      }
    }
    if (lane == (k & 31)) {
      uint64_t* b = bar + in_stage;
      unsigned char* dst = ring + in_stage * STAGE;
      lim_of[in_stage] = src_lim;
      if (src_lim & 255 && src_lim >> 8 && src[1] == src[0] + BLOCK / 128) {
        mbar_arrive_expect_tx(b, 2 * BLOCK);
        bulk_load(dst, a.pool.base + ((int64_t)src[0] << 7), 2 * BLOCK, b);
      } else if (src_lim) {
        mbar_arrive_expect_tx(b, ((src_lim & 255 ? 1 : 0) + (src_lim >> 8 ? 1 : 0)) * BLOCK);
        if (src_lim & 255) bulk_load(dst, a.pool.base + ((int64_t)src[0] << 7), BLOCK, b);
        if (src_lim >> 8) bulk_load(dst + BLOCK, a.pool.base + ((int64_t)src[1] << 7), BLOCK, b);
      } else {
        mbar_arrive(b);  // nothing to fetch
      }
    }
    if (++in_stage == S) in_stage = 0;
  };
  for (int k = 0; k < S - 1; ++k) request(k);

  const int tokA = (g & 1) ? 4 + ((g >> 1) ^ 1) : g >> 1;  // token of fragment row g (row g + 8: 8 more)
  const float zero[4] = {0.f, 0.f, 0.f, 0.f};
  int k = 0, stage = 0;
  unsigned phase = 0;
  for (;;) {  // one segment: the part of a group that this CTA's range holds
    const int gs = pre[row] + head * size, seg_end = min(hi, gs + size);
    const __nv_bfloat16* q0 = a.q + ((int64_t)(a.row0 + row) * a.hq + (int64_t)head * group) * D;
    {  // the next group's queries, on their way while this one is done
      const int nh = head + 1 < a.pool.hkv ? head + 1 : 0, nr = nh ? row : row + 1;
      if (warp == 0 && nr < a.rows) {
        const __nv_bfloat16* nq = a.q + ((int64_t)(a.row0 + nr) * a.hq + (int64_t)nh * group) * D;
        for (int i = lane * 64; i < group * D; i += 32 * 64) asm volatile("prefetch.global.L1 [%0];" ::"l"(nq + i));
      }
    }
    // queries as the B operand, scaled to fp16 range, and their sums by group; the warps share the
    // fragments (each finds the scale for itself)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      uint4 v[NG * KW];
      float far = 0.f;
#pragma unroll
      for (int i = 0; i < NG * KW; ++i) {
        v[i] = make_uint4(0, 0, 0, 0);
        if (nt * 8 + g < group)
          v[i] = __ldg(reinterpret_cast<const uint4*>(q0 + (nt * 8 + g) * D + i / KW * G + t * (G / 4) + i % KW * 8));
      }
#pragma unroll
      for (int i = 0; i < NG * KW; ++i) {
        uint32_t* u = reinterpret_cast<uint32_t*>(&v[i]);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          u[e] = (u[e] & a.q_and) ^ a.q_xor;
          far = max3(far, fabsf(low_half(u[e])), fabsf(high_half(u[e])));
        }
      }
      far = fmaxf(far, __shfl_xor_sync(0xffffffffu, far, 1));
      far = fmaxf(far, __shfl_xor_sync(0xffffffffu, far, 2));
      // 2^up brings the largest query to [2^13, 2^14); bounded so that 2^up and 2^-up are numbers
      const int up = max(-110, min(110, 140 - (int)(__float_as_uint(far) >> 23)));
      const float mul = __int_as_float((127 + up) << 23);
#pragma unroll
      for (int gr = 0; gr < NG; ++gr) {
        if ((nt * NG + gr) % W != warp) continue;
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < KW; ++i) {
          const uint4 x = v[gr * KW + i];
          float f[8] = {low_half(x.x), high_half(x.x), low_half(x.y), high_half(x.y),
                        low_half(x.z), high_half(x.z), low_half(x.w), high_half(x.w)};
#pragma unroll
          for (int e = 0; e < 8; ++e) f[e] *= mul, sum += f[e];
          // dimension pairs (e, e + 4), as nibbles e and e + 4 of a word share a register; odd
          // nibbles are 16 times their code
          qfrag[(nt * NG * KW + gr * KW + i) * 32 + lane] =
              make_uint4(pack_f16(f[0], f[4]), pack_f16(f[1] * 0.0625f, f[5] * 0.0625f), pack_f16(f[2], f[6]),
                         pack_f16(f[3] * 0.0625f, f[7] * 0.0625f));
        }
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        if (t == 0) qsum[gr][nt * 8 + g] = sum * 0x1p-24f;
      }
      // (not zero, which a masked score would make a NaN of)
      if (t == 0 && warp == 0) qscale[nt * 8 + g] = fmaxf(a.scale2 * __int_as_float((127 - up) << 23) * 0x1p24f, 0x1p-126f);
    }
    __syncthreads();  // and the last group's merge is over
    float cs[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) cs[nt][0] = qscale[nt * 8 + 2 * t], cs[nt][1] = qscale[nt * 8 + 2 * t + 1];
    // per column: the largest score mx; rel = 2^(mx - the largest log2(p s)), which O carries
    float o[NT][MI][4], mean[NT][NG][2], mx[NT][2], rel[NT][2], den[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int i = 0; i < MI; ++i) o[nt][i][0] = o[nt][i][1] = o[nt][i][2] = o[nt][i][3] = 0.f;
#pragma unroll
      for (int gr = 0; gr < NG; ++gr) mean[nt][gr][0] = mean[nt][gr][1] = 0.f;
      mx[nt][0] = mx[nt][1] = -INFINITY;
      rel[nt][0] = rel[nt][1] = 1.f;
      den[nt][0] = den[nt][1] = 0.f;
    }

    for (; k < n && lo + warp + k * W < seg_end; ++k) {
      if (!mbar_try_wait(bar + stage, phase) && !mbar_wait_bounded(bar + stage, phase) && lane == 0) {
        atomicAdd(&g_kv4_timeouts, 1u);
        if (a.error_flag) atomicOr(a.error_flag, MRB_KV_TIMEOUT);
      }
      __syncwarp();
      const int lim = lim_of[stage];
      const unsigned char* st = ring + stage * STAGE;
      request(k + S - 1);  // into the stage of the unit before this one
      if (++stage == S) stage = 0, phase ^= 1u;
      if (lim == 0) continue;
      // ---- S^T = K Q^T for the unit's tiles, scaled group by group
      float sc[KD_TILES][NT][4], top[KD_TILES][2];
#pragma unroll
      for (int j = 0; j < KD_TILES; ++j)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) sc[j][nt][0] = sc[j][nt][1] = sc[j][nt][2] = sc[j][nt][3] = 0.f;
      const unsigned char* ka = st + tokA * (D / 2) + t * (G / 8);
      const unsigned char* pa = st + 2 * CODES + tokA * NG * 4;
#pragma unroll
      for (int j = 0; j < KD_TILES; ++j)
#pragma unroll
        for (int gr = 0; gr < NG; ++gr) {
          uint32_t wa[KW], wb[KW];
          load_words<KW>(wa, ka + j * BLOCK + gr * (G / 2));
          load_words<KW>(wb, ka + j * BLOCK + 8 * (D / 2) + gr * (G / 2));
          float acc[NT][4];
#pragma unroll
          for (int i = 0; i < KW; ++i)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              const uint4 qf = qfrag[(nt * NG * KW + gr * KW + i) * 32 + lane];
              const uint32_t ua = wa[i], ub = wb[i], ha = ua >> 8, hb = ub >> 8;
              mma_16816(acc[nt], ua & 0x000f000fu, ub & 0x000f000fu, ua & 0x00f000f0u, ub & 0x00f000f0u, qf.x, qf.y,
                        i == 0 ? zero : acc[nt]);
              mma_16816(acc[nt], ha & 0x000f000fu, hb & 0x000f000fu, ha & 0x00f000f0u, hb & 0x00f000f0u, qf.z, qf.w,
                        acc[nt]);
            }
          const uint32_t pA = *reinterpret_cast<const uint32_t*>(pa + j * BLOCK + gr * 4);
          const uint32_t pB = *reinterpret_cast<const uint32_t*>(pa + j * BLOCK + 8 * NG * 4 + gr * 4);
          const float sA = low_half(pA), sB = low_half(pB), mA = high_half(pA), mB = high_half(pB);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            const float2 qs = *reinterpret_cast<const float2*>(&qsum[gr][nt * 8 + 2 * t]);
#pragma unroll
            for (int e = 0; e < 4; ++e)
              sc[j][nt][e] = fmaf(e < 2 ? sA : sB, acc[nt][e], fmaf(e < 2 ? mA : mB, e & 1 ? qs.y : qs.x, sc[j][nt][e]));
          }
        }
      // ---- the largest scale of each token's V
#pragma unroll
      for (int j = 0; j < KD_TILES; ++j)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t w[NG];
          load_words<NG>(w, pa + j * BLOCK + PARAMS + h * 8 * NG * 4);
          uint32_t most = w[0];
#pragma unroll
          for (int gr = 1; gr < NG; ++gr) most = max_bf16x2(most, w[gr]);
          top[j][h] = low_half(most) * KD_ROOM;
        }
      bool in[KD_TILES][2];
#pragma unroll
      for (int j = 0; j < KD_TILES; ++j) in[j][0] = in[j][1] = true;
      if (lim != FULL) {  // some tokens do not count; their places hold anything
#pragma unroll
        for (int j = 0; j < KD_TILES; ++j)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            in[j][h] = tokA + 8 * h < (lim >> (8 * j) & 255);
            top[j][h] = in[j][h] ? top[j][h] : 0.f;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int e = 0; e < 2; ++e) sc[j][nt][2 * h + e] = in[j][h] ? sc[j][nt][2 * h + e] : -INFINITY;
          }
      }
      // ---- p = 2^(score - mx); weights p s, times rel, go to fp16
      float p[KD_TILES][NT][4], big = 0.f;
      auto weigh = [&]() {
        big = 0.f;
#pragma unroll
        for (int j = 0; j < KD_TILES; ++j)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float v = fast_exp2(fmaf(sc[j][nt][e], cs[nt][e & 1], -mx[nt][e & 1]));
              p[j][nt][e] = v;
              big = max3(big, v, v * (top[j][e >> 1] * rel[nt][e & 1]));
            }
      };
      weigh();
      if (__any_sync(0xffffffffu, big > 256.f)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float m = -INFINITY, u = -INFINITY;
#pragma unroll
            for (int j = 0; j < KD_TILES; ++j)
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const float y = sc[j][nt][2 * h + e] * cs[nt][e];
                m = fmaxf(m, y);
                u = fmaxf(u, y + fast_log2(top[j][h]));
              }
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) {
              m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
              u = fmaxf(u, __shfl_xor_sync(0xffffffffu, u, d));
            }
            m = fmaxf(m, mx[nt][e]);
            // before a first number there are only zeros, or a NaN that stays
            const bool some = mx[nt][e] != -INFINITY;
            const float was = mx[nt][e] - fast_log2(rel[nt][e]);
            if (some) u = fmaxf(u, was);
            u = fmaxf(u, m - 100.f);  // scales that vanish
            const float f = some ? fast_exp2(mx[nt][e] - m) : 1.f, fo = some ? fast_exp2(was - u) : 1.f;
            if (m != -INFINITY) mx[nt][e] = m, rel[nt][e] = fast_exp2(m - u);
            den[nt][e] *= f;
#pragma unroll
            for (int gr = 0; gr < NG; ++gr) mean[nt][gr][e] *= f;
#pragma unroll
            for (int i = 0; i < MI; ++i) o[nt][i][e] *= fo, o[nt][i][e + 2] *= fo;
          }
        weigh();
      }
#pragma unroll
      for (int j = 0; j < KD_TILES; ++j) {
        // ---- O^T += V^T P^T, weights scaled group by group
        const unsigned char* bl = st + j * BLOCK;
        uint32_t pA[NG], pB[NG];
        load_words<NG>(pA, bl + 2 * CODES + PARAMS + tokA * NG * 4);
        load_words<NG>(pB, bl + 2 * CODES + PARAMS + (tokA + 8) * NG * 4);
        if (lim != FULL) {
#pragma unroll
          for (int gr = 0; gr < NG; ++gr) pA[gr] = in[j][0] ? pA[gr] : 0u, pB[gr] = in[j][1] ? pB[gr] : 0u;
        }
        float wt[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          den[nt][0] += p[j][nt][0] + p[j][nt][2];
          den[nt][1] += p[j][nt][1] + p[j][nt][3];
#pragma unroll
          for (int e = 0; e < 4; ++e) wt[nt][e] = p[j][nt][e] * rel[nt][e & 1];
        }
        // the four tokens of this lane's V fragment columns 2t, 2t + 1, 2t + 8, 2t + 9
        const unsigned char* v0 = bl + CODES + t * (D / 2);
        const unsigned char* v1 = bl + CODES + (4 + (t ^ 1)) * (D / 2);
#pragma unroll
        for (int gr = 0; gr < NG; ++gr) {
          const float sA = low_half(pA[gr]), sB = low_half(pB[gr]), mA = high_half(pA[gr]), mB = high_half(pB[gr]);
          uint32_t pb[NT][2];
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            pb[nt][0] = transpose_8x8(pack_f16(wt[nt][0] * sA, wt[nt][1] * sA));
            pb[nt][1] = transpose_8x8(pack_f16(wt[nt][2] * sB, wt[nt][3] * sB));
            mean[nt][gr][0] = fmaf(p[j][nt][0], mA, fmaf(p[j][nt][2], mB, mean[nt][gr][0]));
            mean[nt][gr][1] = fmaf(p[j][nt][1], mA, fmaf(p[j][nt][3], mB, mean[nt][gr][1]));
          }
          constexpr int VW = G == 128 ? 2 : 1;
          uint32_t w[4][VW];
          const int at = gr * (G / 2) + (G == 32 ? 4 * (g >> 1) : g * (G / 16));
          load_words<VW>(w[0], v0 + at);
          load_words<VW>(w[1], v1 + at);
          load_words<VW>(w[2], v0 + 8 * (D / 2) + at);
          load_words<VW>(w[3], v1 + 8 * (D / 2) + at);
#pragma unroll
          for (int i = 0; i < VW; ++i)
#pragma unroll
            for (int h = 0; h < (G == 32 ? 1 : 2); ++h) {
              const uint32_t sel = G == 32 ? ((g & 1) ? 0x7632u : 0x5410u) : h ? 0x7632u : 0x5410u;
              const uint32_t xa = __byte_perm(w[0][i], w[1][i], sel), xb = __byte_perm(w[2][i], w[3][i], sel);
              const uint32_t ya = xa >> 8, yb = xb >> 8;
              const int at_o = gr * GI + i * 4 + h * 2;
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                mma_16816(o[nt][at_o], xa & 0x000f000fu, xa & 0x00f000f0u, xb & 0x000f000fu, xb & 0x00f000f0u,
                          pb[nt][0], pb[nt][1], o[nt][at_o]);
                mma_16816(o[nt][at_o + 1], ya & 0x000f000fu, ya & 0x00f000f0u, yb & 0x000f000fu, yb & 0x00f000f0u,
                          pb[nt][0], pb[nt][1], o[nt][at_o + 1]);
              }
            }
        }
      }
      __syncwarp();  // every lane is done with the stage before it is requested again
    }

    // ---- segment end: the CTAs that hold units of this group; none here: nothing to add
    if (!a.by_group) first = cta_of(gs + extra), parts = cta_of(gs + size - 1) - first + 1;
    if (c >= first) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float all = den[nt][e];
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) all += __shfl_xor_sync(0xffffffffu, all, d);
          const float f = 1.f / rel[nt][e];
#pragma unroll
          for (int gr = 0; gr < NG; ++gr) {
            float y = mean[nt][gr][e];
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) y += __shfl_xor_sync(0xffffffffu, y, d);
#pragma unroll
            for (int i = gr * GI; i < (gr + 1) * GI; ++i) {
              o[nt][i][e] = fmaf(o[nt][i][e] * 0x1p24f, f, y);
              o[nt][i][e + 2] = fmaf(o[nt][i][e + 2] * 0x1p20f, f, y);  // odd nibbles: 16 times their code
            }
          }
          if (g == 0) stat[warp][nt * 8 + 2 * t + e][0] = mx[nt][e], stat[warp][nt * 8 + 2 * t + e][1] = all;
        }
#pragma unroll
        for (int i = 0; i < MI; ++i)
          merge[(warp * NT * MI + nt * MI + i) * 32 + lane] =
              make_float4(o[nt][i][0], o[nt][i][2], o[nt][i][1], o[nt][i][3]);
      }
      __syncthreads();
      // a CTA's part lies at its own number; where ranges are cut anywhere, a CTA may end one group
      // and begin another, and the begun one's part lies after all others
      float* mine = a.part + (int64_t)(c == first && !a.by_group ? gridDim.x + c : c) * KD_PART<D, NT>;
      auto part_of = [&](int j) {
        return a.part + (int64_t)(j == 0 && !a.by_group ? (int)gridDim.x + first : first + j) * KD_PART<D, NT>;
      };
      __nv_bfloat16* out = a.out + ((int64_t)(a.row0 + row) * a.hq + (int64_t)head * group) * D;
      // items: two consecutive dimensions of one column, [NT * MI][lane][column of the lane's two]
      auto column = [&](int item) { return (item >> 6) / MI * 8 + 2 * ((item >> 1) & 3) + (item & 1); };
      auto write_out = [&](int item, float2 v, float l) {
        const int i = (item >> 6) % MI, col = column(item), d = i / GI * G + ((item >> 3) & 7) * (G / 8) + 2 * (i % GI);
        if (col >= group) return;
        const float inv = l == 0.f ? 0.f : 1.f / l;
        *reinterpret_cast<uint32_t*>(out + col * D + d) = pack_bf16(v.x * inv, v.y * inv);
      };
      constexpr int ITEMS = NT * MI * 64, PER = (ITEMS + W * 32 - 1) / (W * 32);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const int col = nt * 8 + 2 * ((tid >> 1) & 3) + (tid & 1);  // of all this thread's items
        float m = -INFINITY, l = 0.f, f[W];
#pragma unroll
        for (int u = 0; u < W; ++u) m = fmaxf(m, stat[u][col][0]);
#pragma unroll
        for (int u = 0; u < W; ++u) {
          f[u] = kd_factor(make_float2(stat[u][col][0], stat[u][col][1]), m);
          l = fmaf(stat[u][col][1], f[u], l);
        }
        if (parts > 1 && tid < 8) __stcg(reinterpret_cast<float2*>(mine + NT * MI * 128) + col, make_float2(m, l));
        for (int item = nt * MI * 64 + tid; item < (nt + 1) * MI * 64; item += W * 32) {
          const float2* m2 = reinterpret_cast<const float2*>(merge) + item;
          float2 v = make_float2(0.f, 0.f);
#pragma unroll
          for (int w = 0; w < W; ++w) {
            const float2 u = m2[w * NT * MI * 64];
            v.x = fmaf(u.x, f[w], v.x);
            v.y = fmaf(u.y, f[w], v.y);
          }
          if (parts == 1) write_out(item, v, l);
          else __stcg(reinterpret_cast<float2*>(mine) + item, v);
        }
      }
      if (parts > 1) {
        __threadfence();
        __syncthreads();
        if (tid == 0) is_last = atomicAdd(&a.counters[first], 1u) == (unsigned)(parts - 1);
        __syncthreads();
        if (is_last) {
          __threadfence();
          auto stat_of = [&](int j, int col) {
            return __ldcg(reinterpret_cast<const float2*>(part_of(j) + NT * MI * 128) + col);
          };
          // (max, sum) of the first parts, then each chunk's factors
          float2* pf = reinterpret_cast<float2*>(merge);  // [KD_CHUNK][COLS]
          for (int i = tid; i < min(parts, KD_CHUNK) * COLS; i += W * 32) pf[i] = stat_of(i / COLS, i % COLS);
          __syncthreads();
          for (int col = warp; col < COLS; col += W) {
            float m = -INFINITY, l = 0.f;
            for (int j = lane; j < parts; j += 32) m = fmaxf(m, (j < KD_CHUNK ? pf[j * COLS + col] : stat_of(j, col)).x);
            m = warp_max(m);
            for (int j = lane; j < parts; j += 32) {
              const float2 u = j < KD_CHUNK ? pf[j * COLS + col] : stat_of(j, col);
              l = fmaf(u.y, kd_factor(u, m), l);
            }
            l = warp_sum(l);
            if (lane == 0) total[col] = l, most[col] = m;
          }
          // a thread takes its items together, up to 24 loads in flight
          constexpr int AHEAD = 24 / PER;
          float2 v[PER];
#pragma unroll
          for (int e = 0; e < PER; ++e) v[e] = make_float2(0.f, 0.f);
          for (int c0 = 0; c0 < parts; c0 += KD_CHUNK) {
            const int count = min(KD_CHUNK, parts - c0);
            __syncthreads();
            for (int i = tid; i < count * COLS; i += W * 32) {
              const float2 u = c0 == 0 ? pf[i] : stat_of(c0 + i / COLS, i % COLS);
              pf[i].x = kd_factor(u, most[i % COLS]);
            }
            __syncthreads();
            for (int j0 = 0; j0 < count; j0 += AHEAD) {
              float2 u[AHEAD][PER];
#pragma unroll
              for (int j = 0; j < AHEAD; ++j)
#pragma unroll
                for (int e = 0; e < PER; ++e)
                  if (j0 + j < count && tid + e * W * 32 < ITEMS)
                    u[j][e] = __ldcg(reinterpret_cast<const float2*>(part_of(c0 + j0 + j)) + tid + e * W * 32);
#pragma unroll
              for (int j = 0; j < AHEAD; ++j)
#pragma unroll
                for (int e = 0; e < PER; ++e)
                  if (j0 + j < count && tid + e * W * 32 < ITEMS) {
                    const float f = pf[(j0 + j) * COLS + column(tid + e * W * 32)].x;
                    v[e].x = fmaf(u[j][e].x, f, v[e].x);
                    v[e].y = fmaf(u[j][e].y, f, v[e].y);
                  }
            }
          }
#pragma unroll
          for (int e = 0; e < PER; ++e)
            if (tid + e * W * 32 < ITEMS) write_out(tid + e * W * 32, v[e], total[column(tid + e * W * 32)]);
          if (tid == 0) a.counters[first] = 0u;  // ready for the next launch
        }
      }
    }
    if (seg_end == hi) break;
    if (++head == a.pool.hkv) {  // the next group: of the next row that has tokens
      head = 0;
      do ++row;
      while (pre[row + 1] == pre[row]);
      size = (pre[row + 1] - pre[row]) / a.pool.hkv;
    }
  }
  // every unit was waited for; after a wait that ran out, wait (bounded) once more for each stage's
  // last copy, so that none is still landing when the CTA ends
  for (int j = max(0, n - S); j < n; ++j) mbar_wait_bounded(bar + j % S, (unsigned)(j / S) & 1u);
}

// Warps a CTA, twelve an SM in all (eight where two column blocks need more registers). Few groups,
// of a long context, are each cut into many parts, whose sum is the last CTA's work: CTAs of a
// whole SM leave the fewest (131071 tokens x 28/4 heads: 37 us, against 49 with four warps and 82 with
// two). Else small CTAs: a group's end then holds up few warps. 32 rows of 256..4096 tokens x 32/4 heads:
// 29 us with four warps, 31 with two, 35 with twelve; 256 rows x 32/8 heads of 256 tokens: 45 us with two,
// 49 with four, 78 with twelve. (Single calls, with a cold L2 and the launch: 7 us more than calls in a row.)
static int kd_warps(int64_t rows, int64_t hkv, int nt) {
  const int64_t groups = rows * hkv;
  if (nt == 1 && groups >= 4 * num_sms()) return 2;
  return groups >= 64 ? 4 : kd_sm_warps(nt);
}

static int64_t kd_row_units(int64_t hkv, int64_t max_total, int warps) {
  return hkv * ((max_total + KD_UNIT - 1) / KD_UNIT + warps);
}
static int kd_grid(int64_t rows, int64_t hkv, int64_t max_total, int nt, int warps) {
  const int64_t ctas = (int64_t)num_sms() * (kd_sm_warps(nt) / warps);
  const int64_t want = rows * std::max(kd_row_units(hkv, max_total, warps) / (2 * warps), 2 * hkv);
  return (int)std::max<int64_t>(1, std::min(std::min<int64_t>(ctas, KD_COUNTERS / 4), want));
}
static size_t kd_workspace(int64_t rows, int64_t hq, int64_t hkv, int64_t d, int64_t max_total) {
  const int nt = hq / hkv > 8 ? 2 : 1;
  const int grid = kd_grid(rows, hkv, max_total, nt, kd_warps(rows, hkv, nt));
  return KD_COUNTERS + (size_t)grid * 2 * 4 * (size_t)(nt * (d / 16) * 128 + nt * 16);
}

template <int D, int G, int NT, int W>
static int launch_decode(Kv4DecodeArgs& a, int64_t rows, int64_t max_total, cudaStream_t s) {
  const char* what = "kv4_paged_attention";
  const int64_t units = kd_row_units(a.pool.hkv, max_total, W);
  if (units > INT32_MAX) return fail(MRB_ERR_UNSUPPORTED, "%s: too many heads of too many tokens", what);
  const int64_t step = std::min<int64_t>(KD_MAX_ROWS, INT32_MAX / units);
  for (int64_t r0 = 0; r0 < rows; r0 += step) {
    a.row0 = (int)r0;
    a.rows = (int)std::min(step, rows - r0);
    const int grid = kd_grid(a.rows, a.pool.hkv, max_total, NT, W);
    // the warps' states, or two numbers for each column of a chunk of parts
    a.merge_bytes = std::max(W * NT * (D / 16) * 512, KD_CHUNK * NT * 8 * 8);
    a.by_group = (int64_t)a.rows * a.pool.hkv * 2 <= grid;
    const size_t fixed = (size_t)a.merge_bytes + NT * (D / 32) * 512 + (size_t)(a.rows + 1) * 4;
    const size_t room = 216 * 1024 * W / KD_SM_WARPS<NT>;  // of 227 KB an SM
    a.stages = (int)std::min<size_t>(KD_MAX_STAGES, (room - fixed) / ((size_t)W * KD_TILES * kv4_block_bytes(D, G)));
    const size_t smem = fixed + (size_t)W * a.stages * KD_TILES * kv4_block_bytes(D, G);
    const int rc = ensure_dynamic_smem((const void*)kv4_decode_kernel<D, G, NT, W>, smem, what);
    if (rc != MRB_OK) return rc;
    launch_kernel(kv4_decode_kernel<D, G, NT, W>, dim3(grid), dim3(W * 32), smem, s, true, a);
    const int st = launch_status(what);
    if (st != MRB_OK) return st;
  }
  return MRB_OK;
}
template <int D, int G>
static int launch_decode(Kv4DecodeArgs& a, int64_t rows, int64_t max_total, cudaStream_t s) {
  const int nt = a.hq / a.pool.hkv > 8 ? 2 : 1, warps = kd_warps(rows, a.pool.hkv, nt);
  if (nt == 1)
    return warps == 2   ? launch_decode<D, G, 1, 2>(a, rows, max_total, s)
           : warps == 4 ? launch_decode<D, G, 1, 4>(a, rows, max_total, s)
                        : launch_decode<D, G, 1, KD_SM_WARPS<1>>(a, rows, max_total, s);
  return warps == 4 ? launch_decode<D, G, 2, 4>(a, rows, max_total, s) : launch_decode<D, G, 2, 8>(a, rows, max_total, s);
}

}  // namespace mrb

extern "C" int64_t mrb_kv4_paged_attention_timeouts(void) {
  unsigned v = 0;
  if (cudaMemcpyFromSymbol(&v, mrb::g_kv4_timeouts, sizeof(v)) != cudaSuccess) return -1;
  return (int64_t)v;
}

extern "C" size_t mrb_kv4_paged_attention_workspace(int64_t rows, int64_t hq, int64_t hkv, int64_t head_dim,
                                                    int64_t max_total_tokens) {
  if (rows < 1 || hkv < 1 || hq < 1 || max_total_tokens < 1) return 0;
  return mrb::kd_workspace(rows, hq, hkv, head_dim, max_total_tokens);
}

extern "C" int mrb_kv4_paged_attention(const void* q, int64_t rows, int64_t hq, int64_t hkv, int64_t head_dim,
                                       int64_t group, const void* pool, int64_t num_pages, int64_t page_size,
                                       int64_t stride_page, int64_t stride_head, const int32_t* block_table,
                                       int64_t num_seqs, int64_t block_table_stride, int64_t max_pages_per_seq, const int32_t* row_seq,
                                       const int32_t* row_len, float scale, int64_t max_total_tokens, void* out,
                                       void* workspace, size_t workspace_bytes, int32_t* error_flag, void* stream) {
  using namespace mrb;
  const char* what = "kv4_paged_attention";
  Kv4DecodeArgs a = {};
  const int rc = kv4_check_attention(what, q, rows, rows, hq, hkv, head_dim, group, pool, num_pages, page_size,
                                     stride_page, stride_head, block_table, num_seqs, block_table_stride, max_pages_per_seq,
                                     row_len, scale, out, &a.pool);
  if (rc != MRB_OK) return rc;
  if (max_total_tokens < 0) return fail(MRB_ERR_ARG, "%s: bad sizes", what);
  if (rows == 0) {
    clear_error();
    return MRB_OK;
  }
  const int64_t most = std::min(max_total_tokens, max_pages_per_seq * page_size);
  const size_t need = most > 0 ? kd_workspace(rows, hq, hkv, head_dim, most) : 0;
  if (need && (!workspace || workspace_bytes < need || !aligned(workspace, 16)))
    return fail(MRB_ERR_ARG, "%s: needs a 16-byte aligned workspace of %zu bytes", what, need);
  a.q = (const __nv_bfloat16*)q;
  a.out = (__nv_bfloat16*)out;
  a.block_table = block_table;
  a.row_seq = row_seq;
  a.row_len = row_len;
  a.error_flag = error_flag;
  a.counters = (unsigned*)workspace;
  a.part = (float*)((char*)workspace + KD_COUNTERS);
  a.bt_stride = block_table_stride;
  a.num_seqs = num_seqs;
  a.hq = (int)hq;
  a.cap = (int)most;
  a.q_and = scale == 0.f ? 0u : 0xffffffffu;
  a.q_xor = scale < 0.f ? 0x80008000u : 0u;
  a.scale2 = (scale == 0.f ? 1.f : fabsf(scale)) * 1.4426950408889634f;
  cudaStream_t s = (cudaStream_t)stream;
  if (head_dim == 64) return group == 32 ? launch_decode<64, 32>(a, rows, most, s) : launch_decode<64, 64>(a, rows, most, s);
  if (group == 32) return launch_decode<128, 32>(a, rows, most, s);
  if (group == 64) return launch_decode<128, 64>(a, rows, most, s);
  return launch_decode<128, 128>(a, rows, most, s);
}
