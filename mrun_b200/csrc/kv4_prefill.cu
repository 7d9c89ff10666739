// Causal attention of ragged query blocks over the 4-bit paged K/V pool, on the tcgen05 tensor cores.
//
// A row tile is 256 query rows of one KV head: as many tokens of one request as fit with all the
// group's query heads (row = token * group + head), in two halves of 128 rows. A CTA walks its keys in
// steps of 128 tokens:
//   S_i = Q_i K^T (A, B in shared memory, fp32 in TMEM), W_i = 2^(S_i - M) (two threads a row), back to
//   TMEM in fp16 over S_i, O_i += W_i V (A in TMEM, B in shared memory, fp32 in TMEM).
// Eight warps turn codes into fp16 tiles in shared memory, once for both halves; sixteen do the
// softmax, eight a half; one lane issues the products. While one half's scores are in the softmax the
// other's products run, and the next tile's K is ready before its turn.
//
// One CTA an SM takes an equal share of all tiles' keys, laid end to end (see the plan below), tile by
// tile: the next one's codes are fetched while the last products of this one run.
//
// K and V are m + s c by one fp16 fused multiply-add a pair of codes, which a mask leaves as the
// subnormal c 2^-24 (an odd nibble: 16 c 2^-24) with the factors taken into s. To stay inside fp16,
// a tile of K is scaled by a power of two to at most 16 2^-10, where fp16 ends 2^-18 below the largest
// key; where its tokens' sizes differ by more than 2^6, codes are made whole numbers first and the tile is
// scaled to at most 2^15. V is scaled by the tile or, where its tokens' sizes differ as much, token by
// token; scores, weights and row sums take the powers
// back exactly (a weight carries its token's power, so the running maximum M is that of score plus
// power, and a token with huge values and no weight costs others no precision). Queries are scaled
// to fp16 by a power of two a row. Weights are rounded to fp16 (11 bits); M moves only when a row's
// weights of one step pass 2^13 together (so that no maximum is taken in most steps), and O is
// rescaled in TMEM then. A weight 2^-25 below 2^M vanishes: n such tokens cost at most n 2^-25 of an output.
//
// Bound by the softmax's exponentials (16 a clock an SM: 2048 clocks a step of 256 rows x 128 keys,
// as many as the products take at the tensor peak) and by shared memory (the products' operands and
// the dequantised tiles: 2048 clocks a step). A step takes 4,000 clocks: the weights lie over the
// scores, so a half's next scores wait for the product that reads its weights. 4096 tokens at 16384 x
// 28/4 heads: 1.07 ms in single calls after a pause, 1010 TFLOP/s, and 1.16 one after another, under the
// power limit; 512 tokens alone: 29 us, of which 7 us are the plan and the first loads, 4 us a tile's
// queries, and 5 us its first step.
#include "kv4.cuh"
#include "qrow_common.cuh"
#include "tc_common.cuh"

#include <algorithm>

namespace mrb {

constexpr int KF_ROWS = 256;  // query rows a CTA
constexpr int KF_KEYS = 128;  // keys a step
// three kinds of warpgroups: softmax (four), codes to tiles (two), the products (one lane of the last).
// Launched with 72 registers a thread; 4 x 88 + 2 x 64 + 24 is seven times that.
constexpr int KF_SOFTMAX = 512, KF_FILL = 256, KF_THREADS = 896;
constexpr int KF_PASSES = KF_KEYS / (KF_FILL / 4);  // four lanes a token
constexpr int KF_SOFTMAX_REGS = 88, KF_FILL_REGS = 64, KF_ISSUE_REGS = 24;
constexpr int KF_META = 4;  // steps whose scales are kept
constexpr int KF_PIECES = 16;  // pieces planned in one go
constexpr int KF_TILE_COST = 640;  // of a row tile besides its steps (20,000 clocks; a step: 4,000), in keys
constexpr int KF_LEAST = 4;  // steps: no piece at a divided tile's ends is shorter (dividing: 45,000 clocks)
// Keys a CTA, before more CTAs divide tiles: joining many parts costs what it saves (8 tokens at 16000 x
// 28/4 heads: 63 us, with 512 keys 87, with 2048 72).
constexpr int KF_LEAST_KEYS = 1024;
constexpr int KF_COUNTERS = MRB_KV4_COUNTER_BYTES;  // of the workspace, one a CTA

__device__ unsigned g_kv4_prefill_timeouts = 0;

struct Kv4PrefillArgs {
  const __nv_bfloat16* q;
  __nv_bfloat16* out;
  Kv4Pool pool;
  const int32_t *block_table, *row_seq, *row_len, *q_starts;
  int32_t* error_flag;
  unsigned* counters;
  float* part;
  int64_t tokens, bt_stride, num_seqs;
  int rows, hq, cap;
  bool zero_rest;  // query tokens of no block give zeros
  uint32_t page_magic, group_magic;  // of a page's 16-token blocks and of a group, as kf_divide takes them
  uint32_t q_and, q_xor;  // applied to query pairs: a negative or zero scale
  float scale2;           // |softmax scale| log2(e)
};

__device__ __forceinline__ void umma_f16_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t desc_b, uint32_t idesc,
                                            bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, {%5, %6, %7, %8}, p;\n\t}"
      ::"r"(tmem_d), "r"(tmem_a), "l"(desc_b), "r"(idesc), "r"((uint32_t)accumulate), "r"(0u), "r"(0u), "r"(0u), "r"(0u)
      : "memory");
}
// 32 consecutive 32-bit TMEM columns of this thread's lane, stored; completed by tmem_wait_st.
__device__ __forceinline__ void tmem_st_32cols(uint32_t taddr, const uint32_t* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};"
      ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]),
      "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]),
      "r"(v[18]), "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]),
      "r"(v[27]), "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
      : "memory");
}
// 16 columns of this thread's lane on their way to registers, which hold them after tmem_wait_ld (the
// wait names the registers so that nothing reads them before it).
__device__ __forceinline__ void tmem_ld_16cols_async(uint32_t taddr, uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
        "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_wait_ld(uint32_t (&v)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]), "+r"(v[8]),
                 "+r"(v[9]), "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15])::"memory");
}
__device__ __forceinline__ void tmem_ld_8cols_async(uint32_t taddr, uint32_t (&v)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7])
               : "r"(taddr));
}
__device__ __forceinline__ void tmem_wait_ld(uint32_t (&v)[8]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7])::"memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// A token-major tile [128 tokens][D] of fp16 as the N x K operand of W V: 128-byte swizzled rows of 64
// dimensions, 8-token atoms 1024 B apart (stride byte offset), the second 64 dimensions 16 KB on
// (leading byte offset); the dimensions are the operand's contiguous (MN) axis.
__device__ __forceinline__ uint64_t kf_desc_v(uint32_t saddr) {
  uint64_t d = (uint64_t)((saddr >> 4) & 0x3FFFu);
  d |= (uint64_t)(16384 >> 4) << 16;
  d |= (uint64_t)(1024 >> 4) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;
  return d;
}

__device__ __forceinline__ void tmem_st_16cols(uint32_t taddr, const uint32_t* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
      ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]),
      "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st_8cols(uint32_t taddr, const uint32_t* v) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), "r"(v[0]),
               "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}

// two fp32 operations in one instruction
__device__ __forceinline__ uint64_t kf_pair(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ float2 kf_split(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t kf_fma_pair(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t kf_add_pair(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float kf_exp2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float kf_pow2(int e) {  // 2^e for -149 <= e <= 127
  return e >= -126 ? __int_as_float((e + 127) << 23) : __int_as_float(1 << (e + 149));
}
__device__ __forceinline__ uint32_t kf_half2(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t kf_fma2(uint32_t a, uint32_t b, uint32_t c) {
  const __half2 r = __hfma2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b),
                            *reinterpret_cast<const __half2*>(&c));
  return *reinterpret_cast<const uint32_t*>(&r);
}
template <int N>
__device__ __forceinline__ void kf_more_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void kf_fewer_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

template <int N>
__device__ __forceinline__ void kf_copy(void* dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(smem_u32(dst)), "l"(src), "n"(N) : "memory");
}

__device__ __forceinline__ float kf_max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
// n / d for 0 <= n < 2^27: magic is 2^32 / d rounded up (0: d is 1), one too many at most
__device__ __forceinline__ int kf_divide(int n, int d, uint32_t magic) {
  if (magic == 0) return n;
  const int q = (int)__umulhi((uint32_t)n, magic);
  return q * d > n ? q - 1 : q;
}

__device__ __forceinline__ void kf_pair_sync(int id) { asm volatile("bar.sync %0, 64;" ::"r"(id) : "memory"); }
__device__ __forceinline__ bool kf_elected() {  // true in one lane, the same each time
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
  return p != 0;
}

// the line in equal shares: `share` keys, and one more in `rest` of them, spread evenly
struct KfCuts {
  int64_t share;
  int rest, ctas;
  __device__ __forceinline__ int64_t at(int k) const { return share * k + (unsigned)(rest * k) / (unsigned)ctas; }
  // the first cut at x or after it
  __device__ __forceinline__ int first(int64_t x) const {
    int k = max(0, min((int)((float)x / (float)max(share, (int64_t)1)), ctas));
    while (k > 0 && at(k - 1) >= x) --k;
    while (k < ctas && at(k) < x) ++k;
    return k;
  }
};
// One CTA's share of one tile: steps [j0, j1) of the tile's `steps`
struct KfPiece {
  int64_t seq;
  int q0, first, last;  // the block's first query; the tile's tokens in the block
  int before;           // cached tokens before the block
  int head, keys, steps, j0, j1;
  int low, parts;  // of a divided tile: CTAs low - 1 .. low + parts - 2 hold its parts in order
};

struct KfShared {
  float power[KF_META][KF_KEYS];  // log2 of each token's V scale (-inf: not there, NaN: V holds one)
  float k_scale[KF_META], v_power[KF_META], v_undo[KF_META];
  int uniform[KF_META];  // all tokens there, with the tile's power
  __align__(16) float red[2][KF_FILL / 32][4];
  uint64_t s_full[2], w_full[2], o_full[2], o_done[2], q_full;
  uint64_t k_full[2], k_empty[2], v_full[2], v_empty[2], meta_full[KF_META];
  float top[2][2][128];  // the halves' largest scores of a row, then their sums
  int seek[2][4][2];     // a pair's wish to move the maximum, by turn
  uint32_t tmem;
  int dead;  // a wait ran out: no later one waits
  KfPiece piece[KF_PIECES];
  int pieces, more, joins;
  int rest;  // the first query of no block
  int cursor_row, cursor_tile, cursor_head;  // of the plan: where it goes on (row -1: not begun)
  int64_t cursor_at;
  KfCuts cuts;
  float query_scale[2][128];
};

// Bounded wait; after one ran out anywhere in the CTA none waits again (the outputs are void then, and
// counted as such).
__device__ __forceinline__ void kf_wait(uint64_t* bar, unsigned parity, KfShared& sh) {
  for (int i = 0; i < (1 << 20); ++i) {
    if (mbar_try_wait(bar, parity)) return;
    if ((i & 255) == 0 && *(volatile int*)&sh.dead) return;
  }
  if (atomicExch(&sh.dead, 1) == 0) atomicAdd(&g_kv4_prefill_timeouts, 1u);
}

__device__ __forceinline__ void kf_all_sync() { asm volatile("bar.sync 0, 896;" ::: "memory"); }

// ---- the plan
//
// The work is measured in keys: a tile is as long as the keys that its last token sees, and KF_TILE_COST
// more. All tiles in a line (by request, tile, head) are cut into equal shares, one a CTA, so that every
// SM has as much to do whatever the blocks' lengths (4096 tokens at 16384, 456 tiles on 148 SMs: a
// sixth less time than with whole tiles only, where twelve of them made a last round; 64 tokens at 8000, 16
// tiles: 61 us against 155). A tile under a cut is divided at a step, or goes to one side as a whole if
// the cut is within KF_LEAST steps of its ends.
struct KfBlock {
  int q0, count, tiles;
  int64_t base;  // keys before the block
};
__device__ __forceinline__ KfBlock kf_block(const Kv4PrefillArgs& a, int r, int span) {
  KfBlock b;
  b.q0 = a.q_starts[r];
  b.count = a.q_starts[r + 1] - b.q0;
  if (b.q0 < 0 || (int64_t)b.q0 + b.count > a.tokens) b.count = 0;  // not a block of these queries
  b.tiles = b.count > 0 ? (b.count + span - 1) / span : 0;
  b.base = max(0, min(max(a.row_len[r], 0), a.cap) - b.count);
  return b;
}
// the length of a block's first t < tiles tiles of one head, and of all
__device__ __forceinline__ int64_t kf_length(const KfBlock& b, int span, int64_t t) {
  const int64_t whole = t < b.tiles ? span * (t * (t + 1) / 2) : b.tiles ? span * (t * (t - 1) / 2) + b.count : 0;
  return t * (b.base + KF_TILE_COST) + whole;
}
// One warp lists this CTA's next pieces. (A function of its own, as kf_join, so that its variables leave
// the softmax its registers.)
__device__ __noinline__ void kf_plan(const Kv4PrefillArgs& a, KfShared& sh, int span, int lane) {
  const int hkv = a.pool.hkv, cta = blockIdx.x;
  if (sh.cursor_row < 0) {
    if (lane == 0) sh.rest = max(0, a.q_starts[a.rows]);
    int64_t work = 0, tiles = 0;
    for (int r = lane; r < a.rows; r += 32) {
      const KfBlock b = kf_block(a, r, span);
      if (b.count > 0 && a.row_len[r] > a.cap && cta == 0 && a.error_flag) atomicOr(a.error_flag, MRB_KV_TOO_LONG);
      work += kf_length(b, span, b.tiles);
      tiles += b.tiles;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      work += __shfl_xor_sync(0xffffffffu, work, o);
      tiles += __shfl_xor_sync(0xffffffffu, tiles, o);
    }
    work *= hkv;
    tiles *= hkv;
    // no more CTAs than keep a tile's parts few, but enough that no two whole tiles share one needlessly
    const int64_t most = max(work / KF_LEAST_KEYS, 2 * tiles);
    const int ctas = (int)max((int64_t)1, min((int64_t)gridDim.x, most));
    // the block under this share's first key
    int64_t at = 0;
    int row = a.rows;
    const KfCuts cuts = {work / ctas, (int)(work % ctas), ctas};
    const int64_t begin = cuts.at(cta);
    if (cta < ctas && work > 0) {
      for (int r0 = 0; r0 < a.rows; r0 += 32) {
        int64_t mine = 0;
        if (r0 + lane < a.rows) {
          const KfBlock b = kf_block(a, r0 + lane, span);
          mine = kf_length(b, span, b.tiles) * hkv;
        }
        int64_t incl = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int64_t u = __shfl_up_sync(0xffffffffu, incl, o);
          if (lane >= o) incl += u;
        }
        const unsigned has = __ballot_sync(0xffffffffu, at + incl > begin);
        if (has) {
          const int l = __ffs(has) - 1;
          row = r0 + l;
          at += __shfl_sync(0xffffffffu, incl - mine, l);
          break;
        }
        at += __shfl_sync(0xffffffffu, incl, 31);
      }
    }
    int t = 0, head = 0;
    if (row < a.rows) {
      const KfBlock b = kf_block(a, row, span);
      const int64_t x = begin - at;
      int lo = 0, hi = b.tiles - 1;
      while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (kf_length(b, span, mid) * hkv <= x) lo = mid; else hi = mid - 1;
      }
      t = lo;
      const int64_t from = kf_length(b, span, t);
      head = (int)((x - from * hkv) / (kf_length(b, span, t + 1) - from));
    }
    __syncwarp();
    if (lane == 0) {
      sh.cursor_row = row, sh.cursor_tile = t, sh.cursor_head = head;
      sh.cursor_at = at, sh.cuts = cuts;
    }
    __syncwarp();
  }
  const KfCuts cuts = sh.cuts;
  int row = sh.cursor_row, t = sh.cursor_tile, head = sh.cursor_head, n = 0;
  int64_t at = sh.cursor_at;
  bool more = false;
  if (row < a.rows) {
    const int64_t begin = cuts.at(cta), end = cuts.at(cta + 1);
    KfBlock b = kf_block(a, row, span);
    int len = max(a.row_len[row], 0);
    while (true) {
      const int64_t before = kf_length(b, span, t), length = kf_length(b, span, t + 1) - before;
      const int64_t from = at + before * hkv + head * length;
      if (t < b.tiles && from >= end) break;
      if (t < b.tiles) {
        if (n == KF_PIECES) {
          more = true;
          break;
        }
        const int first = t * span, last = min(b.count, first + span) - 1;
        const int keys = min(len - b.count + last + 1, a.cap);  // keys that some row sees
        const int steps = keys > 0 ? (keys + KF_KEYS - 1) / KF_KEYS : 0;
        auto step_at = [&](int64_t cut) {
          const int64_t x = cut - from - KF_TILE_COST;
          const int j = (int)min((int64_t)steps, x > 0 ? x / KF_KEYS : 0);
          return j < KF_LEAST ? 0 : j > steps - KF_LEAST ? steps : j;
        };
        // (a cut short of a tile of less than KF_LEAST steps leaves it whole to the later share)
        const int j0 = from >= begin ? 0 : step_at(begin), j1 = from + length <= end ? steps : step_at(end);
        if (j1 > j0 || (steps == 0 && from >= begin)) {
          if (lane == 0) {
            KfPiece& p = sh.piece[n];
            p.seq = a.row_seq ? a.row_seq[row] : row;
            p.q0 = b.q0, p.first = first, p.last = last, p.before = len - b.count;
            p.head = head, p.keys = keys, p.steps = steps, p.j0 = j0, p.j1 = j1;
            p.low = p.parts = 0;
            if (j1 - j0 < steps) {  // the cuts inside the tile are low .. high
              p.low = cuts.first(from + KF_TILE_COST + KF_LEAST * KF_KEYS);
              const int64_t past = from + KF_TILE_COST + (steps - KF_LEAST + 1) * (int64_t)KF_KEYS;
              p.parts = cuts.first(min(past, from + length)) - p.low + 1;
            }
          }
          ++n;
        }
        if (++head < hkv) continue;
        head = 0;
        if (++t < b.tiles) continue;
      }
      // the next block
      at += kf_length(b, span, b.tiles) * hkv;
      t = 0;
      if (++row >= a.rows) break;
      b = kf_block(a, row, span);
      len = max(a.row_len[row], 0);
    }
  }
  __syncwarp();
  if (lane == 0) {
    sh.pieces = n, sh.more = more;
    sh.cursor_row = row, sh.cursor_tile = t, sh.cursor_head = head, sh.cursor_at = at;
  }
}

// 8 dimensions, in the order in which words of codes unpack
__device__ __forceinline__ void kf_store(__nv_bfloat16* out, const uint32_t* v, float f) {
  float d[8];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    d[k] = __uint_as_float(v[2 * k]) * f;
    d[k + 4] = __uint_as_float(v[2 * k + 1]) * f;
  }
  uint4 u;
  uint32_t* p = reinterpret_cast<uint32_t*>(&u);
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const __nv_bfloat162 b = __floats2bfloat162_rn(d[2 * k], d[2 * k + 1]);
    p[k] = *reinterpret_cast<const uint32_t*>(&b);
  }
  *reinterpret_cast<uint4*>(out) = u;
}
// a part in the workspace: outputs [D / 8][thread] in fours, then (maximum, sum) [thread]
__host__ __device__ constexpr int kf_slot(int d) { return KF_SOFTMAX * (d / 2 + 2); }

// Joins a divided tile's parts, each thread its half row: part p lies in CTA low - 1 + p, the first at
// its share's end, the others at their beginnings.
template <int D>
__device__ __noinline__ void kf_join(const float* part, int low, int parts, int thread, __nv_bfloat16* out) {
  const auto slot = [&](int p) { return part + (int64_t)(2 * (low - 1 + p) + (p == 0)) * kf_slot(D); };
  const auto of = [&](int p) {
    return __ldcg(reinterpret_cast<const float2*>(slot(p) + KF_SOFTMAX * (D / 2)) + thread);
  };
  float top = -INFINITY, sum = 0.f;
#pragma unroll 4
  for (int p = 0; p < parts; ++p) top = fmaxf(top, of(p).x);
  // a part without a key has sums of nothing, or NaN
  const auto factor = [&](float x) { return x == -INFINITY ? 1.f : kf_exp2(x - top); };
#pragma unroll 1
  for (int c = 0; c < D / 16; c += 4) {
    float o[32] = {};
    sum = 0.f;
#pragma unroll 1
    for (int p = 0; p < parts; ++p) {
      const float4* const from = reinterpret_cast<const float4*>(slot(p)) + 2 * c * KF_SOFTMAX + thread;
      const float2 x = of(p);
      float4 y[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = __ldcg(from + e * KF_SOFTMAX);
      const float g = factor(x.x);
      sum = fmaf(x.y, g, sum);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        o[4 * e] = fmaf(y[e].x, g, o[4 * e]), o[4 * e + 1] = fmaf(y[e].y, g, o[4 * e + 1]);
        o[4 * e + 2] = fmaf(y[e].z, g, o[4 * e + 2]), o[4 * e + 3] = fmaf(y[e].w, g, o[4 * e + 3]);
      }
    }
    const float f = sum == 0.f ? 0.f : 0x1p10f / sum;
    uint32_t v[32];
#pragma unroll
    for (int e = 0; e < 32; ++e) v[e] = sum == 0.f ? 0u : __float_as_uint(o[e]);
#pragma unroll
    for (int e = 0; e < 4; ++e) kf_store(out + (c + e) * 8, v + 8 * e, f);
  }
}

// A piece's queries to shared memory, a row's 16-byte columns to as many lanes: a warp reads whole rows,
// all its rows at once.
template <int D>
__device__ __noinline__ void kf_place_queries(const Kv4PrefillArgs& a, KfShared& sh, unsigned char* sq, int n) {
  constexpr int COLS = D / 8, EACH = 16 * COLS / 32, TILE_BYTES = D / 64 * 16384;
  const KfPiece& piece = sh.piece[n];
  const int group = a.hq / a.pool.hkv, span = KF_ROWS / group;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, i = warp >> 3, col = lane % COLS;
  uint4 x[EACH];
#pragma unroll
  for (int k = 0; k < EACH; ++k) {
    const int row = warp * 16 + k * (32 / COLS) + lane / COLS, t = kf_divide(row, group, a.group_magic);
    const int token = piece.first + t;
    const bool there = t < span && token <= piece.last;
    const int64_t from = ((int64_t)(piece.q0 + token) * a.hq + piece.head * group + (row - t * group)) * COLS + col;
    x[k] = there ? __ldg(reinterpret_cast<const uint4*>(a.q) + from) : make_uint4(0, 0, 0, 0);
  }
#pragma unroll
  for (int k = 0; k < EACH; ++k) {
    const int r = (warp & 7) * 16 + k * (32 / COLS) + lane / COLS;
    const uint32_t u[4] = {x[k].x & a.q_and, x[k].y & a.q_and, x[k].z & a.q_and, x[k].w & a.q_and};
    float most = 0.f, f[8];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      f[2 * e] = __uint_as_float((u[e] ^ a.q_xor) << 16), f[2 * e + 1] = __uint_as_float((u[e] ^ a.q_xor) & 0xffff0000u);
      most = fmaxf(most, fmaxf(fabsf(f[2 * e]), fabsf(f[2 * e + 1])));
    }
#pragma unroll
    for (int o = 1; o < COLS; o <<= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
    // 2^up brings the largest query to [2^13, 2^14); bounded so that 2^up and 2^-up are numbers
    const int up = max(-110, min(110, 140 - (int)(__float_as_uint(most) >> 23)));
    const float mul = kf_pow2(up);
    if (col == 0) sh.query_scale[i][r] = kf_pow2(-up);
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] *= mul;
    // dimensions in the order 0 4 1 5 2 6 3 7, as words of codes unpack
    *reinterpret_cast<uint4*>(sq + i * TILE_BYTES + r * 128 + (col >> 3) * 16384 + (((col & 7) ^ (r & 7)) << 4)) =
        make_uint4(kf_half2(f[0], f[4]), kf_half2(f[1], f[5]), kf_half2(f[2], f[6]), kf_half2(f[3], f[7]));
  }
  fence_proxy_async_smem();
  mbar_arrive(&sh.q_full);
}

// Outputs of queries of no block, by the filling warps when their last tile is filled. (In the issuing
// warpgroup, whose idle warps could write them at once, it cost the products' loop registers: nine ragged
// blocks 343 us, and 337 so.)
__device__ __noinline__ void kf_zero_rest(const Kv4PrefillArgs& a, int rest, int row) {
  uint4* const out = reinterpret_cast<uint4*>(a.out);
  const int64_t end = a.tokens * row, step = gridDim.x * KF_FILL;
  for (int64_t x = (int64_t)rest * row + blockIdx.x * KF_FILL + threadIdx.x - KF_SOFTMAX; x < end; x += step)
    out[x] = make_uint4(0u, 0u, 0u, 0u);
}

template <int D, int G>
__global__ void __launch_bounds__(KF_THREADS, 1) kv4_prefill_kernel(const __grid_constant__ Kv4PrefillArgs a) {
  constexpr int NG = D / G, HALVES = D / 64, TILE_BYTES = HALVES * 16384;
  constexpr int BLOCK = kv4_block_bytes(D, G), CODES = kv4_codes_bytes(D), PARAMS = kv4_params_bytes(D, G);
  extern __shared__ unsigned char raw[];
  __shared__ KfShared sh;
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  unsigned char* sq = smem;                   // two row tiles of queries
  unsigned char* sk = sq + 2 * TILE_BYTES;    // two stages of K
  unsigned char* sv = sk + 2 * TILE_BYTES;    // two stages of V
  const int tid = threadIdx.x, lane = tid & 31;
  const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  const int group = a.hq / a.pool.hkv, span = KF_ROWS / group;  // tokens a tile
  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sh.s_full[i], 1);
      mbar_init(&sh.w_full[i], KF_SOFTMAX / 2);
      mbar_init(&sh.o_full[i], 1);
      mbar_init(&sh.o_done[i], 1);
      mbar_init(&sh.k_full[i], KF_FILL);
      mbar_init(&sh.k_empty[i], 1);
      mbar_init(&sh.v_full[i], KF_FILL);
      mbar_init(&sh.v_empty[i], 1);
    }
    for (int i = 0; i < KF_META; ++i) mbar_init(&sh.meta_full[i], KF_FILL);
    mbar_init(&sh.q_full, KF_SOFTMAX);
    sh.dead = 0;
    sh.cursor_row = -1;
    for (int i = 0; i < 16; ++i) (&sh.seek[0][0][0])[i] = 0;
    fence_proxy_async_smem();
  }
  pdl_launch_dependents();
  pdl_wait();
  if (warp == (KF_SOFTMAX + KF_FILL) / 32) tmem_alloc(&sh.tmem, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sh.tmem;  // columns: S 0, S 1 (W over them), O 0, O 1, 128 each

  if (warp < KF_SOFTMAX / 32) {
    // ------------------------------------------------------------ queries, softmax, output
    // two threads a row, half of the keys (and of the dimensions) each, in warps that lie four apart
    kf_more_registers<KF_SOFTMAX_REGS>();
    const int i = warp >> 3, half = (warp >> 2) & 1, r = tid & 127, rho = i * 128 + r;
    const int pair = 2 + i * 4 + (warp & 3);  // the two warps' named barrier
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t ts = tmem + lanes + i * 128 + half * (KF_KEYS / 2);      // this thread's scores
    const uint32_t tw = tmem + lanes + i * 128 + half * (KF_KEYS / 4);      // its weights, over the row's scores
    const uint32_t to = tmem + lanes + 256 + i * 128 + half * (D / 2);      // its outputs
    int walked = 0, turns = 0;  // steps and pieces of this CTA so far, which the barriers' phases go by
    bool more;
    do {
      if (warp == 0) kf_plan(a, sh, span, lane);
      kf_all_sync();
      if (sh.pieces > 0 && sh.piece[0].j1 > sh.piece[0].j0) kf_place_queries<D>(a, sh, sq, 0);
#pragma unroll 1
      for (int n = 0; n < sh.pieces; ++n) {
        const KfPiece& piece = sh.piece[n];
        const int j0 = piece.j0, j1 = piece.j1;
        const int token = piece.first + rho / group;
        const bool live = rho < span * group && token <= piece.last;
        const int pos = live ? piece.before + token : INT32_MAX;  // a dead row masks nothing
        float mrow = 0.f;
        if (j1 > j0) {
          asm volatile("bar.sync %0, 256;" ::"r"(11 + i) : "memory");
          mrow = a.scale2 * sh.query_scale[i][r] * 0x1p10f;
        }
        int nearest = pos;  // the fewest keys a row of this warp sees, less one
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) nearest = min(nearest, __shfl_xor_sync(0xffffffffu, nearest, o));
        float M = -INFINITY, den = 0.f;
#pragma unroll 1
        for (int j = j0; j < j1; ++j) {
          const int at_step = walked + j - j0, m = at_step % KF_META;
          kf_wait(&sh.meta_full[m], (at_step / KF_META) & 1, sh);
          float mult = mrow * sh.k_scale[m], power = sh.v_power[m];
          const int limit = pos - j * KF_KEYS;  // the last key of the tile that this row sees
          kf_wait(&sh.s_full[i], at_step & 1, sh);
          __syncwarp();
          tc_fence_after();
          if (!sh.uniform[m] || j * KF_KEYS + KF_KEYS - 1 > nearest) {
            // masks and the tokens' own powers go into the scores first
            const float* const powers = &sh.power[m][half * (KF_KEYS / 2)];
            const int mine = limit - half * (KF_KEYS / 2);  // the last that it sees of this half
#pragma unroll 1
            for (int c = 0; c < KF_KEYS / 2; c += 32) {
              uint32_t v[2][16];
              tmem_ld_16cols_async(ts + c, v[0]);
              tmem_ld_16cols_async(ts + c + 16, v[1]);
#pragma unroll
              for (int b = 0; b < 2; ++b) {
                tmem_wait_ld(v[b]);
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                  const int key = c + b * 16 + e;
                  v[b][e] = __float_as_uint(key <= mine ? fmaf(__uint_as_float(v[b][e]), mult, powers[key]) : -INFINITY);
                }
                tmem_st_16cols(ts + c + b * 16, v[b]);
              }
            }
            tmem_wait_st();
            mult = 1.f;
            power = 0.f;
          }
          uint32_t w[KF_KEYS / 4];
          float plain;  // the sum of the row's weights of this half
          // again after the maximum has moved (a few turns where scores are past 2^27); a piece's first step
          // begins with its maximum
#pragma unroll 1
          for (int turn = j == j0 ? -1 : 0;; ++turn) {
            const float ref = M == -INFINITY ? 0.f : M;
            uint32_t buf[2][8];
            if (turn >= 0) {
              tmem_ld_8cols_async(ts, buf[0]);
              const uint64_t bias2 = kf_pair(power - ref, power - ref), mult2 = kf_pair(mult, mult);
              uint64_t sums[2] = {kf_pair(0.f, 0.f), kf_pair(0.f, 0.f)};
#pragma unroll
              for (int c = 0; c < 8; ++c) {
                tmem_wait_ld(buf[c & 1]);
                if (c < 7) tmem_ld_8cols_async(ts + (c + 1) * 8, buf[(c + 1) & 1]);
                uint32_t(&s)[8] = buf[c & 1];
#pragma unroll
                for (int e = 0; e < 8; e += 2) {
                  const float2 x = kf_split(
                      kf_fma_pair(kf_pair(__uint_as_float(s[e]), __uint_as_float(s[e + 1])), mult2, bias2));
                  const float p = kf_exp2(x.x), q = kf_exp2(x.y);
                  sums[(e >> 1) & 1] = kf_add_pair(sums[(e >> 1) & 1], kf_pair(p, q));
                  w[c * 4 + e / 2] = kf_half2(p, q);
                }
              }
              const float2 both = kf_split(kf_add_pair(sums[0], sums[1]));
              plain = both.x + both.y;
              // Weights that sum to 2^13 at most are all inside fp16, whatever M; a row without one yet has no
              // M. Both warps of a pair go by the same flag, and the barrier also keeps one's weights off the
              // other's scores.
              const bool seek = plain > 8192.f || (turn == 0 && M == -INFINITY && limit >= 0);
              int* const flag = &sh.seek[i][warp & 3][turn & 1];
              if (__any_sync(0xffffffffu, seek) && lane == 0) *flag = 1;
              kf_pair_sync(pair);
              const int moves = *(volatile int*)flag;
              if (turn == 7 || !moves) break;
            }
            float top = -INFINITY;
#pragma unroll 1
            for (int c = 0; c < KF_KEYS / 2; c += 32) {
              uint32_t v[2][16];
              tmem_ld_16cols_async(ts + c, v[0]);
              tmem_ld_16cols_async(ts + c + 16, v[1]);
#pragma unroll
              for (int b = 0; b < 2; ++b) {
                tmem_wait_ld(v[b]);
#pragma unroll
                for (int e = 0; e < 16; ++e) top = fmaxf(top, fmaf(__uint_as_float(v[b][e]), mult, power - ref));
              }
            }
            sh.top[i][half][r] = top;
            kf_pair_sync(pair);
            // read by both before this barrier, next set after another
            if (lane == 0 && half == 0) sh.seek[i][warp & 3][turn & 1] = 0;
            top = fmaxf(top, sh.top[i][half ^ 1][r]);
            float f = 1.f;
            if (M == -INFINITY) {
              M = top;  // no key so far: only zeros, or a NaN that stays
            } else if (top > 0.f) {
              f = kf_exp2(-top);
              M += top;
            }
            den *= f;
            if (j > j0 && __any_sync(0xffffffffu, f != 1.f)) {
#pragma unroll 1
              for (int c = 0; c < D / 16; ++c) {
                tmem_ld_8cols_async(to + c * 8, buf[0]);
                tmem_wait_ld(buf[0]);
#pragma unroll
                for (int e = 0; e < 8; ++e) buf[0][e] = __float_as_uint(__uint_as_float(buf[0][e]) * f);
                tmem_st_8cols(to + c * 8, buf[0]);
              }
              tmem_wait_st();
            }
          }
          if (sh.uniform[m]) {
            den = fmaf(plain, sh.v_undo[m], den);
          } else {  // each weight with its token's power taken back; a token that is not there has none
            const float* const powers = &sh.power[m][half * (KF_KEYS / 2)];
            const float ref = M == -INFINITY ? 0.f : M;
#pragma unroll 1
            for (int c = 0; c < KF_KEYS / 2; c += 8) {
              uint32_t v[8];
              tmem_ld_8cols_async(ts + c, v);
              tmem_wait_ld(v);
#pragma unroll
              for (int e = 0; e < 8; ++e)
                den = fmaf(kf_exp2(__uint_as_float(v[e]) - ref), kf_exp2(fminf(-powers[c + e], 126.f)), den);
            }
            kf_pair_sync(pair);  // neither's weights go over the other's scores before these reads
          }
          tmem_st_32cols(tw, w);
          tmem_wait_st();
          tc_fence_before();
          mbar_arrive(&sh.w_full[i]);
        }
        walked += j1 - j0;
        if (j1 > j0) {
          sh.top[i][half][r] = den;
          kf_pair_sync(pair);
          den += sh.top[i][half ^ 1][r];
          kf_wait(&sh.o_full[i], turns & 1, sh);
          ++turns;
          __syncwarp();
          tc_fence_after();
        }
        // the next piece's queries, which no product holds up now, go in before this piece's outputs go out
        if (n + 1 < sh.pieces && sh.piece[n + 1].j1 > sh.piece[n + 1].j0) kf_place_queries<D>(a, sh, sq, n + 1);
        __nv_bfloat16* const out =
            a.out + ((int64_t)(piece.q0 + token) * a.hq + (int64_t)piece.head * group + rho % group) * D + half * (D / 2);
        if (j1 - j0 == piece.steps) {
          const float f = den == 0.f ? 0.f : 0x1p10f / den;
#pragma unroll
          for (int c = 0; c < D / 32; ++c) {
            uint32_t v[16] = {};
            if (j1 > j0) {
              tmem_ld_16cols_async(to + c * 16, v);
              tmem_wait_ld(v);
            }
            if (den == 0.f)
#pragma unroll
              for (int e = 0; e < 16; ++e) v[e] = 0u;
            if (live) {
              kf_store(out + c * 16, v, f);
              kf_store(out + c * 16 + 8, v + 8, f);
            }
          }
        } else {
          // ---- a part: sums, maximum and outputs to the workspace; the last of the tile's parts joins them
          const int low = piece.low, parts = piece.parts;
          float* const mine = a.part + (int64_t)(2 * blockIdx.x + (j0 == 0)) * kf_slot(D);
#pragma unroll
          for (int c = 0; c < D / 32; ++c) {
            uint32_t v[16];
            tmem_ld_16cols_async(to + c * 16, v);
            tmem_wait_ld(v);
            if (live)
#pragma unroll
              for (int e = 0; e < 16; e += 4)
                __stcg(reinterpret_cast<uint4*>(mine) + (c * 4 + e / 4) * KF_SOFTMAX + tid,
                       make_uint4(v[e], v[e + 1], v[e + 2], v[e + 3]));
          }
          __stcg(reinterpret_cast<float2*>(mine + KF_SOFTMAX * (D / 2)) + tid, make_float2(M, den));
          __threadfence();
          asm volatile("bar.sync 10, 512;" ::: "memory");
          if (tid == 0) {
            unsigned* const counter = a.counters + low;
            const int turn = (int)atomicAdd(counter, 1u);
            sh.joins = turn == parts - 1;
            if (turn == parts - 1) *counter = 0u;  // for the next call
            __threadfence();
          }
          asm volatile("bar.sync 10, 512;" ::: "memory");
          if (sh.joins && live) kf_join<D>(a.part, low, parts, tid, out);
        }
        tc_fence_before();
      }
      more = sh.more;
      kf_all_sync();
    } while (more);
  } else if (warp < (KF_SOFTMAX + KF_FILL) / 32) {
    // ------------------------------------------------------------ codes to fp16 tiles
    kf_fewer_registers<KF_FILL_REGS>();
    // four lanes a token, a quarter of its dimensions each; KF_PASSES passes
    // Each thread copies the codes and parameters of its next tile into its own places of shared
    // memory while it works on this one, and reads the page numbers of the one after.
    constexpr int KW = D / 32, SPAN = KF_KEYS / KF_PASSES;  // words of codes a lane and pass, tokens a pass
    const int ft = tid - KF_SOFTMAX, fw = warp - KF_SOFTMAX / 32, part = lane & 3, gp = part * (D / 4) / G;
    const int tok0 = fw * 8 + (lane >> 2);
    unsigned char* ahead = sv + 2 * TILE_BYTES + ft * (KW * 4);   // codes [2 KF_PASSES][threads]: K's passes, then V's
    unsigned char* ahead_p = sv + 2 * TILE_BYTES + 2 * KF_PASSES * KF_FILL * (KW * 4) + ft * 4;  // parameters, alike
    uint32_t kw[KF_PASSES][KW], vw[KF_PASSES][KW], kp[KF_PASSES], vp[KF_PASSES];
    // a warp's eight tokens of a pass lie in one 16-token block
    const int rw = tok0 % KV4_TILE, page_tiles = a.pool.page_size / KV4_TILE;
    const int code_at = rw * (D / 2) + part * (D / 8), param_at = 2 * CODES + (rw * NG + gp) * 4;
    const unsigned char* mine;
    const int32_t* pages;
    int keys, steps;
    bool mapped;
    // Lanes of a quarter warp write eight different 16-byte columns: the upper dimensions' lanes take
    // their words in another order.
    const int swap = KW == 4 && part >= 2 ? 8 : 0;
    int place[KW];
#pragma unroll
    for (int c = 0; c < KW; ++c) {
      const int chunk = KW == 4 ? (part & 1) * 4 + (c ^ (swap >> 2)) : part * 2 + c;
      place[c] = (KW == 4 ? (part >> 1) * 16384 : 0) + tok0 * 128 + ((chunk ^ (tok0 & 7)) << 4);
    }
    int page[KF_PASSES];
    auto load_pages = [&](int j) {
#pragma unroll
      for (int p = 0; p < KF_PASSES; ++p) {
        const int tile = j * (KF_KEYS / KV4_TILE) + p * (SPAN / KV4_TILE) + (fw >> 1);
        page[p] = mapped && tile * KV4_TILE < keys ? pages[kf_divide(tile, page_tiles, a.page_magic)] : -1;
      }
    };
    auto copy = [&](int j) -> unsigned {  // returns the passes whose token is there
      unsigned have = 0;
#pragma unroll
      for (int p = 0; p < KF_PASSES; ++p) {
        const int tile = j * (KF_KEYS / KV4_TILE) + p * (SPAN / KV4_TILE) + (fw >> 1);
        const int in = tile - kf_divide(tile, page_tiles, a.page_magic) * page_tiles;
        if (page[p] >= 0 && page[p] < a.pool.num_pages) {
          if (j * KF_KEYS + p * SPAN + tok0 < keys) have |= 1u << p;
          const unsigned char* b = mine + page[p] * a.pool.stride_page + in * BLOCK;
#pragma unroll
          for (int v = 0; v < 2; ++v) {
            kf_copy<KW * 4>(ahead + (v * KF_PASSES + p) * KF_FILL * (KW * 4), b + v * CODES + code_at);
            kf_copy<4>(ahead_p + (v * KF_PASSES + p) * KF_FILL * 4, b + v * PARAMS + param_at);
          }
        } else if (tile * KV4_TILE < keys && a.error_flag && lane == 0) {
          atomicOr(a.error_flag, MRB_KV_UNMAPPED);
        }
      }
      cp_async_commit_group();
      return have;
    };
    auto take = [&](unsigned have) {
#pragma unroll
      for (int p = 0; p < KF_PASSES; ++p) {
        const bool ok = have >> p & 1;
#pragma unroll
        for (int v = 0; v < 2; ++v) {
          uint32_t(&w)[KW] = v ? vw[p] : kw[p];
          const unsigned char* src = ahead + (v * KF_PASSES + p) * KF_FILL * (KW * 4);
          if constexpr (KW == 4) {  // swapped lanes: words 2 3 0 1
            const uint2 x = *reinterpret_cast<const uint2*>(src + swap), y = *reinterpret_cast<const uint2*>(src + (swap ^ 8));
            w[0] = x.x, w[1] = x.y, w[2] = y.x, w[3] = y.y;
          } else {
            const uint2 x = *reinterpret_cast<const uint2*>(src);
            w[0] = x.x, w[1] = x.y;
          }
          uint32_t& prm = v ? vp[p] : kp[p];
          prm = *reinterpret_cast<const uint32_t*>(ahead_p + (v * KF_PASSES + p) * KF_FILL * 4);
          prm = ok ? prm : 0u;  // codes times nothing
        }
      }
    };
    // fp16 values of one pass, scaled by 2^-(e + 10): up14 is 2^(14 - e), down10 2^(-10 - e)
    auto fill = [&](unsigned char* tile, int p, const uint32_t (&w)[KW], uint32_t prm, float up14, float down10) {
      const float s14 = __uint_as_float(prm << 16) * up14, m10 = __uint_as_float(prm & 0xffff0000u) * down10;
      const uint32_t even = kf_half2(s14, s14), odd = kf_half2(s14 * 0.0625f, s14 * 0.0625f), add = kf_half2(m10, m10);
#pragma unroll
      for (int c = 0; c < KW; ++c) {
        const uint32_t x = w[c], y = x >> 8;
        *reinterpret_cast<uint4*>(tile + p * SPAN * 128 + place[c]) =
            make_uint4(kf_fma2(x & 0x000f000fu, even, add), kf_fma2(x & 0x00f000f0u, odd, add),
                       kf_fma2(y & 0x000f000fu, even, add), kf_fma2(y & 0x00f000f0u, odd, add));
      }
    };
    // of a tile whose tokens are far apart: codes as whole numbers, so that the scales leave room, and the
    // values scaled by up = 2^(11 - e), to 2^15 at most
    auto fill_far = [&](unsigned char* tile, int p, const uint32_t (&w)[KW], uint32_t prm, float up) {
      const float s = __uint_as_float(prm << 16) * up, m = __uint_as_float(prm & 0xffff0000u) * up;
      const uint32_t mul = kf_half2(s, s), add = kf_half2(m, m);
      const auto number = [](uint32_t x) {  // two codes: 1024 + c, less 1024
        return kf_fma2((x & 0x000f000fu) | 0x64006400u, 0x3c003c00u, 0xe400e400u);
      };
#pragma unroll
      for (int c = 0; c < KW; ++c) {
        const uint32_t x = w[c];
        *reinterpret_cast<uint4*>(tile + p * SPAN * 128 + place[c]) =
            make_uint4(kf_fma2(number(x), mul, add), kf_fma2(number(x >> 4), mul, add),
                       kf_fma2(number(x >> 8), mul, add), kf_fma2(number(x >> 12), mul, add));
      }
    };
    auto power_of = [](float most) { return max(-60, (int)(__float_as_uint(most) >> 23) - 127 - 3); };
    int walked = 0;
    bool more;
    do {
      kf_all_sync();
      const int pieces = sh.pieces;
      more = sh.more;
#pragma unroll 1
      for (int n = 0; n < pieces; ++n) {
        const KfPiece& piece = sh.piece[n];
        const int j0 = piece.j0, j1 = piece.j1;
        mine = a.pool.base + (int64_t)piece.head * a.pool.stride_head;
        pages = a.block_table + piece.seq * a.bt_stride;
        mapped = piece.seq >= 0 && piece.seq < a.num_seqs;
        keys = piece.keys, steps = piece.steps;
        unsigned next = 0;
        if (j1 > j0) {
          load_pages(j0);
          next = copy(j0);
          load_pages(j0 + 1);
        }
#pragma unroll 1
        for (int j = j0; j < j1; ++j, ++walked) {
          const int st = walked & 1, m = walked % KF_META;
          const unsigned have = next;
          cp_async_wait_group<0>();
          take(have);
          if (j + 1 < j1) {
            next = copy(j + 1);
            load_pages(j + 2);
          }
          // ---- the tile's sizes, and the smallest token's of K; where V's are far apart or no numbers, each
          // token's
          float kmost = 0.f, kleast = INFINITY, vmost = 0.f, vleast = INFINITY, size[KF_PASSES];
          bool plain = have == (1u << KF_PASSES) - 1u;
#pragma unroll
          for (int p = 0; p < KF_PASSES; ++p) {
            const float ks = __uint_as_float(kp[p] << 16), km = __uint_as_float(kp[p] & 0xffff0000u);
            float kx = fmaxf(fabsf(km), fabsf(fmaf(15.f, ks, km)));
            kx = kx < 3e38f ? kx : 0.f;  // a NaN stays one, whatever the scale
            if (NG > 1) kx = fmaxf(kx, __shfl_xor_sync(0xffffffffu, kx, 2));  // of the token's other groups
            if (NG > 2) kx = fmaxf(kx, __shfl_xor_sync(0xffffffffu, kx, 1));
            kmost = fmaxf(kmost, kx);
            kleast = fminf(kleast, kx > 0.f ? kx : kleast);
            const float vs = __uint_as_float(vp[p] << 16), vm = __uint_as_float(vp[p] & 0xffff0000u);
            size[p] = kf_max_nan(fabsf(vm), fabsf(fmaf(15.f, vs, vm)));
            const float vx = size[p] < 3e38f ? size[p] : 0.f;
            plain = plain && size[p] < 3e38f;
            vmost = fmaxf(vmost, vx);
            vleast = fminf(vleast, vx > 0.f ? vx : vleast);
          }
          // of numbers that are not negative, as their bits
          kmost = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(kmost)));
          kleast = __uint_as_float(__reduce_min_sync(0xffffffffu, __float_as_uint(kleast)));
          vmost = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(vmost)));
          vleast = __uint_as_float(__reduce_min_sync(0xffffffffu, __float_as_uint(plain ? vleast : 0.f)));
          if (lane == 0) *reinterpret_cast<float4*>(sh.red[st][fw]) = make_float4(kmost, vmost, vleast, kleast);
          asm volatile("bar.sync 1, 256;" ::: "memory");
          const float4 other = *reinterpret_cast<const float4*>(sh.red[st][lane % (KF_FILL / 32)]);
          kmost = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(other.x)));
          vmost = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(other.y)));
          vleast = __uint_as_float(__reduce_min_sync(0xffffffffu, __float_as_uint(other.z)));
          kleast = __uint_as_float(__reduce_min_sync(0xffffffffu, __float_as_uint(other.w)));
          const int ke = power_of(kmost), ve = power_of(vmost);
          const bool uniform = vleast > 0.f && vleast >= vmost * 0x1p-6f;  // (0: not every token is there)
          const bool far = kleast < kmost * 0x1p-6f;  // keys beside which others would lose bits
          const float k14 = kf_pow2((far ? 11 : 14) - ke), k10 = kf_pow2(-10 - ke), ve14 = kf_pow2(14 - ve), ve10 = kf_pow2(-10 - ve);
          float v14[KF_PASSES], v10[KF_PASSES];
#pragma unroll
          for (int p = 0; p < KF_PASSES; ++p) v14[p] = ve14, v10[p] = ve10;
          if (!uniform) {
#pragma unroll
            for (int p = 0; p < KF_PASSES; ++p) {
              float x = size[p] < 3e38f ? size[p] : 0.f;
              const bool nan = __ballot_sync(0xffffffffu, !(size[p] < 3e38f)) >> (lane & 28) & 15u;
              x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
              x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
              const int te = power_of(x);
              v14[p] = kf_pow2(14 - te);
              v10[p] = kf_pow2(-10 - te);
              if (nan) {  // the weight carries it, so that rows that do not see the token stay clean
                vp[p] = 0u;
#pragma unroll
                for (int e = 0; e < KW; ++e) vw[p][e] = 0u;
              }
              if (part == 0) {
                const int tok = p * SPAN + tok0;
                sh.power[m][tok] = !(have >> p & 1) ? -INFINITY : nan ? __int_as_float(0x7fffffff) : (float)te;
              }
            }
          } else if (j >= steps - 4) {  // rows that see part of the tile (of 256 tokens at most) go by its tokens
            if (part == 0)
#pragma unroll
              for (int p = 0; p < KF_PASSES; ++p) sh.power[m][p * SPAN + tok0] = (float)ve;
          }
          if (ft == 0) {
            sh.k_scale[m] = kf_pow2(far ? ke - 21 : ke);
            sh.v_power[m] = (float)ve;
            sh.v_undo[m] = kf_pow2(-ve);
            sh.uniform[m] = uniform;
          }
          mbar_arrive(&sh.meta_full[m]);
          // ---- K, then V
          if (walked >= 2) kf_wait(&sh.k_empty[st], ((walked >> 1) - 1) & 1, sh);
          __syncwarp();
#pragma unroll
          for (int p = 0; p < KF_PASSES; ++p) {
            if (far) fill_far(sk + st * TILE_BYTES, p, kw[p], kp[p], k14);
            else fill(sk + st * TILE_BYTES, p, kw[p], kp[p], k14, k10);
          }
          fence_proxy_async_smem();
          mbar_arrive(&sh.k_full[st]);
          if (walked >= 2) kf_wait(&sh.v_empty[st], ((walked >> 1) - 1) & 1, sh);
          __syncwarp();
#pragma unroll
          for (int p = 0; p < KF_PASSES; ++p) fill(sv + st * TILE_BYTES, p, vw[p], vp[p], v14[p], v10[p]);
          fence_proxy_async_smem();
          mbar_arrive(&sh.v_full[st]);
        }
      }
      if (a.zero_rest && !more && sh.rest < a.tokens) kf_zero_rest(a, sh.rest, a.hq * (D / 8));
      kf_all_sync();
    } while (more);
  } else {
    // ------------------------------------------------------------ the products
    kf_fewer_registers<KF_ISSUE_REGS>();
    // The whole warp walks the steps with values that are the same for all lanes, and one elected lane
    // issues: products issued from a branch on the lane's number took 160 clocks each, whatever their
    // size, these 66 (128 x 128 x 16, of 64 at the tensor peak).
    constexpr uint32_t IDESC_S = umma_idesc(UMMA_D_F32, 0, 0, 128, KF_KEYS);  // fp16 x fp16
    constexpr uint32_t IDESC_O = umma_idesc(UMMA_D_F32, 0, 0, 128, D) | 1u << 16;  // V: dimensions contiguous
    // descriptors hold addresses in steps of 16 bytes, so operands move by additions
    const uint64_t dq = umma_desc_k_sw128(smem_u32(sq)), dk = umma_desc_k_sw128(smem_u32(sk)), dv = kf_desc_v(smem_u32(sv));
    const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
    auto scores = [&](int i, int at) {
      const uint64_t x = dq + i * (TILE_BYTES >> 4), y = dk + (at & 1) * (TILE_BYTES >> 4);
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) {
        const uint32_t off = ((ks >> 2) * 16384 + (ks & 3) * 32) >> 4;
        umma_f16(tm + i * 128, x + off, y + off, IDESC_S, ks > 0);
      }
      umma_commit(&sh.s_full[i]);
      if (i == 1) umma_commit(&sh.k_empty[at & 1]);
    };
    int walked = 0, turns = 0;
    bool more;
    do {
      kf_all_sync();
      more = sh.more;
      const int pieces = warp == (KF_SOFTMAX + KF_FILL) / 32 ? sh.pieces : 0;
#pragma unroll 1
      for (int n = 0; n < pieces; ++n) {
        const int steps = sh.piece[n].j1 - sh.piece[n].j0;
        if (steps == 0) continue;
        kf_wait(&sh.q_full, turns & 1, sh);
        ++turns;
        kf_wait(&sh.k_full[walked & 1], (walked >> 1) & 1, sh);
        // scores go over the weights of the step before, whose products need not have run in the order
        // of issue (of different shapes they did not)
        if (walked > 0)
          for (int i = 0; i < 2; ++i) kf_wait(&sh.o_done[i], (walked - 1) & 1, sh);
        __syncwarp();
        tc_fence_after();
        if (kf_elected()) scores(0, walked);
        __syncwarp();
        if (kf_elected()) scores(1, walked);
        __syncwarp();
#pragma unroll 1
        for (int u = 0; u < 2 * steps; ++u) {  // step j of row tile i
          const int i = u & 1, j = u >> 1, at = walked + j;
          if (i == 0) kf_wait(&sh.v_full[at & 1], (at >> 1) & 1, sh);
          kf_wait(&sh.w_full[i], at & 1, sh);
          __syncwarp();
          tc_fence_after();
          if (kf_elected()) {
            const uint64_t y = dv + (at & 1) * (TILE_BYTES >> 4);
#pragma unroll
            for (int ks = 0; ks < KF_KEYS / 16; ++ks)
              umma_f16_ts(tm + 256 + i * 128, tm + i * 128 + ks * 8, y + ks * (2048 >> 4), IDESC_O, j > 0 || ks > 0);
            if (i == 1) umma_commit(&sh.v_empty[at & 1]);
            umma_commit(&sh.o_done[i]);
            if (j + 1 == steps) umma_commit(&sh.o_full[i]);
          }
          __syncwarp();
          if (j + 1 < steps) {
            kf_wait(&sh.o_done[i], at & 1, sh);
            if (i == 0) kf_wait(&sh.k_full[(at + 1) & 1], ((at + 1) >> 1) & 1, sh);
            __syncwarp();
            tc_fence_after();
            if (kf_elected()) scores(i, at + 1);
            __syncwarp();
          }
        }
        walked += steps;
      }
      kf_all_sync();
    } while (more);
    // every product has completed before TMEM is freed, also after a wait that ran out
    if (turns > 0)
      for (int i = 0; i < 2; ++i) mbar_wait_bounded(&sh.o_full[i], (turns - 1) & 1);
  }
  __syncthreads();
  if (tid == 0 && sh.dead && a.error_flag) atomicOr(a.error_flag, MRB_KV_TIMEOUT);
  if (warp == (KF_SOFTMAX + KF_FILL) / 32) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

static int kf_ctas() { return std::min(num_sms(), KF_COUNTERS / 4 - 1); }

static size_t kf_workspace(int64_t d) {  // counters, and two parts a CTA
  return KF_COUNTERS + (size_t)kf_ctas() * 2 * kf_slot((int)d) * sizeof(float);
}

template <int D, int G>
static int launch_prefill(const Kv4PrefillArgs& a, cudaStream_t s) {
  const char* what = "kv4_prefill_attention";
  const size_t smem = 6 * (D / 64) * 16384 + 2 * KF_PASSES * KF_FILL * (D / 8 + 4) + 1024;
  const int rc = ensure_dynamic_smem((const void*)kv4_prefill_kernel<D, G>, smem, what);
  if (rc != MRB_OK) return rc;
  launch_kernel(kv4_prefill_kernel<D, G>, dim3((unsigned)kf_ctas()), dim3(KF_THREADS), smem, s, true, a);
  return launch_status(what);
}

}  // namespace mrb

extern "C" int64_t mrb_kv4_prefill_attention_timeouts(void) {
  unsigned v = 0;
  if (cudaMemcpyFromSymbol(&v, mrb::g_kv4_prefill_timeouts, sizeof(v)) != cudaSuccess) return -1;
  return (int64_t)v;
}

extern "C" size_t mrb_kv4_prefill_attention_workspace(int64_t head_dim) {
  return head_dim == 64 || head_dim == 128 ? mrb::kf_workspace(head_dim) : 0;
}

namespace mrb {
static int prefill(const void* q, int64_t tokens, int64_t rows, int64_t hq, int64_t hkv, int64_t head_dim, int64_t group,
                   const void* pool, int64_t num_pages, int64_t page_size, int64_t stride_page, int64_t stride_head,
                   const int32_t* block_table, int64_t num_seqs, int64_t block_table_stride, int64_t max_pages_per_seq,
                   const int32_t* q_starts, const int32_t* row_seq, const int32_t* row_len, float scale, void* out,
                   bool zero_rest, void* workspace, size_t workspace_bytes, int32_t* error_flag, void* stream) {
  const char* what = "kv4_prefill_attention";
  Kv4PrefillArgs a = {};
  const int rc = kv4_check_attention(what, q, tokens, rows, hq, hkv, head_dim, group, pool, num_pages, page_size,
                                     stride_page, stride_head, block_table, num_seqs, block_table_stride,
                                     max_pages_per_seq, row_len, scale, out, &a.pool);
  if (rc != MRB_OK) return rc;
  if (tokens == 0 || rows == 0) {
    clear_error();
    return MRB_OK;
  }
  if (!q_starts) return fail(MRB_ERR_ARG, "%s: null pointer", what);
  const size_t need = kf_workspace(head_dim);
  if (!workspace || workspace_bytes < need || !aligned(workspace, 16))
    return fail(MRB_ERR_ARG, "%s: needs a 16-byte aligned workspace of %zu bytes", what, need);
  a.q = (const __nv_bfloat16*)q;
  a.out = (__nv_bfloat16*)out;
  a.block_table = block_table;
  a.row_seq = row_seq;
  a.row_len = row_len;
  a.q_starts = q_starts;
  a.error_flag = error_flag;
  a.counters = (unsigned*)workspace;
  a.part = (float*)((char*)workspace + KF_COUNTERS);
  a.tokens = tokens;
  a.zero_rest = zero_rest;
  a.bt_stride = block_table_stride;
  a.num_seqs = num_seqs;
  a.rows = (int)rows;
  a.hq = (int)hq;
  a.cap = (int)(max_pages_per_seq * page_size);
  const uint64_t tiles = (uint64_t)(page_size / KV4_TILE);
  const auto magic = [](uint64_t d) { return d == 1 ? 0u : (uint32_t)(((1ull << 32) + d - 1) / d); };
  a.page_magic = magic(tiles);
  a.group_magic = magic((uint64_t)(hq / hkv));
  a.q_and = scale == 0.f ? 0u : 0xffffffffu;
  a.q_xor = scale < 0.f ? 0x80008000u : 0u;
  a.scale2 = (scale == 0.f ? 1.f : fabsf(scale)) * 1.4426950408889634f;
  cudaStream_t s = (cudaStream_t)stream;
  if (head_dim == 64) return group == 32 ? launch_prefill<64, 32>(a, s) : launch_prefill<64, 64>(a, s);
  if (group == 32) return launch_prefill<128, 32>(a, s);
  if (group == 64) return launch_prefill<128, 64>(a, s);
  return launch_prefill<128, 128>(a, s);
}
}  // namespace mrb

extern "C" int mrb_kv4_prefill_attention(const void* q, int64_t tokens, int64_t rows, int64_t hq, int64_t hkv,
                                         int64_t head_dim, int64_t group, const void* pool, int64_t num_pages,
                                         int64_t page_size, int64_t stride_page, int64_t stride_head,
                                         const int32_t* block_table, int64_t num_seqs, int64_t block_table_stride,
                                         int64_t max_pages_per_seq, const int32_t* q_starts, const int32_t* row_seq,
                                         const int32_t* row_len, float scale, void* out, void* workspace,
                                         size_t workspace_bytes, int32_t* error_flag, void* stream) {
  return mrb::prefill(q, tokens, rows, hq, hkv, head_dim, group, pool, num_pages, page_size, stride_page, stride_head,
                      block_table, num_seqs, block_table_stride, max_pages_per_seq, q_starts, row_seq, row_len, scale,
                      out, false, workspace, workspace_bytes, error_flag, stream);
}

extern "C" int mrb_kv4_prefill_attention_all(const void* q, int64_t tokens, int64_t rows, int64_t hq, int64_t hkv,
                                             int64_t head_dim, int64_t group, const void* pool, int64_t num_pages,
                                             int64_t page_size, int64_t stride_page, int64_t stride_head,
                                             const int32_t* block_table, int64_t num_seqs, int64_t block_table_stride,
                                             int64_t max_pages_per_seq, const int32_t* q_starts,
                                             const int32_t* row_seq, const int32_t* row_len, float scale, void* out,
                                             void* workspace, size_t workspace_bytes, int32_t* error_flag,
                                             void* stream) {
  return mrb::prefill(q, tokens, rows, hq, hkv, head_dim, group, pool, num_pages, page_size, stride_page, stride_head,
                      block_table, num_seqs, block_table_stride, max_pages_per_seq, q_starts, row_seq, row_len, scale,
                      out, true, workspace, workspace_bytes, error_flag, stream);
}
