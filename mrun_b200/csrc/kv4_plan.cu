// The page plan of one serving step, built on the GPU from the requests' lengths: pages taken
// from the free stack, block tables, and each new token's position, sequence and cache slot.
//
// With l_r tokens committed and n_r new ones, request r holds ceil(l_r / P) pages and needs
// ceil((l_r + n_r) / P). Exclusive sums over the requests of n_r and of the fresh pages give
// every token its request and every fresh page its place in the free stack (the j-th fresh page
// is free_pages[free_count - 1 - j]), so the plan depends on the inputs alone.
//
// The work is a few bytes a token, so the time is latency (32 decode requests: 14 us a call from Python, 7
// on the device; 1000 mixed ones, 3.2 MB: 16 us on the device, 26 with clusters of eight CTAs): one
// launch of one cluster. Every CTA
// computes the same sums over all requests in shared memory (they are read by all before any
// state is written, with a cluster barrier between), then the CTAs share the tokens. A step that
// does not fit is found before the barrier, by every CTA alike, and changes nothing.
#include "common.cuh"
#include "qrow_common.cuh"

#include <atomic>

namespace mrb {

constexpr int KP_THREADS = 1024;
constexpr int KP_MAX_ROWS = 8192;
constexpr int KP_MAX_SEQS = 1 << 18;
constexpr int KP_MAX_CTAS = 16;

struct PlanArgs {
  const int32_t* new_tokens;
  const int32_t* row_seq;
  const int32_t* lengths;
  int32_t* lengths_out;
  int32_t* block_table;
  const int32_t* free_pages;
  const int32_t* free_count;
  int32_t* free_count_out;
  int32_t *q_starts, *row_len, *positions, *token_rows, *slots, *error_flag;
  int64_t bt_stride;
  int rows, max_seqs, max_pages, num_free, page_size, max_tokens;
};

// Shared memory, sized by the step: four words a request and one bit a sequence.
struct PlanSmem {
  int* start;      // [rows + 1] tokens before each request
  int* pstart;     // [rows + 1] fresh pages before each request
  int* len;        // [rows] committed tokens
  int* seq;        // [rows] sequence
  uint32_t* seen;  // [max_seqs / 32] sequences of this step
  __device__ PlanSmem(unsigned char* raw, int rows) {
    start = reinterpret_cast<int*>(raw);
    pstart = start + rows + 1;
    len = pstart + rows + 1;
    seq = len + rows;
    seen = reinterpret_cast<uint32_t*>(seq + rows);
  }
  static size_t bytes(int64_t rows, int64_t max_seqs) { return 4 * (4 * rows + 2 + (max_seqs + 31) / 32); }
};

__device__ __forceinline__ int plan_pages(int tokens, int page_size) {  // tokens < 2^31, page_size <= 2^31
  return (int)(((unsigned)tokens + (unsigned)page_size - 1u) / (unsigned)page_size);
}

// the last r in [0, n) with v[r] <= x (v[0] <= x): rows without entries are passed over
__device__ __forceinline__ int plan_find(const int* v, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int m = (lo + hi) >> 1;
    if (v[m] <= x) lo = m; else hi = m;
  }
  return lo;
}

__device__ __forceinline__ void plan_cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

__global__ void __launch_bounds__(KP_THREADS) kv_plan_step_kernel(const PlanArgs a) {
  extern __shared__ __align__(16) unsigned char raw[];
  __shared__ long long wsum[2][KP_THREADS / 32];
  __shared__ int all_bad;
  const PlanSmem s(raw, a.rows);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int gtid = blockIdx.x * KP_THREADS + tid, gsize = gridDim.x * KP_THREADS;
  for (int i = tid; i < (a.max_seqs + 31) / 32; i += KP_THREADS) s.seen[i] = 0u;
  if (tid == 0) all_bad = 0;
  pdl_launch_dependents();
  pdl_wait();
  __syncthreads();

  // ---- every request's tokens and fresh pages; what is wrong with the step
  const int per = (a.rows + KP_THREADS - 1) / KP_THREADS;
  const int r0 = min(tid * per, a.rows), r1 = min(r0 + per, a.rows);
  const int64_t cap = (int64_t)a.max_pages * a.page_size;
  const int have_free = *a.free_count;
  int bad = have_free < 0 || have_free > a.num_free ? MRB_KV_BAD_REQUEST : 0;
  long long toks = 0, pages = 0;
  for (int r = r0; r < r1; ++r) {
    const int seq = a.row_seq ? a.row_seq[r] : r;
    int n = a.new_tokens[r], len = 0, fresh = 0;
    if (seq < 0 || seq >= a.max_seqs || n < 0) {
      bad |= MRB_KV_BAD_REQUEST;
      n = 0;
    } else {
      if (atomicOr(&s.seen[seq >> 5], 1u << (seq & 31)) & (1u << (seq & 31))) bad |= MRB_KV_BAD_REQUEST;
      len = a.lengths[seq];
      if (len < 0 || (int64_t)len + n > cap) {
        bad |= len < 0 ? MRB_KV_BAD_REQUEST : MRB_KV_TABLE_FULL;
        n = 0;
        len = max(len, 0);
      }
      fresh = plan_pages(len + n, a.page_size) - plan_pages(len, a.page_size);
    }
    s.seq[r] = seq;
    s.len[r] = len;
    s.start[r] = n;
    s.pstart[r] = fresh;
    toks += n;
    pages += fresh;
  }
  // block-wide exclusive sums of (tokens, pages)
  long long ti = toks, pi = pages;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long u = __shfl_up_sync(0xffffffffu, ti, o), v = __shfl_up_sync(0xffffffffu, pi, o);
    if (lane >= o) ti += u, pi += v;
  }
  if (lane == 31) wsum[0][warp] = ti, wsum[1][warp] = pi;
  if (bad) atomicOr(&all_bad, bad);
  __syncthreads();
  bad = all_bad;
  long long tb = ti - toks, pb = pi - pages, tall = 0, pall = 0;
#pragma unroll 8
  for (int w = 0; w < KP_THREADS / 32; ++w) {
    if (w < warp) tb += wsum[0][w], pb += wsum[1][w];
    tall += wsum[0][w], pall += wsum[1][w];
  }
  if (tall > a.max_tokens) bad |= MRB_KV_TOKENS_FULL;
  if (!bad && pall > have_free) bad |= MRB_KV_POOL_EMPTY;
  const int total = bad ? 0 : (int)tall, fresh_all = bad ? 0 : (int)pall;
  for (int r = r0; r < r1; ++r) {
    const int n = s.start[r], f = s.pstart[r];
    s.start[r] = bad ? 0 : (int)tb;
    s.pstart[r] = bad ? 0 : (int)pb;
    tb += n;
    pb += f;
  }
  if (tid == 0) s.start[a.rows] = total, s.pstart[a.rows] = fresh_all;
  __syncthreads();
  plan_cluster_sync();  // every CTA has read the old state

  // ---- per request: starts and lengths
  for (int r = gtid; r <= a.rows; r += gsize) {
    a.q_starts[r] = s.start[r];
    if (r == a.rows) break;
    const int now = s.len[r] + (s.start[r + 1] - s.start[r]);
    a.row_len[r] = now;
    if (!bad) a.lengths_out[s.seq[r]] = now;
  }
  if (a.lengths_out != a.lengths)  // the sequences that this step leaves alone
    for (int q = gtid; q < a.max_seqs; q += gsize)
      if (bad || !(s.seen[q >> 5] >> (q & 31) & 1u)) a.lengths_out[q] = a.lengths[q];
  if (gtid == 0) {
    *a.free_count_out = have_free - fresh_all;
    if (bad && a.error_flag) atomicOr(a.error_flag, bad);
  }
  // ---- per fresh page: its table entry
  for (int j = gtid; j < fresh_all; j += gsize) {
    const int r = plan_find(s.pstart, a.rows, j);
    const int at = plan_pages(s.len[r], a.page_size) + (j - s.pstart[r]);
    a.block_table[(int64_t)s.seq[r] * a.bt_stride + at] = a.free_pages[have_free - 1 - j];
  }
  // ---- per token, four to a thread so that the search, the division and the stores are shared and the
  // four page numbers are loaded together
  const int most = INT32_MAX / a.page_size;
  for (int64_t i0 = (int64_t)gtid * 4; i0 < a.max_tokens; i0 += (int64_t)gsize * 4) {
    int pos[4], row[4], slot[4], in[4], page[4];
    int r = -1, at = 0, have = 0;
    const int32_t* fresh = nullptr;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int i = (int)i0 + k;
      pos[k] = row[k] = in[k] = 0;
      page[k] = -1;
      if (i >= total) continue;
      if (r < 0 || i >= s.start[r + 1]) {
        r = plan_find(s.start, a.rows, i);
        pos[k] = s.len[r] + (i - s.start[r]);
        at = (int)((unsigned)pos[k] / (unsigned)a.page_size);
        in[k] = pos[k] - at * a.page_size;
        have = plan_pages(s.len[r], a.page_size);
        fresh = a.free_pages + (have_free - 1 - s.pstart[r] + have);  // less at: its page
      } else {
        pos[k] = pos[k - 1] + 1;
        in[k] = in[k - 1] + 1;
        if (in[k] == a.page_size) in[k] = 0, ++at;
      }
      row[k] = s.seq[r];
      page[k] = *(at < have ? a.block_table + (int64_t)row[k] * a.bt_stride + at : fresh - at);
    }
#pragma unroll
    for (int k = 0; k < 4; ++k)  // -1: an unmapped page, or one whose slots 32 bits cannot number
      slot[k] = page[k] < 0 || page[k] >= most ? -1 : page[k] * a.page_size + in[k];
    if (i0 + 4 <= a.max_tokens) {  // the arrays are 16-byte aligned
      *reinterpret_cast<int4*>(a.positions + i0) = make_int4(pos[0], pos[1], pos[2], pos[3]);
      *reinterpret_cast<int4*>(a.token_rows + i0) = make_int4(row[0], row[1], row[2], row[3]);
      *reinterpret_cast<int4*>(a.slots + i0) = make_int4(slot[0], slot[1], slot[2], slot[3]);
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (i0 + k < a.max_tokens)
          a.positions[i0 + k] = pos[k], a.token_rows[i0 + k] = row[k], a.slots[i0 + k] = slot[k];
    }
  }
}

// Returns the pages of the given sequences to the free stack: in request order, each
// sequence's pages in table order, on top of what is there. One CTA (a step retires a few
// requests; the pages of all of them are a few thousand words).
__global__ void __launch_bounds__(KP_THREADS) kv_release_kernel(const int32_t* seqs, int rows, int32_t* lengths,
                                                               int max_seqs, int32_t* block_table, int64_t bt_stride,
                                                               int max_pages, int32_t* free_pages, int num_free,
                                                               int32_t* free_count, int page_size,
                                                               int32_t* error_flag) {
  __shared__ int count, flag;
  pdl_launch_dependents();
  pdl_wait();
  if (threadIdx.x == 0) count = *free_count, flag = 0;
  __syncthreads();
  for (int r = 0; r < rows; ++r) {
    const int seq = seqs[r];
    const int base = count;
    const int len = seq < 0 || seq >= max_seqs ? -1 : lengths[seq];
    const int pages = len < 0 ? -1 : (int)(((int64_t)len + page_size - 1) / page_size);
    __syncthreads();  // everyone has read count and the length
    if (pages < 0 || pages > max_pages || base < 0 || (int64_t)base + pages > num_free) {
      if (threadIdx.x == 0) flag |= MRB_KV_BAD_REQUEST;
      continue;
    }
    int32_t* row = block_table + (int64_t)seq * bt_stride;
    for (int j = threadIdx.x; j < max_pages; j += KP_THREADS) {
      if (j < pages) free_pages[base + j] = row[j];
      row[j] = -1;
    }
    if (threadIdx.x == 0) lengths[seq] = 0, count = base + pages;
    __syncthreads();
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    *free_count = count;
    if (flag && error_flag) atomicOr(error_flag, flag);
  }
}

}  // namespace mrb

namespace mrb {
// Whether a cluster of KP_MAX_CTAS CTAs, each with `smem` bytes, fits the current device as it is now
// configured: more than eight have to be asked for, and a GPU may have fewer SMs together. Asked once for
// a size that is larger than those that fit, or smaller than those that do not.
static bool plan_wide_clusters(size_t smem) {
  static std::atomic<int64_t> fits[64], fails[64];  // largest and smallest size + 1
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev > 63) return false;
  const int64_t size = (int64_t)smem + 1, bad = fails[dev].load();
  if (size <= fits[dev].load()) return true;
  if (bad && size >= bad) return false;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(KP_MAX_CTAS);
  cfg.blockDim = dim3(KP_THREADS);
  cfg.dynamicSmemBytes = smem;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = KP_MAX_CTAS;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  int clusters = 0;
  const bool ok = cudaFuncSetAttribute((const void*)kv_plan_step_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed,
                                       1) == cudaSuccess &&
                  cudaOccupancyMaxActiveClusters(&clusters, (const void*)kv_plan_step_kernel, &cfg) == cudaSuccess &&
                  clusters > 0;
  if (!ok) cudaGetLastError();
  (ok ? fits : fails)[dev].store(size);
  return ok;
}
}  // namespace mrb

extern "C" int mrb_kv_plan_step(const int32_t* new_tokens, const int32_t* row_seq, int64_t rows,
                                const int32_t* lengths, int32_t* lengths_out, int64_t max_seqs, int32_t* block_table,
                                int64_t block_table_stride, int64_t max_pages_per_seq, const int32_t* free_pages,
                                int64_t num_free, const int32_t* free_count, int32_t* free_count_out,
                                int64_t page_size, int64_t max_tokens, int32_t* q_starts, int32_t* row_len,
                                int32_t* positions, int32_t* token_rows, int32_t* slots, int32_t* error_flag,
                                void* stream) {
  using namespace mrb;
  if (rows < 0 || max_seqs < 1 || max_pages_per_seq < 1 || block_table_stride < max_pages_per_seq || num_free < 0 ||
      page_size < 1 || max_tokens < 0)
    return fail(MRB_ERR_ARG, "kv_plan_step: bad sizes");
  if (rows > KP_MAX_ROWS || max_seqs > KP_MAX_SEQS)
    return fail(MRB_ERR_UNSUPPORTED, "kv_plan_step: at most %d requests a step and %d sequences", KP_MAX_ROWS,
                KP_MAX_SEQS);
  if (max_pages_per_seq > INT32_MAX / page_size || max_tokens > INT32_MAX - 4 || num_free > INT32_MAX)
    return fail(MRB_ERR_UNSUPPORTED, "kv_plan_step: positions, tokens and pages must be numbered in 32 bits");
  if (!lengths || !lengths_out || !block_table || !free_count || !free_count_out || !q_starts ||
      (rows > 0 && (!new_tokens || !row_len)) || (num_free > 0 && !free_pages) ||
      (max_tokens > 0 && (!positions || !token_rows || !slots)))
    return fail(MRB_ERR_ARG, "kv_plan_step: null pointer");
  if (!aligned(positions, 16) || !aligned(token_rows, 16) || !aligned(slots, 16))
    return fail(MRB_ERR_ARG, "kv_plan_step: positions, token_rows and slots must be 16-byte aligned");
  PlanArgs a = {};
  a.new_tokens = new_tokens;
  a.row_seq = row_seq;
  a.lengths = lengths;
  a.lengths_out = lengths_out;
  a.block_table = block_table;
  a.free_pages = free_pages;
  a.free_count = free_count;
  a.free_count_out = free_count_out;
  a.q_starts = q_starts;
  a.row_len = row_len;
  a.positions = positions;
  a.token_rows = token_rows;
  a.slots = slots;
  a.error_flag = error_flag;
  a.bt_stride = block_table_stride;
  a.rows = (int)rows;
  a.max_seqs = (int)max_seqs;
  a.max_pages = (int)max_pages_per_seq;
  a.num_free = (int)num_free;
  a.page_size = (int)page_size;
  a.max_tokens = (int)max_tokens;
  const size_t smem = PlanSmem::bytes(rows, max_seqs);
  const int rc = ensure_dynamic_smem((const void*)kv_plan_step_kernel, smem, "kv_plan_step");
  if (rc != MRB_OK) return rc;
  const int64_t want = (max_tokens + 4 * KP_THREADS - 1) / (4 * KP_THREADS);
  int ctas = 1;
  while (ctas < KP_MAX_CTAS && ctas < want) ctas *= 2;
  if (ctas > 8 && !plan_wide_clusters(smem)) ctas = 8;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(KP_THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = (cudaStream_t)stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ctas;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  cudaLaunchKernelEx(&cfg, kv_plan_step_kernel, a);
  return launch_status("kv_plan_step");
}

extern "C" int mrb_kv_release(const int32_t* seqs, int64_t rows, int32_t* lengths, int64_t max_seqs,
                              int32_t* block_table, int64_t block_table_stride, int64_t max_pages_per_seq,
                              int32_t* free_pages, int64_t num_free, int32_t* free_count, int64_t page_size,
                              int32_t* error_flag, void* stream) {
  using namespace mrb;
  if (rows < 0 || max_seqs < 1 || max_pages_per_seq < 1 || block_table_stride < max_pages_per_seq || num_free < 0 ||
      page_size < 1)
    return fail(MRB_ERR_ARG, "kv_release: bad sizes");
  if (rows > INT32_MAX || max_seqs > INT32_MAX || num_free > INT32_MAX || max_pages_per_seq > INT32_MAX / page_size)
    return fail(MRB_ERR_UNSUPPORTED, "kv_release: positions and pages must be numbered in 32 bits");
  if ((rows > 0 && !seqs) || !lengths || !block_table || !free_count || (num_free > 0 && !free_pages))
    return fail(MRB_ERR_ARG, "kv_release: null pointer");
  if (rows == 0) {
    clear_error();
    return MRB_OK;
  }
  launch_kernel(kv_release_kernel, dim3(1), dim3(KP_THREADS), 0, (cudaStream_t)stream, true, seqs, (int)rows, lengths,
                (int)max_seqs, block_table, block_table_stride, (int)max_pages_per_seq, free_pages, (int)num_free,
                free_count, (int)page_size, error_flag);
  return launch_status("kv_release");
}
