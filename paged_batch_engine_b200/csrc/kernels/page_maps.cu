// The integers of a step made on the device from its requests' lengths: where each request's rows begin, each row's request,
// position and cache slot, and the requests' block tables, from one list of the pages that they hold, request by request.
//
//   need_r  = ceil((context_r + q_len_r) / (P * stride))      first_r = sum of need before r      q_start_r = sum of q_len
//   row t of request r: position = context_r + t - q_start_r, entry = position / stride,
//                       slot = pages[first_r + entry / P] * P + entry % P
//   table[r, i] = pages[first_r + i] for i < need_r, else -1
//
// Every block makes both running sums over the requests for itself (a few hundred additions beside a launch) and then takes
// its share of the rows and table entries; a row finds its request by bisection.  Bound by latency: the integers of 64
// requests of 8,192 tokens are 170 KB and take 4.2 us, those of 15,292 rows of 64 requests (1.7 MB) 5.3.  Sums are 64 bits wide;
// what does not fit an output (a page list that ends early; a slot, position, length or start beyond 2^31 - 1) is written as -1.
#include "common.cuh"
#include "opt_in.cuh"
#include "pdl.cuh"

using namespace pbe;

namespace {
constexpr int THREADS = 512;
constexpr int MOST_REQUESTS = 8192;

struct MapsParams {
  const int32_t* q_len;
  const int32_t* context;
  const int32_t* pages;        // null: pages are numbered as they are needed
  int32_t* q_start;
  int32_t* seq_len;
  int32_t* positions;
  int32_t* request_of_row;
  int32_t* slots;
  int32_t* table;
  int requests, rows, width, page_tokens, stride;
  long long num_pages;
};

// running sum over the block (each thread's own included); `carry` is what came before, and becomes what comes after
__device__ __forceinline__ long long block_scan(long long v, long long* warp_sums, long long& carry) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += u;
  }
  __syncthreads();
  if (lane == 31) warp_sums[warp] = v;
  __syncthreads();
  long long before = carry, all = 0;
  for (int w = 0; w < THREADS / 32; ++w) {
    const long long s = warp_sums[w];
    if (w < warp) before += s;
    all += s;
  }
  carry += all;
  return before + v;
}

__device__ __forceinline__ int fitting(long long x) { return x > 0x7fffffffLL ? -1 : (int)x; }
__device__ __forceinline__ int page_at(const MapsParams& p, long long i) {
  if (p.pages == nullptr) return i < p.num_pages ? (int)i : -1;
  return i < p.num_pages ? p.pages[i] : -1;
}

__global__ void __launch_bounds__(THREADS) page_maps_kernel(MapsParams p) {
  extern __shared__ long long sums[];                  // [requests] ends of the rows, [requests] first pages
  __shared__ long long warp_sums[THREADS / 32];
  long long* row_end = sums;
  long long* first = sums + p.requests;
  pdl_launch_dependents();
  pdl_wait();
  const long long per_page = (long long)p.page_tokens * p.stride;
  long long rows_before = 0, pages_before = 0;
  for (int r0 = 0; r0 < p.requests; r0 += THREADS) {
    const int r = r0 + threadIdx.x;
    const bool live = r < p.requests;
    const long long q = live ? max(0, p.q_len[r]) : 0;
    const long long seq = live ? q + max(0, p.context[r]) : 0;
    const long long need = (seq + per_page - 1) / per_page;
    const long long end = block_scan(q, warp_sums, rows_before);
    const long long last = block_scan(need, warp_sums, pages_before);
    if (live) {
      row_end[r] = end;
      first[r] = last - need;
      if (blockIdx.x == 0) {
        p.q_start[r] = fitting(end - q);
        p.seq_len[r] = fitting(seq);
      }
    }
  }
  __syncthreads();
  const long long items = (long long)p.rows + (long long)p.requests * p.width;
  for (long long item = (long long)blockIdx.x * THREADS + threadIdx.x; item < items; item += (long long)gridDim.x * THREADS) {
    if (item < p.rows) {
      int lo = 0, hi = p.requests;                     // the first request whose rows end behind this row
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (row_end[mid] > item) hi = mid; else lo = mid + 1;
      }
      long long pos = 0, slot = -1;
      if (lo < p.requests) {
        const long long q = max(0, p.q_len[lo]);
        pos = max(0, p.context[lo]) + item - (row_end[lo] - q);
        const long long entry = pos / p.stride;
        const int page = page_at(p, first[lo] + entry / p.page_tokens);
        if (page >= 0) slot = (long long)page * p.page_tokens + entry % p.page_tokens;
      }
      p.positions[item] = fitting(pos);
      p.request_of_row[item] = lo < p.requests ? lo : -1;
      p.slots[item] = fitting(slot);
    } else {
      const long long at = item - p.rows;
      const int r = (int)(at / p.width), i = (int)(at - (long long)r * p.width);
      const long long need = (r + 1 < p.requests ? first[r + 1] : pages_before) - first[r];
      p.table[at] = i < need ? page_at(p, first[r] + i) : -1;
    }
  }
}
}  // namespace

PBE_EXPORT int pbe_page_maps_most_requests() { return MOST_REQUESTS; }

// out: q_start [requests], seq_len [requests], positions [rows], request_of_row [rows], slots [rows], table [requests, width],
// each on the next multiple of four integers.
PBE_EXPORT int pbe_page_maps(const int32_t* q_len, const int32_t* context, const int32_t* pages, long long num_pages,
                             int32_t* out, int requests, int rows, int width, int page_tokens, int stride,
                             cudaStream_t stream) {
  if (requests <= 0 || requests > MOST_REQUESTS || rows < 0 || width < 0 || page_tokens <= 0 || stride <= 0)
    return (int)cudaErrorInvalidValue;
  const size_t r = ((size_t)requests + 3) / 4 * 4, n = ((size_t)rows + 3) / 4 * 4;
  MapsParams p{q_len, context, pages, out, out + r, out + 2 * r, out + 2 * r + n, out + 2 * r + 2 * n, out + 2 * r + 3 * n,
               requests, rows, width, page_tokens, stride, num_pages};
  const size_t smem = (size_t)requests * 2 * sizeof(long long);
  static OptIn opt_in;
  if (smem > 48 * 1024)
    if (const cudaError_t e = opt_in(smem, page_maps_kernel)) return (int)e;
  const long long items = (long long)rows + (long long)requests * width;
  long long blocks = (items + THREADS - 1) / THREADS;
  blocks = blocks < 1 ? 1 : blocks > 148 ? 148 : blocks;
  launch_k(page_maps_kernel, (unsigned)blocks, THREADS, smem, stream, p);
  return launch_status();
}
