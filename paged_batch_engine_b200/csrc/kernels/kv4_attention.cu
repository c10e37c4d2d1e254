// Causal attention over 4-bit pages (kv4.cuh) for decoded tokens and short portions.
//
// Codes are operands as they are.  A code shifted to the low bits of a bfloat16 is the number code * 2^-133 (in bits 4-7,
// sixteen times that), exactly: one AND takes a pair of codes out of a word and makes a tensor-core operand of it, nothing is
// converted and nothing rounded.  The group's numbers come in outside the products:
//   scores   S[h, t] = sum_g s[t, g] (Q_g . code_g)[h, t] + sum_g lo[t, g] Qsum[h, g]
//   output   O[h, c] = sum_t (P[h, t] s[t, g]) code[t, c] + sum_t P[h, t] lo[t, g]
// The first sums run over each group's 32 channels (two mma.sync m16n8k16) and are scaled in float32; the second are one small
// product each, Qsum in three bfloat16 terms.  Q and P carry a factor 2^64, so that the products of the tiny codes stay
// in float32's normal range for |Q| < 2^63 and spans of values below 2^60.
//
// Both products have the keys' or the channels' codes as A (16 keys, 16 channels) and the rows (packed: query row x head of the
// group) as B, eight at a time, so eight rows leave no lane idle; the weights pass from the one's result to the other's operand
// through movmatrix.  Sums are float32; weights times s are rounded to float16 once (2^-11; a running exponent of each row, over
// the s of the values that it sees, keeps them in its range: 2^-20 of the largest keeps all bits, 2^-31 none).  A warp takes tiles of 16 keys, one record each, through a ring of its own in shared
// memory (cp.async, four deep), and keeps a running maximum that moves only when it grew by 2^8.
//
// Work is cut by bytes, not by requests: the tiles of all (request, head, row tile) laid end to end are shared out evenly over
// the blocks, so one long context among short ones leaves no block idle.  A block's warps merge their parts in shared memory;
// an item that several blocks share is merged by a second kernel, always in the blocks' order.  Few items of not too many keys
// (CLUSTER) go to a cluster of blocks each instead, which share its tiles and merge through distributed shared memory: one
// launch less, and no parts in memory.
//
// 28 heads on 4 of 128, bfloat16: 64 requests of 300 to 8,192 keys (175 MB) 58 us, 3.0 TB/s; a tile more costs what 4.9 TB/s
// would, the rest, some 18 us, is the lists, the beginning and end of each block's pieces of items (2.5 us each) and the second
// kernel.  A tile takes 406 instructions a warp, some 185 of them on the ALU pipe (80 to take codes out; eight fewer changed
// nothing), and four blocks a multiprocessor issue 0.57 a scheduler and clock over the whole call: bound by instructions and
// their latencies, not by bytes.  One request of 131,071 keys (40 heads on 8, 168 MB) 53 us; in clusters, 8 of 2,048 keys 11 us,
// one of 777 7 us: chains of latency.
//
// Float32: queries and weights as three bfloat16 terms each.  There the two sums' cancellation would show (a head's output is
// often a fortieth of its values' lo), so codes come as code - 8 (one OR and one subtraction a pair, exact) beside lo + 8 s, and
// what they sum to is small where the output is: 2.2e-6 of the output's norm from 64 bits without, 4e-7 so
// (a plain float32 implementation 9.5e-7).
#include <cooperative_groups.h>
#include <cuda_fp16.h>

#include <atomic>

#include "common.cuh"
#include "kv4.cuh"
#include "kv4_params.cuh"
#include "mma_sync.cuh"
#include "opt_in.cuh"
#include "pdl.cuh"

using namespace pbe;
using namespace pbe::kv4;
using namespace pbe::mma_sync;
namespace cg = cooperative_groups;

namespace {
struct Shared {                // an item that several blocks share, as the block that begins it notes it
  int parts, slot;             // parts: 0: none.  The first part's slot; the others' are 2 (block + 1), 2 (block + 2), ...
  int rows, q_start;           // its packed rows (at most a tile's) and the query row of the first
  int head, first;             // first head of its key/value head; packed row of the first, within the request
  int pad[2];
};
struct Split {
  float* part_o;               // [2 blocks][rows of a tile][D]
  float* part_ml;              // [2 blocks][rows of a tile][2]
  Shared* shared;              // [blocks]
  int most_packed;             // requests of more packed rows are another kernel's
};

constexpr int WARPS = 4;
constexpr int STAGES = 4;
constexpr int MIN_UNITS = 8;   // tiles a block takes at least, two a warp: KV4_UNITS of ops.py, which sizes the grid by it
constexpr int MOST_REQUESTS = 8192;
constexpr float UP = 18446744073709551616.f;           // 2^64
constexpr float CODE = 590295810358705651712.f;        // 2^69 = 2^133 / 2^64: products of bfloat16 codes
constexpr float CODE16 = 16777216.f;                   // 2^24: products of float16 codes
constexpr int ROOM = 6;                                // weights are kept 2^6 times too large
constexpr int MOST_E = 60;

struct Request {
  int rows, seq, pos0, first, tiles, row_tiles;        // first: the first 16-key tile, tiles: how many, at least one
};
__device__ __forceinline__ Request request(const Kv4AttnParams& p, const Split& s, int rows, int seq, int tile_rows) {
  Request q;
  q.rows = max(0, rows);
  q.seq = max(0, seq);
  q.pos0 = q.seq - q.rows;
  const long long packed = (long long)q.rows * (p.heads / p.kv_heads);
  q.row_tiles = packed > s.most_packed ? 0 : (int)((packed + tile_rows - 1) / tile_rows);      // tile_rows: 8 or 16
  const int low = p.window > 0 ? max(0, max(0, q.pos0) - p.window + 1) : 0;    // (rows before the first key see none)
  q.first = low / REC_TOKENS;
  q.tiles = max(1, (int)(((unsigned)q.seq + REC_TOKENS - 1) / REC_TOKENS) - q.first);
  return q;
}
// a / b, a not negative: almost always in 32 bits, where a division is a tenth of one in 64
__device__ __forceinline__ long long quotient(long long a, int b) {
  return a >> 32 ? a / b : (long long)((unsigned)a / (unsigned)b);
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ unsigned pack2(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const unsigned*>(&h);
}
__device__ __forceinline__ unsigned pack2_f16(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const unsigned*>(&h);
}
__device__ __forceinline__ unsigned transposed(unsigned x) {
  unsigned y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
// a product alone, with nothing added to it
__device__ __forceinline__ void mma_first(float (&c)[4], const unsigned (&a)[4], unsigned b0, unsigned b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ void mma_f16(float (&c)[4], const unsigned (&a)[4], unsigned b0, unsigned b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float low_half(unsigned w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float high_half(unsigned w) { return __uint_as_float(w & 0xffff0000u); }
// the even codes of a word's halves, less 8, as bfloat16: 128 + code is one OR away, and 136 from it exact
__device__ __forceinline__ unsigned centred(unsigned w) {
  const unsigned x = (w & 0x000f000fu) | 0x43004300u, mid = 0x43084308u;
  const __nv_bfloat162 y = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&x), *reinterpret_cast<const __nv_bfloat162*>(&mid));
  return *reinterpret_cast<const unsigned*>(&y);
}
// x and y as pairs of N bfloat16 terms, the largest first
template <int N>
__device__ __forceinline__ void split(float x, float y, unsigned (&t)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    t[i] = pack2(x, y);
    x -= low_half(t[i]);
    y -= high_half(t[i]);
  }
}
// the half `sel` names (HALF0 or HALF1) of a word, a bfloat16, as a float
constexpr unsigned HALF0 = 0x1044, HALF1 = 0x3244;
__device__ __forceinline__ float half_of(unsigned w, unsigned sel) { return __uint_as_float(__byte_perm(w, 0u, sel)); }
// N words from shared memory, as wide as they come
template <int N>
__device__ __forceinline__ void words(unsigned (&w)[N], const unsigned char* p) {
  static_assert(N == 2 || N == 4, "");
  if constexpr (N == 4) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
  } else {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    w[0] = v.x, w[1] = v.y;
  }
}

// T: the queries' type; NT: tiles of eight packed rows a warp; TERMS: bfloat16 terms of queries and weights; CLUSTER: an item
// has a cluster of blocks
template <typename T, int D, int NT, int TERMS, bool CLUSTER>
__global__ void __launch_bounds__(WARPS * 32, (TERMS == 1 && (NT == 1 || D == 64)) ? 4 : 2)
kv4_attention_kernel(Kv4AttnParams p, Split sp) {
  constexpr int G = D / GROUP, REC = rec_bytes(D), MT = 8 * NT, RING = WARPS * STAGES * REC;
  constexpr int MERGE = WARPS * MT * (D + 2 + G) * 4;
  constexpr int SHARED = RING > MERGE ? RING : MERGE;
  extern __shared__ __align__(16) unsigned char smem[];
  float* merged = reinterpret_cast<float*>(smem + SHARED);           // CLUSTER: this block's part [row][D], then [row][2]
  // where each request's units (CLUSTER: items) end
  long long* ends = reinterpret_cast<long long*>(smem + SHARED + (CLUSTER ? MT * (D + 2) * 4 : 0));
  int2* known = reinterpret_cast<int2*>(ends + p.requests);          // its q_len and seq_len
  int* starts = reinterpret_cast<int*>(known + p.requests);          // its q_start
  __shared__ long long warp_sums[WARPS];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r8 = lane >> 2, j = lane & 3;
  const int H = p.heads, KV = p.kv_heads, HG = H / KV, per_page = p.page_tokens / REC_TOKENS;
  const int page_shift = (per_page & (per_page - 1)) == 0 ? 31 - __clz(per_page) : -1;
  // With settled inputs only the queries and the newest keys are waited for: the lists are made, and the first tiles asked for,
  // beside the launch that writes those.
  bool waited = !p.settled;
  if (waited) pdl_wait();

  // a unit: one tile of 16 keys for one head and row tile
  long long total = 0;
  for (int r0 = 0; r0 < p.requests; r0 += WARPS * 32) {
    const int r = r0 + threadIdx.x;
    long long v = 0;
    if (r < p.requests) {
      const int2 x = make_int2(p.q_len[r], p.seq_len[r]);
      known[r] = x;
      starts[r] = p.q_start[r];
      const Request q = request(p, sp, x.x, x.y, MT);
      v = (long long)(CLUSTER ? 1 : q.tiles) * q.row_tiles * KV;
    }
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long u = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += u;
    }
    if (lane == 31) warp_sums[warp] = v;
    __syncthreads();
    long long before = total;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      if (w < warp) before += warp_sums[w];
      total += warp_sums[w];
    }
    if (r < p.requests) ends[r] = before + v;
    __syncthreads();
  }
  const long long per_block = CLUSTER ? 0 : max((long long)MIN_UNITS, quotient(total + gridDim.x - 1, gridDim.x));
  pdl_launch_dependents();
  const float to_log2 = p.scale * 1.4426950408889634f * (TERMS == 1 ? CODE : 1.f);

  unsigned char* ring = smem + warp * STAGES * REC;
  const int ranks = CLUSTER ? (int)cg::this_cluster().num_blocks() : 1, rank = CLUSTER ? (int)cg::this_cluster().block_rank() : 0;
  long long unit = CLUSTER ? blockIdx.x / ranks : per_block * blockIdx.x;
  const long long unit0 = unit, unit_end = CLUSTER ? total : min(unit + per_block, total);
  Shared note = {};
  while (unit < unit_end) {
    // ---- the next item, or this block's part of it
    int req = 0;                                       // the first request whose units end behind this one
    for (;; req += 32) {
      const unsigned past = __ballot_sync(0xffffffffu, req + lane < p.requests && ends[req + lane] > unit);
      if (past != 0) {
        req += __ffs(past) - 1;
        break;
      }
    }
    const int2 given = known[req];
    const Request q = request(p, sp, given.x, given.y, MT);
    const long long begin = req > 0 ? ends[req - 1] : 0;
    const int item = (int)(CLUSTER ? unit - begin : quotient(unit - begin, q.tiles));
    const int t_begin = (int)(CLUSTER ? (long long)q.tiles * rank / ranks : (unit - begin) - (long long)item * q.tiles);
    const int t_end = (int)(CLUSTER ? (long long)q.tiles * (rank + 1) / ranks : min((long long)q.tiles, t_begin + (unit_end - unit)));
    const int kvh = q.row_tiles == 1 ? item : item / q.row_tiles, row_tile = item - kvh * q.row_tiles;
    const int packed = q.rows * HG, pr0 = row_tile * MT;
    const int q0 = starts[req];
    auto row_of = [&](int pr) { return q.rows == 1 ? 0 : pr / HG; };     // the request's row of a packed one
    const int pos_min = q.pos0 + row_of(pr0), pos_max = q.pos0 + row_of(min(pr0 + MT, packed) - 1);
    const int low_min = p.window > 0 ? max(0, pos_min) - p.window + 1 : 0, low_max = p.window > 0 ? max(0, pos_max) - p.window + 1 : 0;

    // ---- this warp's tiles, t_begin + warp, + WARPS, ...: the first are on their way before the queries are looked at
    const int mine = t_end - t_begin > warp ? (t_end - t_begin - warp + WARPS - 1) / WARPS : 0;
    const int32_t* table = p.block_table + (long long)req * p.bt_stride;
    auto record = [&](int i) {                         // the record of this warp's tile i, -1: none to be seen
      if (i >= mine) return -1;
      const int t = q.first + t_begin + warp + i * WARPS, blk = page_shift >= 0 ? t >> page_shift : t / per_page;
      if (blk >= p.table_pages || t * REC_TOKENS > pos_max || t * REC_TOKENS + REC_TOKENS <= low_min) return -1;
      const int page = table[blk];
      return page >= 0 && page < p.num_pages ? (page * KV + kvh) * per_page + (t - blk * per_page) : -1;
    };
    int recs = record(lane), recs_next = record(32 + lane);
    unsigned there = 0;                                // bit i: the tile issued i tiles ago has a record
    auto issue = [&](int i) {
      if (i > 0 && (i & 31) == 0) {
        recs = recs_next;
        recs_next = record(i + 32 + lane);
      }
      const int rec = __shfl_sync(0xffffffffu, recs, i & 31);
      there = there << 1 | (rec >= 0 ? 1u : 0u);
      if (rec >= 0) {
        const unsigned char* src = p.pages + (long long)rec * REC + lane * 16;
        unsigned char* dst = ring + (i % STAGES) * REC + lane * 16;
#pragma unroll
        for (int c = 0; c < (REC + 511) / 512; ++c)
          if (REC % 512 == 0 || c * 512 + lane * 16 < REC) cp16(dst + c * 512, src + c * 512, true);
      }
      cp_commit();
    };
    if (!waited && mine > 0) {                         // tiles that hold keys of this step's own rows come after the wait
      const int last = q.first + t_begin + warp + min(STAGES - 2, mine - 1) * WARPS;
      if ((long long)(last + 1) * REC_TOKENS > q.pos0) {
        pdl_wait();
        waited = true;
      }
    }
#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i) issue(i);
    if (!waited) pdl_wait();
    waited = true;

    // this lane's rows of the scores, 8 k + 2 j and the next, and their positions
    int pos[NT][2];
#pragma unroll
    for (int k = 0; k < NT; ++k)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int pr = pr0 + 8 * k + 2 * j + e;
        pos[k][e] = pr < packed ? q.pos0 + row_of(pr) : -1;
      }
    // ---- queries: B fragments (row 8 k + r8), and their sums over each group
    unsigned qb[TERMS][G * 2][NT][2], zb[NT][2];
    float qs[NT][2][G];                                // TERMS > 1: the sums of this lane's rows of the scores
#pragma unroll
    for (int k = 0; k < NT; ++k) {
      const int pr = pr0 + 8 * k + r8;
      const int row = row_of(pr);
      const bool live = pr < packed && q0 >= 0 && q0 + row < p.rows;
      const T* src = (const T*)p.q + (live ? ((size_t)(q0 + row) * H + kvh * HG + (pr - row * HG)) * D + 8 * j : 0);
      float qsum[G];
#pragma unroll
      for (int g = 0; g < G; ++g) {
        float x[8];
        if constexpr (sizeof(T) == 2) {
          uint4 w = make_uint4(0, 0, 0, 0);
          if (live) w = *reinterpret_cast<const uint4*>(src + 32 * g);
          const unsigned u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
          for (int i = 0; i < 4; ++i) x[2 * i] = low_half(u[i]), x[2 * i + 1] = high_half(u[i]);
        } else {
          float4 a = make_float4(0, 0, 0, 0), b = a;
          if (live) {
            a = *reinterpret_cast<const float4*>(src + 32 * g);
            b = *reinterpret_cast<const float4*>(src + 32 * g + 4);
          }
          x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
        }
        qsum[g] = ((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7]));
        qsum[g] += __shfl_xor_sync(0xffffffffu, qsum[g], 1);
        qsum[g] += __shfl_xor_sync(0xffffffffu, qsum[g], 2);
#pragma unroll
        for (int i = 0; i < 4; ++i) {                  // pair i of the word: its codes come 16 times too large for odd i
          const float f = TERMS > 1 ? 1.f : i & 1 ? UP / 16.f : UP;
          unsigned t[TERMS];
          split<TERMS>(x[2 * i] * f, x[2 * i + 1] * f, t);
#pragma unroll
          for (int e = 0; e < TERMS; ++e) qb[e][2 * g + (i >> 1)][k][i & 1] = t[e];
        }
      }
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int g = 0; g < G; ++g) qs[k][e][g] = TERMS > 1 ? __shfl_sync(0xffffffffu, qsum[g], (2 * j + e) * 4) : 0.f;
      // TERMS == 1: three terms of the sums along the product's k: term * G + g
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int at = 2 * j + 8 * half, term = at / G, g0 = at % G;
        float a = 0.f, b = 0.f;
#pragma unroll
        for (int g = 0; g < G; g += 2)
          if (g == g0) a = qsum[g] / CODE, b = qsum[g + 1] / CODE;
        unsigned t[3];
        split<3>(a, b, t);
        zb[k][half] = term == 0 ? t[0] : term == 1 ? t[1] : term == 2 ? t[2] : 0u;
      }
    }

    float o[NT][2 * G][4] = {}, z[NT][G][2] = {}, m[NT][2], l[NT][2] = {};
    float e_run[NT][2];                                // a row's exponent: whole numbers, as they enter the weights' exponent
    int e_low = MOST_E;                                // the least of the lane's; rows that are none have the most
#pragma unroll
    for (int k = 0; k < NT; ++k)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        m[k][e] = -INFINITY;
        e_run[k][e] = pos[k][e] < 0 ? MOST_E : -MOST_E;
        e_low = min(e_low, pos[k][e] < 0 ? MOST_E : -MOST_E);
      }
    const unsigned mine_half = r8 & 1 ? HALF1 : HALF0, both_halves = r8 & 1 ? 0x7632 : 0x5410;

    auto code = [](unsigned w) { return TERMS > 1 ? centred(w) : w & 0x000f000fu; };
    auto code16 = [](unsigned w) { return TERMS > 1 ? centred(w >> 4) : w & 0x00f000f0u; };
    for (int i = 0; i < mine; ++i) {
      cp_wait<STAGES - 2>();
      __syncwarp();                                    // the tile has landed, and the one before is read
      const bool seen = there >> (STAGES - 2) & 1;
      const unsigned char* rec = ring + (i % STAGES) * REC;
      issue(i + STAGES - 1);
      if (!seen) continue;
      const int key0 = (q.first + t_begin + warp + i * WARPS) * REC_TOKENS;
      const unsigned char* num = rec + numbers(D);

      // ---- scores of keys r8 and r8 + 8
      unsigned kw[2][G];
      float ks[2][G], s[NT][4];                        // s: [key r8, rows 2j, 2j + 1, then key r8 + 8]
      unsigned lo[2];
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        unsigned w[G];
        words<G>(kw[n], rec + (n * 8 + r8) * (D / 2) + j * (4 * G));
        words<G>(w, num + K_S * D + (n * 4 + (r8 >> 1)) * (4 * G));
#pragma unroll
        for (int g = 0; g < G; ++g) ks[n][g] = half_of(w[g], mine_half);
        if constexpr (TERMS == 1) {
          unsigned u[2];
          words<2>(u, num + K_LO * D + (n * 4 + (r8 >> 1)) * (4 * G) + (G == 4 ? (j & 1) * 8 : 0));
          lo[n] = __byte_perm(u[0], u[1], both_halves);
        } else {
          words<G>(w, num + K_LO * D + (n * 4 + (r8 >> 1)) * (4 * G));
#pragma unroll
          for (int k = 0; k < NT; ++k)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              s[k][2 * n + e] = 0.f;
#pragma unroll
              for (int g = 0; g < G; ++g) {
                const float middle = fmaf(8.f, ks[n][g], half_of(w[g], mine_half));
                s[k][2 * n + e] = fmaf(middle, qs[k][e][g], s[k][2 * n + e]);
              }
            }
        }
      }
      if constexpr (TERMS == 1) {
        const unsigned a[4] = {lo[0], lo[1], lo[0], lo[1]};
#pragma unroll
        for (int k = 0; k < NT; ++k) mma_first(s[k], a, zb[k][0], zb[k][1]);
      }
#pragma unroll
      for (int g = 0; g < G; ++g) {
        float c[NT][4];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const unsigned x = h ? kw[0][g] >> 8 : kw[0][g], y = h ? kw[1][g] >> 8 : kw[1][g];
          const unsigned a[4] = {code(x), code(y), code16(x), code16(y)};
#pragma unroll
          for (int k = 0; k < NT; ++k)
#pragma unroll
            for (int e = 0; e < TERMS; ++e) {
              const unsigned(&b)[2] = qb[e][2 * g + h][k];
              if (h == 0 && e == 0) mma_first(c[k], a, b[0], b[1]);
              else mma(c[k], a, b[0], b[1]);
            }
        }
#pragma unroll
        for (int k = 0; k < NT; ++k) {
          s[k][0] = fmaf(ks[0][g], c[k][0], s[k][0]);
          s[k][1] = fmaf(ks[0][g], c[k][1], s[k][1]);
          s[k][2] = fmaf(ks[1][g], c[k][2], s[k][2]);
          s[k][3] = fmaf(ks[1][g], c[k][3], s[k][3]);
        }
      }
      // ---- the values' numbers of the same keys
      float vs[2][G], vlo[2][G];
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        unsigned w[G], u[G];
        words<G>(w, num + V_S * D + (n * 4 + (r8 >> 1)) * (4 * G));
        words<G>(u, num + V_LO * D + (n * 4 + (r8 >> 1)) * (4 * G));
#pragma unroll
        for (int g = 0; g < G; ++g) vs[n][g] = half_of(w[g], mine_half), vlo[n][g] = half_of(u[g], mine_half);
      }
#pragma unroll
      for (int k = 0; k < NT; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[k][e] *= to_log2;
      // ---- masks, on the tiles that need them
      if (key0 + REC_TOKENS - 1 > pos_min || key0 < low_max) {
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          const int key = key0 + n * 8 + r8;
#pragma unroll
          for (int k = 0; k < NT; ++k)
#pragma unroll
            for (int e = 0; e < 2; ++e)
              if (key > pos[k][e] || (p.window > 0 && key <= pos[k][e] - p.window)) s[k][2 * n + e] = -INFINITY;
          if (key > pos_max || key < low_min) {        // numbers of places that hold no key of this row tile may be anything
#pragma unroll
            for (int g = 0; g < G; ++g) vs[n][g] = vlo[n][g] = 0.f;
          }
        }
      }
      // ---- the running maximum, moved only when it grew by more than 2^8, or with it the largest exponent of the values' s that
      // the row has seen (a row's own: what it does not see leaves its weights as they are)
      bool grew = false;
#pragma unroll
      for (int k = 0; k < NT; ++k)
#pragma unroll
        for (int e = 0; e < 2; ++e) grew = grew || fmaxf(s[k][e], s[k][2 + e]) > m[k][e] + 8.f;
      float large[2] = {0.f, 0.f};
      if constexpr (TERMS == 1) {
#pragma unroll
        for (int g = 0; g < G; ++g) large[0] = fmaxf(large[0], vs[0][g]), large[1] = fmaxf(large[1], vs[1][g]);
        grew = grew || (int)(__float_as_uint(fmaxf(large[0], large[1])) >> 23) - 127 > e_low;
      }
      if (__any_sync(0xffffffffu, grew)) {
        e_low = MOST_E;
#pragma unroll
        for (int k = 0; k < NT; ++k)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float top = fmaxf(s[k][e], s[k][2 + e]);
            float most = fmaxf(s[k][e] == -INFINITY ? 0.f : large[0], s[k][2 + e] == -INFINITY ? 0.f : large[1]);
#pragma unroll
            for (int off = 4; off < 32; off <<= 1) {
              top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
              if constexpr (TERMS == 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, off));
            }
            top = fmaxf(top, m[k][e]);
            const int e_now = TERMS == 1 ? max((int)e_run[k][e], min((int)(__float_as_uint(most) >> 23) - 127, MOST_E)) : 0;
            const float a = top == -INFINITY ? 1.f : ex2(m[k][e] - top + (TERMS == 1 ? e_run[k][e] - (float)e_now : 0.f));
            m[k][e] = top;
            e_run[k][e] = e_now;
            e_low = min(e_low, e_now);
            l[k][e] *= a;
#pragma unroll
            for (int c = 0; c < 2 * G; ++c) o[k][c][e] *= a, o[k][c][2 + e] *= a;
#pragma unroll
            for (int g = 0; g < G; ++g) z[k][g][e] *= a;
          }
      }
      // ---- weights, and the values' lo (or middle) that they weigh
      if constexpr (TERMS > 1) {
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int g = 0; g < G; ++g) vlo[n][g] = fmaf(8.f, vs[n][g], vlo[n][g]);
      }
      float w[NT][4];
#pragma unroll
      for (int k = 0; k < NT; ++k)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          // the difference first: it is exact near the maximum, however far that is from zero
          const float top = m[k][e] == -INFINITY ? 0.f : m[k][e];
#pragma unroll
          for (int n = 0; n < 2; ++n) {
            const float d = s[k][2 * n + e] - top;
            w[k][2 * n + e] = TERMS == 1 ? ex2(d + (ROOM - e_run[k][e])) : exp2f(d);
          }
          l[k][e] += w[k][e] + w[k][2 + e];
#pragma unroll
          for (int g = 0; g < G; ++g) z[k][g][e] = fmaf(w[k][e], vlo[0][g], fmaf(w[k][2 + e], vlo[1][g], z[k][g][e]));
        }
      // ---- the codes that they weigh
      unsigned v0[G], v1[G];
      words<G>(v0, rec + v_codes(D) + j * D + r8 * (4 * G));
      words<G>(v1, rec + v_codes(D) + (j + 4) * D + r8 * (4 * G));
#pragma unroll
      for (int g = 0; g < G; ++g) {
        unsigned b[NT][2][TERMS];
#pragma unroll
        for (int k = 0; k < NT; ++k)
#pragma unroll
          for (int n = 0; n < 2; ++n) {
            const float x = w[k][2 * n] * vs[n][g], y = w[k][2 * n + 1] * vs[n][g];
            if constexpr (TERMS == 1) b[k][n][0] = pack2_f16(x, y);
            else split<TERMS>(x, y, b[k][n]);
#pragma unroll
            for (int e = 0; e < TERMS; ++e) b[k][n][e] = transposed(b[k][n][e]);
          }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const unsigned x = h ? v0[g] >> 8 : v0[g], y = h ? v1[g] >> 8 : v1[g];
          const unsigned a[4] = {code(x), code16(x), code(y), code16(y)};
#pragma unroll
          for (int k = 0; k < NT; ++k)
#pragma unroll
            for (int e = 0; e < TERMS; ++e) {
              if constexpr (TERMS == 1) mma_f16(o[k][2 * g + h], a, b[k][0][e], b[k][1][e]);
              else mma(o[k][2 * g + h], a, b[k][0][e], b[k][1][e]);
            }
        }
      }
    }
    cp_wait<0>();
    __syncthreads();                                   // every warp is through with its ring

    // ---- the block's warps merged
    float* om = reinterpret_cast<float*>(smem);        // [warp][row][D]
    float* mm = om + WARPS * MT * D;                   // [warp][row]
    float* lm = mm + WARPS * MT;
    constexpr float even = TERMS == 1 ? CODE16 : 1.f, odd = TERMS == 1 ? even / 16.f : 1.f;
    float* zm = lm + WARPS * MT;                       // [warp][row][G]
#pragma unroll
    for (int k = 0; k < NT; ++k) {
      float unit[2];                                   // of the row's weights
#pragma unroll
      for (int e = 0; e < 2; ++e) unit[e] = TERMS == 1 ? ex2(e_run[k][e] - ROOM) : 1.f;
      // the sums over the keys' lanes of the values' lo: by halves, so that lane r8 is left with one of the 2 G sums (two
      // lanes with the same one where there are four)
      float v[2 * G];
#pragma unroll
      for (int i = 0; i < 2 * G; ++i) v[i] = z[k][i >> 1][i & 1] * unit[i & 1];
#pragma unroll
      for (int n = G, off = 16; n > 0; n >>= 1, off >>= 1) {
        const bool up = lane & off;
#pragma unroll
        for (int i = 0; i < n; ++i) {
          const float other = __shfl_xor_sync(0xffffffffu, up ? v[i] : v[n + i], off);
          v[i] = (up ? v[n + i] : v[i]) + other;
        }
      }
      if (G == 2) v[0] += __shfl_xor_sync(0xffffffffu, v[0], 4);
      const int which = G == 4 ? r8 : r8 >> 1;
      zm[(warp * MT + 8 * k + 2 * j + (which & 1)) * G + (which >> 1)] = v[0];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) l[k][e] += __shfl_xor_sync(0xffffffffu, l[k][e], off);
        const int row = warp * MT + 8 * k + 2 * j + e;
        if (r8 == 0) {
          mm[row] = m[k][e];
          lm[row] = l[k][e] * unit[e];
        }
#pragma unroll
        for (int g = 0; g < G; ++g) {
          const float(&a)[4] = o[k][2 * g], (&b)[4] = o[k][2 * g + 1], x = even * unit[e], y = odd * unit[e];
          *reinterpret_cast<float4*>(om + row * D + 32 * g + 4 * r8) = make_float4(a[e] * x, a[2 + e] * y, b[e] * x, b[2 + e] * y);
        }
      }
    }
    __syncthreads();
    const bool whole = !CLUSTER && t_begin == 0 && t_end == q.tiles;
    const int slot = 2 * blockIdx.x + (unit == unit0 ? 0 : 1);
    auto finish = [&](int row, int c4, float4 x, float sum) {
      const int pr = pr0 + row, at = row_of(pr);
      if (pr >= packed || q0 < 0 || q0 + at >= p.rows) return;
      const float inv = sum > 0.f ? 1.f / sum : sum == 0.f ? 0.f : sum;      // a row whose scores are NaN stays NaN
      T* dst = (T*)p.out + ((size_t)(q0 + at) * H + kvh * HG + (pr - at * HG)) * D + c4;
      if constexpr (sizeof(T) == 2)
        *reinterpret_cast<uint2*>(dst) = make_uint2(pack2(x.x * inv, x.y * inv), pack2(x.z * inv, x.w * inv));
      else
        *reinterpret_cast<float4*>(dst) = make_float4(x.x * inv, x.y * inv, x.z * inv, x.w * inv);
    };
    if (!CLUSTER && t_begin == 0 && !whole) {
      const int last = (int)quotient(unit + q.tiles - 1, (int)per_block);
      note = {last - (int)blockIdx.x + 1, slot, min(MT, packed - pr0), q0, kvh * HG, pr0, {0, 0}};
    }
    for (int e = threadIdx.x; e < MT * (D / 4); e += WARPS * 32) {
      const int row = e / (D / 4), c4 = (e % (D / 4)) * 4;
      float top = -INFINITY;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) top = fmaxf(top, mm[w * MT + row]);
      const float base = top == -INFINITY ? 0.f : top;
      float sum = 0.f;
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < WARPS; ++w) {
        const float f = TERMS == 1 ? ex2(mm[w * MT + row] - base) : exp2f(mm[w * MT + row] - base);
        const float4 y = *reinterpret_cast<const float4*>(om + (w * MT + row) * D + c4);
        const float lean = zm[(w * MT + row) * G + c4 / GROUP];
        sum = fmaf(f, lm[w * MT + row], sum);
        x.x = fmaf(f, y.x + lean, x.x), x.y = fmaf(f, y.y + lean, x.y);
        x.z = fmaf(f, y.z + lean, x.z), x.w = fmaf(f, y.w + lean, x.w);
      }
      if (CLUSTER) {
        *reinterpret_cast<float4*>(merged + row * D + c4) = x;
        if (c4 == 0) *reinterpret_cast<float2*>(merged + MT * D + row * 2) = make_float2(top, sum);
      } else if (!whole) {
        const size_t at = (size_t)slot * MT + row;
        *reinterpret_cast<float4*>(sp.part_o + at * D + c4) = x;
        if (c4 == 0) sp.part_ml[at * 2] = top, sp.part_ml[at * 2 + 1] = sum;
      } else {
        finish(row, c4, x, sum);
      }
    }
    if constexpr (CLUSTER) {
      // every block merges a slice of the rows and channels of all blocks' parts, in the order of their ranks
      cg::cluster_group cluster = cg::this_cluster();
      cluster.sync();
      const int each = (MT * (D / 4) + ranks - 1) / ranks;
      for (int i = threadIdx.x; i < each && rank * each + i < MT * (D / 4); i += WARPS * 32) {
        const int row = (rank * each + i) / (D / 4), c4 = ((rank * each + i) % (D / 4)) * 4;
        float top = -INFINITY, sum = 0.f;
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
        for (int r = 0; r < ranks; ++r) top = fmaxf(top, cluster.map_shared_rank(merged, r)[MT * D + row * 2]);
        const float base = top == -INFINITY ? 0.f : top;
#pragma unroll 8
        for (int r = 0; r < ranks; ++r) {
          const float* part = cluster.map_shared_rank(merged, r);
          const float2 ml = *reinterpret_cast<const float2*>(part + MT * D + row * 2);
          const float4 y = *reinterpret_cast<const float4*>(part + row * D + c4);
          const float f = TERMS == 1 ? ex2(ml.x - base) : exp2f(ml.x - base);
          sum = fmaf(f, ml.y, sum);
          x.x = fmaf(f, y.x, x.x), x.y = fmaf(f, y.y, x.y), x.z = fmaf(f, y.z, x.z), x.w = fmaf(f, y.w, x.w);
        }
        finish(row, c4, x, sum);
      }
      cluster.sync();                                  // nobody's part is written anew, or gone, while it is read
      unit += gridDim.x / ranks;
      continue;
    }
    __syncthreads();                                   // the merged parts are read before the ring is filled again
    unit += t_end - t_begin;
  }
  if (!waited) pdl_wait();                             // what comes after this kernel counts on all that came before it
  if (!CLUSTER && threadIdx.x == 0) sp.shared[blockIdx.x] = note;
}

// Items that several blocks share: block b merges the one that block b of the kernel above began and did not end.  A warp
// takes one row and every PARTS-th of the item's parts (one request of 32,768 keys has 74, whose loads one warp a row would
// wait for in turn: 53 us), eight loads on their way.
constexpr int MERGE_WARPS = 16;

template <typename T, int D, int MT, int ROWS>         // MT rows a tile, ROWS of them a block
__global__ void __launch_bounds__(MERGE_WARPS * 32) kv4_merge_kernel(Kv4AttnParams p, Split sp) {
  static_assert(MT % ROWS == 0 && MERGE_WARPS % ROWS == 0, "a warp a row and part");
  constexpr int PARTS = MERGE_WARPS / ROWS, C = D / 32;  // C: columns a lane
  __shared__ float held[PARTS > 1 ? PARTS : 1][ROWS][D], held_m[MERGE_WARPS], held_l[MERGE_WARPS];
  pdl_launch_dependents();
  pdl_wait();
  const Shared item = sp.shared[blockIdx.x];
  if (item.parts == 0) return;
  const int H = p.heads, HG = H / p.kv_heads, last = item.parts - 1;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, in_block = warp % ROWS, part = warp / ROWS;
  const int row = blockIdx.y * ROWS + in_block;
  auto slot = [&](int i) { return (size_t)(i == 0 ? item.slot : 2 * ((int)blockIdx.x + i)) * MT + row; };
  float top = -INFINITY, sum = 0.f, x[C] = {};
  for (int b = part; b <= last; b += PARTS * 32) {                 // 32 of the warp's parts at a time
    const int n = min(32, (last - b) / PARTS + 1);
    const float m = lane < n ? sp.part_ml[slot(b + lane * PARTS) * 2] : -INFINITY;
    const float l = lane < n ? sp.part_ml[slot(b + lane * PARTS) * 2 + 1] : 0.f;
    const float now = fmaxf(top, warp_max(m)), base = now == -INFINITY ? 0.f : now;
    const float old = exp2f(top - base), f = exp2f(m - base);
    top = now;
    sum = fmaf(sum, old, warp_sum(f * l));
#pragma unroll
    for (int c = 0; c < C; ++c) x[c] *= old;
#pragma unroll 8
    for (int i = 0; i < n; ++i) {
      const float w = __shfl_sync(0xffffffffu, f, i);
      const float* src = sp.part_o + slot(b + i * PARTS) * D + C * lane;
#pragma unroll
      for (int c = 0; c < C; c += 2) {
        const float2 y = *reinterpret_cast<const float2*>(src + c);
        x[c] = fmaf(w, y.x, x[c]);
        x[c + 1] = fmaf(w, y.y, x[c + 1]);
      }
    }
  }
  if (PARTS > 1) {
#pragma unroll
    for (int c = 0; c < C; ++c) held[part][in_block][C * lane + c] = x[c];
    if (lane == 0) held_m[warp] = top, held_l[warp] = sum;
    __syncthreads();
    if (part > 0) return;
    float most = top;
#pragma unroll
    for (int o = 1; o < PARTS; ++o) most = fmaxf(most, held_m[o * ROWS + in_block]);
    const float base = most == -INFINITY ? 0.f : most, own = exp2f(top - base);
    sum *= own;
#pragma unroll
    for (int c = 0; c < C; ++c) x[c] *= own;
#pragma unroll
    for (int o = 1; o < PARTS; ++o) {
      const float f = exp2f(held_m[o * ROWS + in_block] - base);
      sum = fmaf(f, held_l[o * ROWS + in_block], sum);
#pragma unroll
      for (int c = 0; c < C; ++c) x[c] = fmaf(f, held[o][in_block][C * lane + c], x[c]);
    }
  }
  const int pr = item.first + row, at = pr / HG, q0 = item.q_start;
  if (row >= item.rows || q0 < 0 || q0 + at >= p.rows) return;
  const float inv = sum > 0.f ? 1.f / sum : sum == 0.f ? 0.f : sum;
  T* dst = (T*)p.out + ((size_t)(q0 + at) * H + item.head + (pr - at * HG)) * D + C * lane;
#pragma unroll
  for (int c = 0; c < C; c += 2) {
    if constexpr (sizeof(T) == 2) *reinterpret_cast<unsigned*>(dst + c) = pack2(x[c] * inv, x[c + 1] * inv);
    else *reinterpret_cast<float2*>(dst + c) = make_float2(x[c] * inv, x[c + 1] * inv);
  }
}

// a kernel's clusters of more than eight blocks, allowed once a device
class WideClusters {
 public:
  template <typename Kernel>
  cudaError_t operator()(Kernel* kernel) {
    int device = 0;
    if (const cudaError_t e = cudaGetDevice(&device)) return e;
    if (device < DEVICES && set_[device].load(std::memory_order_acquire)) return cudaSuccess;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e == cudaSuccess && device < DEVICES) set_[device].store(true, std::memory_order_release);
    return e;
  }

 private:
  static constexpr int DEVICES = 16;
  std::atomic<bool> set_[DEVICES] = {};
};

template <typename T, int D, int NT, int TERMS>
int launch(const Kv4AttnParams& p, const Split& sp, int blocks, int cluster, bool few_items, cudaStream_t stream) {
  constexpr int MT = 8 * NT, ring = WARPS * STAGES * rec_bytes(D), merge = WARPS * MT * (D + 2 + D / GROUP) * 4;
  const size_t lists = (size_t)p.requests * (sizeof(long long) + sizeof(int2) + sizeof(int));
  const size_t smem = (ring > merge ? ring : merge) + lists;
  if (cluster > 0) {
    static OptIn opt_in;
    static WideClusters wide;
    const auto kernel = kv4_attention_kernel<T, D, NT, TERMS, true>;
    if (const cudaError_t e = opt_in(smem + MT * (D + 2) * 4, kernel)) return (int)e;
    if (const cudaError_t e = wide(kernel)) return (int)e;
    launch_k_cluster(kernel, blocks, WARPS * 32, smem + MT * (D + 2) * 4, stream, cluster, p, sp);
    return launch_status();
  }
  static OptIn opt_in;
  if (const cudaError_t e = opt_in(smem, kv4_attention_kernel<T, D, NT, TERMS, false>)) return (int)e;
  launch_k(kv4_attention_kernel<T, D, NT, TERMS, false>, blocks, WARPS * 32, smem, stream, p, sp);
  // few items in many parts (a long context alone in its step): a quarter of an item's rows a block, four times the warps a row
  if (blocks > 1 && few_items) launch_k(kv4_merge_kernel<T, D, MT, MT / 4>, dim3(blocks - 1, 4), MERGE_WARPS * 32, 0, stream, p, sp);
  else if (blocks > 1) launch_k(kv4_merge_kernel<T, D, MT, MT>, blocks - 1, MERGE_WARPS * 32, 0, stream, p, sp);
  return launch_status();
}

}  // namespace

// cluster 0: the tiles are shared evenly; workspace: 8 floats a block, then 2 blocks * tile rows * (head_dim + 2).  cluster 1 to
// 16: that many blocks an item at a time (blocks a multiple of it), no workspace.  tile_rows: 8, or 16 (bfloat16); requests of
// more than most_packed packed rows are left out.
PBE_EXPORT int pbe_kv4_attention(const Kv4AttnParams* params, float* workspace, int blocks, int head_dim, int tile_rows,
                                 int cluster, int most_packed, int dtype, cudaStream_t stream) {
  const Kv4AttnParams p = *params;
  if (p.requests <= 0 || p.rows <= 0) return 0;
  if (p.requests > MOST_REQUESTS || blocks < 1 || (head_dim != 64 && head_dim != 128) ||
      !(tile_rows == 8 || (tile_rows == 16 && dtype == PBE_BF16)) || cluster < 0 || cluster > 16 || (cluster > 0 && blocks % cluster) ||
      (cluster == 0 && workspace == nullptr))
    return (int)cudaErrorInvalidValue;
  Split sp;
  sp.shared = reinterpret_cast<Shared*>(workspace);
  sp.part_o = workspace + (size_t)blocks * (sizeof(Shared) / sizeof(float));
  sp.part_ml = sp.part_o + (size_t)2 * blocks * tile_rows * head_dim;
  sp.most_packed = most_packed;
  const bool few_items = (long long)p.requests * p.kv_heads * 8 <= blocks;
  auto go = [&](auto d64, auto d128) { return (head_dim == 64 ? d64 : d128)(p, sp, blocks, cluster, few_items, stream); };
  typedef __nv_bfloat16 B;
  if (dtype == PBE_F32) return go(launch<float, 64, 1, 3>, launch<float, 128, 1, 3>);
  return tile_rows == 8 ? go(launch<B, 64, 1, 1>, launch<B, 128, 1, 1>) : go(launch<B, 64, 2, 1>, launch<B, 128, 2, 1>);
}
