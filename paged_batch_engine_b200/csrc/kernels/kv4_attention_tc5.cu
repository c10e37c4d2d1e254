// Causal attention over 4-bit pages (kv4.cuh) for prompt portions, on the fifth-generation tensor cores.
//
// One block owns a row tile of 128 packed rows (query row x head of the group) of one key/value head and walks over its keys in
// tiles of 64, four records:
//   S = Q K^T     tcgen05.mma, 128 x 64 x D, into two alternating score buffers in tensor memory;
//   softmax       warps 0-3, one thread a row: tcgen05.ld, maximum, exponentials, sum; the running maximum moves only after it
//                 grew by 2^8, so the output accumulator is rarely rescaled;
//   O += P V      P goes back into the columns of its scores and is the A operand from tensor memory.
// Warps 4-7 turn records into operands, a record of each tile a warp: words are loaded a tile ahead into registers, and
// lo + s * code is one float16 multiply-add a pair of channels, since a code in the low bits of a float16 is already a number
// (code * 2^-24).  Keys become 64 rows of D channels, values D rows of 64 keys (their words hold pairs of keys, so that is
// how they lie), both K-major under the 128-byte swizzle; the rows of the values are ordered (group, i, r), so that eight
// lanes write eight different banks, and the epilogue puts the channels back in order.  Warp 8 issues the products.
//
// All operands are float16, with sums in float32: eleven bits where bfloat16 keeps eight, so the rounding of keys, values and
// weights stays below the output's.  Ranges are kept by exponents: a row's queries, and a record's keys and values, are scaled
// by powers of two that the softmax takes out again (keys in the factor before the exponential, values as an offset within
// it, with a running reference for the output's unit).  Spans of keys and values from 2^-60 to 2^60 are held.
//
// Two blocks share a multiprocessor (256 columns of tensor memory and 100 KB each).  Few row tiles with many keys are split
// along the keys and merged by a second kernel.  Every mbarrier wait is bounded; one that runs out sets *err, and the roles run
// to their end.
#include <cuda.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "kv4.cuh"
#include "kv4_params.cuh"
#include "opt_in.cuh"
#include "pdl.cuh"
#include "tcgen05.cuh"

using namespace pbe;
using namespace pbe::kv4;
using namespace pbe::tc5;

namespace {
constexpr int BM = 128, BN = 64;        // packed rows of a block, keys of a tile
constexpr int RECS = BN / REC_TOKENS;   // records of a tile, one a dequantising warp
constexpr int THREADS = 288;
constexpr int TMEM_COLS = 256;
constexpr int S_COL = 0, O_COL = 128;
constexpr int ROOM = 6;                 // weights are kept 2^6 times too large: float16 reaches further down
constexpr int MOST_E = 60;

struct Tc5Split {
  float* part_o;               // [tiles * KV * splits][128][D]
  float* part_ml;              // [tiles * KV * splits][128][2]: maximum (log2), sum
  int most_packed;             // requests of at most as many packed rows are another kernel's
  int splits;
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float pow2(int e) { return __int_as_float(max(1, min(254, e + 127)) << 23); }
__device__ __forceinline__ unsigned h2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const unsigned*>(&h);
}
__device__ __forceinline__ unsigned hfma(unsigned a, unsigned b, unsigned c) {
  unsigned d;
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}
__device__ __forceinline__ unsigned hmul(unsigned a, unsigned b) {
  unsigned d;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
constexpr unsigned SIXTEENTH = 0x2c002c00u;            // 1/16 twice
// the four pairs of a word: lo + s * code each
__device__ __forceinline__ void four_pairs(unsigned w, unsigned s, unsigned lo, unsigned (&out)[4]) {
  const unsigned s16 = hmul(s, SIXTEENTH);
  out[0] = hfma(w & 0x000f000fu, s, lo);
  out[1] = hfma(w & 0x00f000f0u, s16, lo);
  out[2] = hfma((w >> 8) & 0x000f000fu, s, lo);
  out[3] = hfma((w >> 8) & 0x00f000f0u, s16, lo);
}
// byte offset of 16-byte chunk `chunk` of a 128-byte row under the 128-byte swizzle
__device__ __forceinline__ unsigned swizzled(int row, int chunk) { return (unsigned)(row * 128 + ((chunk ^ (row & 7)) << 4)); }
__device__ __forceinline__ uint32_t idesc_f16(int m, int n) {
  return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

struct Tile {
  int req, row_tile, index;    // index: among all row tiles; req < 0: none
};
// the row tile that a block works on, found by every warp for itself
__device__ __forceinline__ Tile tile_of(const Kv4AttnParams& p, int most_packed, int target) {
  const int lane = threadIdx.x & 31, G = p.heads / p.kv_heads;
  int before = 0;
  for (int r0 = 0; r0 < p.requests; r0 += 32) {
    const int r = r0 + lane;
    int n = 0;
    if (r < p.requests) {
      const long long packed = (long long)max(0, p.q_len[r]) * G;
      n = packed > most_packed ? (int)((packed + BM - 1) / BM) : 0;
    }
    int end = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, end, o);
      if (lane >= o) end += u;
    }
    const int all = __shfl_sync(0xffffffffu, end, 31);
    if (target < before + all) {
      const unsigned past = __ballot_sync(0xffffffffu, before + end > target);
      const int who = __ffs(past) - 1;
      const int n_who = __shfl_sync(0xffffffffu, n, who), end_who = __shfl_sync(0xffffffffu, end, who);
      // the last tiles of a request see the most keys: they come first
      return {r0 + who, before + end_who - 1 - target, target};
    }
    before += all;
  }
  return {-1, 0, target};
}

template <int D>
__global__ void __launch_bounds__(THREADS, 2)
kv4_attention_tc5_kernel(Kv4AttnParams p, Tc5Split sp, int* err) {
  constexpr int G = D / GROUP, REC = rec_bytes(D);
  constexpr int Q_BYTES = BM * D * 2, T_BYTES = BN * D * 2;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* base = reinterpret_cast<unsigned char*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  unsigned char* Qs = base;                            // [D / 64][128 rows][128 B]
  unsigned char* Ks = Qs + Q_BYTES;                    // [2][D / 64][64 keys][128 B]
  unsigned char* Vs = Ks + 2 * T_BYTES;                // [2][D rows][64 keys: 128 B]
  unsigned* nums = reinterpret_cast<unsigned*>(Vs + 2 * T_BYTES);   // [4 warps][keys s, lo: 16 tokens x G; values s, lo: 8 pairs x G]
  __shared__ __align__(8) uint64_t k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2], e_full[4], p_full, o_ready, q_full;
  __shared__ float key_unit[4][RECS];                  // 2^exponent of a record's keys, negative: no key of it is seen
  __shared__ int value_exp[4][RECS];
  __shared__ uint32_t tmem_base_smem;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_wait();
  const int KV = p.kv_heads, H = p.heads, HG = H / KV, per_page = p.page_tokens / REC_TOKENS;
  const int split = blockIdx.x % sp.splits, kvh = blockIdx.x / sp.splits % KV;
  const Tile tile = tile_of(p, sp.most_packed, blockIdx.x / sp.splits / KV);
  if (tile.req < 0) return;
  const int r = tile.req;
  const int nq = p.q_len[r], q0 = p.q_start[r], seq = max(0, p.seq_len[r]);
  const int packed = nq * HG, pr0 = tile.row_tile * BM, rows_here = min(BM, packed - pr0);
  const int pos0 = seq - nq;
  const int pos_min = pos0 + pr0 / HG, pos_max = pos0 + (pr0 + rows_here - 1) / HG;
  const int low_min = p.window > 0 ? max(0, pos_min - p.window + 1) : 0, low_max = p.window > 0 ? pos_max - p.window + 1 : 0;
  const int tile_lo = low_min / BN, tile_hi = pos_max >= 0 ? pos_max / BN + 1 : 0;
  const int all_tiles = max(0, tile_hi - tile_lo);
  const int t_begin = tile_lo + (int)((long long)all_tiles * split / sp.splits);
  const int n_tiles = tile_lo + (int)((long long)all_tiles * (split + 1) / sp.splits) - t_begin;

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&k_full[i], RECS);
      mbar_init(&k_empty[i], 1);
      mbar_init(&v_full[i], RECS);
      mbar_init(&v_empty[i], 1);
      mbar_init(&s_full[i], 1);
    }
    for (int i = 0; i < 4; ++i) mbar_init(&e_full[i], RECS);
    mbar_init(&p_full, 4);
    mbar_init(&o_ready, 1);
    mbar_init(&q_full, 4);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 8) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                 ::"r"(smem_u32(&tmem_base_smem)), "r"(TMEM_COLS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem_base = tmem_base_smem;

  if (warp >= 4 && warp < 8) {
    // ------------------------------------------------------------ records to operands
    const int rec = warp - 4;
    unsigned* kn = nums + rec * (48 * G);              // keys: [16 tokens][G] s twice, then lo twice
    unsigned* vn = kn + 32 * G;                        // values: [8 pairs][G] s, then lo
    const int32_t* table = p.block_table + (long long)r * p.bt_stride;
    auto record = [&](int j) -> long long {            // where tile j's record of this warp lies, -1: nothing to be seen
      const int t = (t_begin + j) * RECS + rec;
      if (j >= n_tiles || t * REC_TOKENS > pos_max || t * REC_TOKENS + REC_TOKENS <= low_min) return -1;
      const int blk = t / per_page;
      const int page = blk < p.table_pages ? table[blk] : -1;
      return page >= 0 && page < p.num_pages ? ((long long)(page * KV + kvh) * per_page + (t - blk * per_page)) * REC : -1;
    };
    // lane's tasks: keys: tokens kt and kt + 8, words j of all groups; values: pairs 4 vc .. 4 vc + 3, r8, half the groups;
    // numbers: four words of one kind and pair
    const int kj = lane & 3, kt = (lane >> 3) + 4 * ((lane >> 2) & 1);
    const int vr = lane & 7, vc = (lane >> 3) & 1, vg = (lane >> 4) * (G / 2);
    const int kind = lane >> 3, np = lane & 7;
    unsigned kw[2][G], vw[4][G / 2], nw[G];
    auto load = [&](long long at) {
      if (at < 0) return;
      const unsigned char* src = p.pages + at;
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        const unsigned char* k = src + (kt + 8 * n) * (D / 2) + kj * (4 * G);
        if constexpr (G == 4) {
          const uint4 x = *reinterpret_cast<const uint4*>(k);
          kw[n][0] = x.x, kw[n][1] = x.y, kw[n][2] = x.z, kw[n][3] = x.w;
        } else {
          const uint2 x = *reinterpret_cast<const uint2*>(k);
          kw[n][0] = x.x, kw[n][1] = x.y;
        }
      }
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        const unsigned char* v = src + v_codes(D) + (4 * vc + n) * D + (vr * G + vg) * 4;
        if constexpr (G == 4) {
          const uint2 x = *reinterpret_cast<const uint2*>(v);
          vw[n][0] = x.x, vw[n][1] = x.y;
        } else {
          vw[n][0] = *reinterpret_cast<const unsigned*>(v);
        }
      }
      const unsigned char* q = src + numbers(D) + kind * D + np * (4 * G);
      if constexpr (G == 4) {
        const uint4 x = *reinterpret_cast<const uint4*>(q);
        nw[0] = x.x, nw[1] = x.y, nw[2] = x.z, nw[3] = x.w;
      } else {
        const uint2 x = *reinterpret_cast<const uint2*>(q);
        nw[0] = x.x, nw[1] = x.y;
      }
    };
    long long at = record(0), at_next = record(1);
    load(at);
    bool ok = true;
    for (int j = 0; j < n_tiles; ++j) {
      const int st = j & 1;
      const bool seen = at >= 0;
      const int key = ((t_begin + j) * RECS + rec) * REC_TOKENS + 2 * np;     // the numbers' two tokens
      // places that hold no key of this row tile may hold anything: their numbers count as zero
      const unsigned keep = !seen ? 0u : (key <= pos_max && key >= low_min ? 0xffffu : 0u) |
                                             (key + 1 <= pos_max && key + 1 >= low_min ? 0xffff0000u : 0u);
      unsigned most = 0;
#pragma unroll
      for (int g = 0; g < G; ++g) {
        nw[g] &= keep;
        most = max(most, max(nw[g] & 0x7fffu, (nw[g] >> 16) & 0x7fffu));
      }
#pragma unroll
      for (int o = 1; o < 8; o <<= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
      // kinds by eights of lanes: lo and s of keys, lo and s of values.  The unit is such that s reaches up to 2^-8 and lo
      // stays within float16
      const int e_own = (int)(most >> 7) - 127, e_other = __shfl_xor_sync(0xffffffffu, e_own, 8);
      const int e_s = kind & 1 ? e_own : e_other, e_lo = kind & 1 ? e_other : e_own;
      const int e = max(-MOST_E, min(MOST_E + 9, max(e_s + 9, e_lo - 14)));
      const float by = pow2((kind & 1 ? 24 : 0) - e);
      unsigned half[G];
#pragma unroll
      for (int g = 0; g < G; ++g)
        half[g] = h2(__uint_as_float(nw[g] << 16) * by, __uint_as_float(nw[g] & 0xffff0000u) * by);
      __syncwarp();                                    // the numbers of the tile before are read
      if (kind < 2) {
        unsigned* dst = kn + (kind == K_S ? 0 : 16 * G) + 2 * np * G;
#pragma unroll
        for (int g = 0; g < G; ++g) {
          dst[g] = __byte_perm(half[g], 0u, 0x1010);
          dst[G + g] = __byte_perm(half[g], 0u, 0x3232);
        }
      } else {
        unsigned* dst = vn + (kind == V_S ? 0 : 8 * G) + np * G;
#pragma unroll
        for (int g = 0; g < G; ++g) dst[g] = half[g];
      }
      if (lane == 0) key_unit[j & 3][rec] = seen ? pow2(e) : -1.f;
      if (lane == 16) value_exp[j & 3][rec] = e;
      __syncwarp();
      if (lane == 0) mbar_arrive(&e_full[j & 3]);
      // ---- keys
      if (lane == 0) ok = ok && mbar_wait(&k_empty[st], ((j >> 1) & 1) ^ 1, err);
      __syncwarp();
      unsigned char* kd = Ks + st * T_BYTES;
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        const int t = kt + 8 * n, row = rec * REC_TOKENS + t;
#pragma unroll
        for (int g = 0; g < G; ++g) {
          unsigned x[4] = {};
          if (seen) four_pairs(kw[n][g], kn[t * G + g], kn[16 * G + t * G + g], x);
          *reinterpret_cast<uint4*>(kd + (g >> 1) * (BN * 128) + swizzled(row, 4 * (g & 1) + kj)) = make_uint4(x[0], x[1], x[2], x[3]);
        }
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&k_full[st]);
        ok = ok && mbar_wait(&v_empty[st], ((j >> 1) & 1) ^ 1, err);
      }
      __syncwarp();
      // ---- values
      unsigned char* vd = Vs + st * T_BYTES;
#pragma unroll
      for (int g = 0; g < G / 2; ++g) {
        unsigned x[4][4] = {};                         // [pair][i]
        if (seen) {
#pragma unroll
          for (int n = 0; n < 4; ++n) four_pairs(vw[n][g], vn[(4 * vc + n) * G + vg + g], vn[8 * G + (4 * vc + n) * G + vg + g], x[n]);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
          *reinterpret_cast<uint4*>(vd + swizzled(32 * (vg + g) + 8 * i + vr, 2 * rec + vc)) = make_uint4(x[0][i], x[1][i], x[2][i], x[3][i]);
      }
      at = at_next;
      load(at);                                        // the next tile's words, while this one is multiplied
      at_next = record(j + 2);
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(&v_full[st]);
    }
    // the commits that release the last tiles arrive whenever the tensor core gets there: not after the block is gone
    if (lane == 0) {
      for (int j = max(0, n_tiles - 2); j < n_tiles && ok; ++j) {
        ok = mbar_wait(&k_empty[j & 1], (j >> 1) & 1, err);
        ok = ok && mbar_wait(&v_empty[j & 1], (j >> 1) & 1, err);
      }
    }
  } else if (warp == 8) {
    if (lane == 0 && n_tiles > 0) {
      // ------------------------------------------------------------ MMA issuer
      const uint32_t idesc_s = idesc_f16(BM, BN), idesc_o = idesc_f16(BM, D);
      const uint32_t q_addr = smem_u32(Qs);
      bool ok = true;
      auto issue_qk = [&](int j) {
        const int st = j & 1;
        ok = ok && mbar_wait(&k_full[st], (j >> 1) & 1, err);
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint32_t k_addr = smem_u32(Ks + st * T_BYTES);
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks)
          umma(tmem_base + S_COL + st * BN, make_desc(q_addr + (ks >> 2) * (BM * 128) + (ks & 3) * 32),
               make_desc(k_addr + (ks >> 2) * (BN * 128) + (ks & 3) * 32), idesc_s, ks > 0 ? 1u : 0u);
        umma_commit(&k_empty[st]);
        umma_commit(&s_full[st]);
      };
      ok = ok && mbar_wait(&q_full, 0, err);
      issue_qk(0);
      if (n_tiles > 1) issue_qk(1);
      for (int j = 0; j < n_tiles && ok; ++j) {
        const int st = j & 1;
        ok = ok && mbar_wait(&v_full[st], (j >> 1) & 1, err);
        ok = ok && mbar_wait(&p_full, j & 1, err);     // P_j written, O rescaled
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint32_t v_addr = smem_u32(Vs + st * T_BYTES);
#pragma unroll
        for (int ks = 0; ks < BN / 16; ++ks)
          umma_ts(tmem_base + O_COL, tmem_base + S_COL + st * BN + ks * 8, make_desc(v_addr + ks * 32), idesc_o,
                  (j > 0 || ks > 0) ? 1u : 0u);
        umma_commit(&v_empty[st]);
        umma_commit(&o_ready);
        if (j + 2 < n_tiles) issue_qk(j + 2);          // into the buffer that P_j has left: the tensor pipe runs in order
      }
    }
  } else {
    // ---------------------------------------------------------------- softmax, correction, epilogue
    const int row = warp * 32 + lane, pr = pr0 + row;
    const bool row_valid = row < rows_here;
    const int q_row = row_valid ? pr / HG : 0, head = kvh * HG + (row_valid ? pr - q_row * HG : 0);
    const bool held = row_valid && q0 >= 0 && q0 + q_row < p.rows;
    const int pos = row_valid ? pos0 + q_row : -1;
    const int lo = p.window > 0 ? pos - p.window + 1 : 0;
    // ---- the row's queries as float16, scaled by a power of two so that the largest lies in [1, 2)
    float row_unit;
    {
      const __nv_bfloat16* src = (const __nv_bfloat16*)p.q + ((size_t)(held ? q0 + q_row : 0) * H + head) * D;
      uint4 w[D / 8];
      unsigned most = 0;
#pragma unroll
      for (int c = 0; c < D / 8; ++c) {
        w[c] = held ? *reinterpret_cast<const uint4*>(src + c * 8) : make_uint4(0, 0, 0, 0);
        most = max(most, max(max(w[c].x & 0x7fffu, (w[c].x >> 16) & 0x7fffu), max(w[c].y & 0x7fffu, (w[c].y >> 16) & 0x7fffu)));
        most = max(most, max(max(w[c].z & 0x7fffu, (w[c].z >> 16) & 0x7fffu), max(w[c].w & 0x7fffu, (w[c].w >> 16) & 0x7fffu)));
      }
      const int e = max(-MOST_E, min(MOST_E, (int)(most >> 7) - 127));
      const float by = pow2(-e);
      row_unit = pow2(e) * p.scale * 1.4426950408889634f;
#pragma unroll
      for (int c = 0; c < D / 8; ++c) {
        const unsigned u[4] = {w[c].x, w[c].y, w[c].z, w[c].w};
        unsigned x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = h2(__uint_as_float(u[i] << 16) * by, __uint_as_float(u[i] & 0xffff0000u) * by);
        *reinterpret_cast<uint4*>(Qs + (c >> 3) * (BM * 128) + swizzled(row, c & 7)) = make_uint4(x[0], x[1], x[2], x[3]);
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(&q_full);
    }
    const uint32_t lane_addr = tmem_base + ((uint32_t)(warp * 32) << 16);
    float m_run = -INFINITY, l_run = 0.f;              // maximum in units of log2
    int e_run = -2 * MOST_E;                           // the output's unit: 2^(e_run - ROOM + m_run)
    bool ok = true;
    for (int j = 0; j < n_tiles; ++j) {
      const int st = j & 1, ts = (t_begin + j) * BN;
      ok = ok && mbar_wait(&s_full[st], (j >> 1) & 1, err);
      ok = ok && mbar_wait(&e_full[j & 3], (j >> 2) & 1, err);
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      float s[BN];
#pragma unroll
      for (int c = 0; c < BN / 32; ++c) tmem_ld32_nowait(lane_addr + S_COL + st * BN + c * 32, &s[c * 32]);
      float unit[RECS];
      int ev[RECS];
      bool whole = ts + BN - 1 <= pos_min && ts >= low_max;
#pragma unroll
      for (int g = 0; g < RECS; ++g) {
        unit[g] = key_unit[j & 3][g] * row_unit;
        ev[g] = value_exp[j & 3][g];
        whole = whole && key_unit[j & 3][g] > 0.f;
      }
      asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
      if (!whole) {
#pragma unroll
        for (int i = 0; i < BN; ++i) {
          const int key = ts + i;
          if (key > pos || key < lo || !(key_unit[j & 3][i / REC_TOKENS] > 0.f)) s[i] = -INFINITY;
        }
#pragma unroll
        for (int g = 0; g < RECS; ++g) unit[g] = fabsf(unit[g]);
      }
      float mx = -INFINITY;
#pragma unroll
      for (int g = 0; g < RECS; ++g) {
        float a = s[g * 16], b = s[g * 16 + 1];
#pragma unroll
        for (int i = 2; i < 16; i += 2) {
          a = fmaxf(a, s[g * 16 + i]);
          b = fmaxf(b, s[g * 16 + i + 1]);
        }
        mx = fmaxf(mx, fmaxf(a, b) * unit[g]);
      }
      // the maximum moves only when it has grown by more than 2^8; the values' unit when a larger one comes
      const int e_new = max(e_run, max(max(ev[0], ev[1]), max(ev[2], ev[3])));
      float m_new = fmaxf(m_run, mx);
      if (m_run != -INFINITY && m_new - m_run <= 8.0f) m_new = m_run;
      const float m_use = m_new == -INFINITY ? 0.f : m_new;
      const float shrink = ex2(m_run - m_use), alpha = shrink * ex2((float)(e_run - e_new));
      float sum = 0.f;
#pragma unroll
      for (int g = 0; g < RECS; ++g) {
        const float off = (float)(ROOM + ev[g] - e_new) - m_use;
        float a = 0.f, b = 0.f;
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
          s[g * 16 + i] = ex2(fmaf(s[g * 16 + i], unit[g], off));
          s[g * 16 + i + 1] = ex2(fmaf(s[g * 16 + i + 1], unit[g], off));
          a += s[g * 16 + i];
          b += s[g * 16 + i + 1];
        }
        sum = fmaf(a + b, ex2((float)min(e_new - ev[g], 126)), sum);
      }
      l_run = fmaf(l_run, shrink, sum);
      {
        uint32_t w[BN / 2];
#pragma unroll
        for (int i = 0; i < BN / 2; ++i) w[i] = h2(s[2 * i], s[2 * i + 1]);
        tmem_st32_nowait(lane_addr + S_COL + st * BN, &w[0]);
      }
      if (j > 0) {
        ok = ok && mbar_wait(&o_ready, (j - 1) & 1, err);
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        if (__any_sync(0xffffffffu, m_new > m_run || e_new > e_run)) {
#pragma unroll
          for (int c = 0; c < D / 32; ++c) {
            float v[32];
            tmem_ld32(lane_addr + O_COL + c * 32, v);
            uint32_t w[32];
#pragma unroll
            for (int i = 0; i < 32; ++i) w[i] = __float_as_uint(v[i] * alpha);
            tmem_st32_nowait(lane_addr + O_COL + c * 32, w);
          }
        }
      }
      m_run = m_new;
      e_run = e_new;
      asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full);
    }
    pdl_launch_dependents();
    if (n_tiles > 0) {
      ok = ok && mbar_wait(&o_ready, (n_tiles - 1) & 1, err);
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    }
    // l is in units of 2^(m_run - ROOM), the output in units of 2^e_run more
    const float back = n_tiles > 0 ? pow2(e_run) : 0.f;
    const float inv = sp.splits > 1 ? back : l_run > 0.f ? back / l_run : l_run == 0.f ? 0.f : l_run;
    const size_t part = ((size_t)tile.index * KV + kvh) * sp.splits + split;
#pragma unroll
    for (int g = 0; g < G; ++g) {
      float v[32];
      if (n_tiles > 0) {                               // block-uniform: every lane takes part in the load
        tmem_ld32(lane_addr + O_COL + g * 32, v);
      } else {
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = 0.f;
      }
      // column 8 i + r is channel 4 r + i
      if (held && sp.splits == 1) {
        __nv_bfloat16* dst = (__nv_bfloat16*)p.out + ((size_t)(q0 + q_row) * H + head) * D + g * 32;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          unsigned w[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int r8 = 2 * c + (k >> 1), i = 2 * (k & 1);
            const __nv_bfloat162 h = __floats2bfloat162_rn(v[8 * i + r8] * inv, v[8 * (i + 1) + r8] * inv);
            w[k] = *reinterpret_cast<const unsigned*>(&h);
          }
          reinterpret_cast<uint4*>(dst)[c] = make_uint4(w[0], w[1], w[2], w[3]);
        }
      } else if (held) {
        float* dst = sp.part_o + (part * BM + row) * D + g * 32;
#pragma unroll
        for (int r8 = 0; r8 < 8; ++r8)
          reinterpret_cast<float4*>(dst)[r8] = make_float4(v[r8] * inv, v[8 + r8] * inv, v[16 + r8] * inv, v[24 + r8] * inv);
        if (g == 0) {
          sp.part_ml[(part * BM + row) * 2] = m_run;
          sp.part_ml[(part * BM + row) * 2 + 1] = l_run;
        }
      }
      __syncwarp();
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  }
  __syncthreads();
  if (warp == 8) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(TMEM_COLS) : "memory");
  }
}

// The splits of a row tile and key/value head merged, a warp a row.
template <int D>
__global__ void __launch_bounds__(256) kv4_tc5_merge_kernel(Kv4AttnParams p, Tc5Split sp) {
  constexpr int C = D / 32;
  pdl_launch_dependents();
  pdl_wait();
  const int KV = p.kv_heads, H = p.heads, HG = H / KV, kvh = blockIdx.x % KV;
  const Tile tile = tile_of(p, sp.most_packed, blockIdx.x / KV);
  if (tile.req < 0) return;
  const int packed = p.q_len[tile.req] * HG, q0 = p.q_start[tile.req], lane = threadIdx.x & 31;
  for (int row = blockIdx.y * 8 + (threadIdx.x >> 5); row < BM; row += gridDim.y * 8) {
    const int pr = tile.row_tile * BM + row, q_row = pr / HG;
    if (pr >= packed || q0 < 0 || q0 + q_row >= p.rows) return;
    const size_t part0 = ((size_t)tile.index * KV + kvh) * sp.splits;
    float top = -INFINITY;
    for (int s = 0; s < sp.splits; ++s) top = fmaxf(top, sp.part_ml[((part0 + s) * BM + row) * 2]);
    const float base = top == -INFINITY ? 0.f : top;
    float sum = 0.f, x[C] = {};
#pragma unroll 4
    for (int s = 0; s < sp.splits; ++s) {
      const size_t at = (part0 + s) * BM + row;
      const float f = exp2f(sp.part_ml[at * 2] - base);
      sum = fmaf(f, sp.part_ml[at * 2 + 1], sum);
#pragma unroll
      for (int c = 0; c < C; c += 2) {
        const float2 y = *reinterpret_cast<const float2*>(sp.part_o + at * D + C * lane + c);
        x[c] = fmaf(f, y.x, x[c]);
        x[c + 1] = fmaf(f, y.y, x[c + 1]);
      }
    }
    const float inv = sum > 0.f ? 1.f / sum : sum == 0.f ? 0.f : sum;
    __nv_bfloat16* dst = (__nv_bfloat16*)p.out + ((size_t)(q0 + q_row) * H + kvh * HG + (pr - q_row * HG)) * D + C * lane;
#pragma unroll
    for (int c = 0; c < C; c += 2) *reinterpret_cast<__nv_bfloat162*>(dst + c) = __floats2bfloat162_rn(x[c] * inv, x[c + 1] * inv);
  }
}

template <int D>
int launch(const Kv4AttnParams& p, const Tc5Split& sp, int tiles, int* err, cudaStream_t stream) {
  const size_t smem = (size_t)BM * D * 2 + 4 * (size_t)BN * D * 2 + RECS * 48 * (D / GROUP) * 4 + 1024;
  static OptIn opt_in;
  if (const cudaError_t e = opt_in(smem, kv4_attention_tc5_kernel<D>)) return (int)e;
  launch_k(kv4_attention_tc5_kernel<D>, (unsigned)(tiles * p.kv_heads * sp.splits), THREADS, smem, stream, p, sp, err);
  if (sp.splits > 1) launch_k(kv4_tc5_merge_kernel<D>, dim3(tiles * p.kv_heads, 4), 256, 0, stream, p, sp);
  return launch_status();
}
}  // namespace

// Requests of more than most_packed packed rows.  tiles: row tiles of 128 packed rows, at least as many as there are.
// workspace (splits > 1): tiles * kv_heads * splits * 128 * (head_dim + 2) floats.
PBE_EXPORT int pbe_kv4_attention_tc5(const Kv4AttnParams* params, float* workspace, int tiles, int splits, int head_dim,
                                     int most_packed, int* err, cudaStream_t stream) {
  const Kv4AttnParams p = *params;
  if (p.requests <= 0 || p.rows <= 0 || tiles <= 0) return 0;
  if ((head_dim != 64 && head_dim != 128) || splits < 1 || !(p.scale > 0.f) || (long long)tiles * p.kv_heads * splits > 0x7fffffffLL)
    return (int)cudaErrorInvalidValue;
  Tc5Split sp;
  sp.part_o = workspace;
  sp.part_ml = workspace + (size_t)tiles * p.kv_heads * splits * BM * head_dim;
  sp.most_packed = most_packed;
  sp.splits = splits;
  return head_dim == 64 ? launch<64>(p, sp, tiles, err, stream) : launch<128>(p, sp, tiles, err, stream);
}
