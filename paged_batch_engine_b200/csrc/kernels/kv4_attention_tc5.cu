// Causal attention over 4-bit pages (kv4.cuh) for prompt portions, on the fifth-generation tensor cores.
//
// One block owns a row tile of 256 packed rows (query row x head of the group) of one key/value head, two halves of 128, and
// walks over its keys in tiles of 64, four records, which both halves read once they are operands:
//   S = Q K^T     tcgen05.mma, 128 x 64 x D, into two alternating score buffers in tensor memory for each half;
//   softmax       warps 0-3 and 4-7, one thread a row: tcgen05.ld, maximum, exponentials, sum; weights are made against the
//                 maximum so far, which moves only when they grow too large for it, so the output is rarely rescaled, and only
//                 then waited for;
//   O += P V      P goes back into the columns of its scores and is the A operand from tensor memory.
// Warps 8-13 turn records into operands, record after record in turn: a record's words are loaded into registers while the
// one before is converted, and lo + s * code is one float16 multiply-add a pair of channels, since a code in the low bits of
// a float16 is already a number (code * 2^-24).  Keys become 64 rows of D channels, values D rows of 64 keys (their words
// hold pairs of keys, so that is how they lie), both K-major under the 128-byte swizzle, four tiles of each in flight; the
// rows of the values are ordered (group, i, r), so that eight lanes write eight different banks, and the epilogue puts the
// channels back in order.  Warps 14 and 15 issue the products, each those of its half.
//
// 4,096 tokens of 28 heads on 4 of 128: 187 us, 643 TFLOP/s (0.39 of the library products' rate; floor 72).  A tile of 256 x 64
// takes some 2,840 clocks, of which its products need 1,024 and its 16,384 exponentials 1,024 of the SM's sixteen a clock: no
// pipe is busy for two fifths of the time.  What is long is each softmax thread's chain (wait, load, multiply-add, exponential,
// rounding, store, fence), with two warps a scheduler to hide it; attention_tc5.cu, two blocks a multiprocessor, takes 1,750 for
// the same exponentials.  512 threads leave 128 registers each, and some spill (head size 128: 92 bytes stored and 244 loaded, 64: 64
// and 188).  With one half a block and two blocks a multiprocessor each
// record was converted twice as often, and four converting warps were what the rest waited for: 269 us; with key tiles of 128
// and one score buffer a half: 286.
//
// All operands are float16, with sums in float32: eleven bits where bfloat16 keeps eight, so the rounding of keys, values and
// weights stays below the output's.  Ranges are kept by exponents: a row's queries, and a record's keys and values, are scaled
// by powers of two that the softmax takes out again (keys in the factor before the exponential, values as an offset within
// it, with a running reference for the output's unit).  Spans of keys and values from 2^-60 to 2^60 are held.  The reference is a
// row's own, made of what it sees, and a record whose tokens lie far apart has units for each (weigh_one_by_one), so no token
// that a row does not see takes its bits.  A value whose span is 2^-20 of the largest that the row sees has its weight in eleven
// bits; below that it loses them, and counts for nothing from 2^-31 on.
//
// A block takes all of tensor memory (two halves of two score buffers of 64 columns and an output of up to 128).  Few row
// tiles with many keys are split along the keys and merged by a second kernel.  Every mbarrier wait is bounded; one that runs
// out sets *err, and the roles run to their end.
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
constexpr int HALF = 128, BM = 2 * HALF, BN = 64;     // packed rows of a block, keys of a tile
constexpr int RECS = BN / REC_TOKENS;   // records of a tile
constexpr int SOFT = 8, CONV = 6, MMA_WARP = SOFT + CONV;    // and one issuing warp a half
constexpr int THREADS = 32 * (MMA_WARP + 2);
constexpr int STAGES = 4;               // tiles of keys and of values that are operands
constexpr int TMEM_COLS = 512;
constexpr int S_COL = 0, O_COL = 256;   // of half h: two score buffers at 128 h, the output at 256 + 128 h
constexpr int ROOM = 6;                 // weights are kept 2^6 times too large: float16 reaches further down
constexpr int MOST_E = 60;
constexpr float FAR = 16384.f;          // beyond this maximum weights are made one by one: its rounding in float32 is 2^-11
constexpr int NOTHING = -(1 << 20);     // the exponent of a token whose numbers are all zero
constexpr int EVEN = 8, UNEVEN = 1024;  // exponents that the tokens of a record may lie apart and share a unit; the mark of others

struct Tc5Split {
  float* part_o;               // [tiles * KV * splits][256][D]
  float* part_ml;              // [tiles * KV * splits][256][2]: maximum (log2), sum
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
// two float32 operations an instruction
struct f32x2 {
  unsigned long long v;
};
__device__ __forceinline__ f32x2 both(float a, float b) {
  f32x2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void apart(f32x2 x, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(x.v)); }
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
  f32x2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
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

// The products' instructions, executed by a whole warp and issued by one elected lane of it.  Code that all lanes run alike
// keeps descriptors and addresses in uniform registers, where the instruction takes them from; issued from a branch of one
// lane, each product waited some 100 cycles for them to be moved there, three times what the tensor core takes for it.
__device__ __forceinline__ void mma_elected(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n.reg .pred p, q;\nelect.sync _|q, 0xffffffff;\nsetp.ne.b32 p, %4, 0;\n"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n"
      ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void mma_ts_elected(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n.reg .pred p, q;\nelect.sync _|q, 0xffffffff;\nsetp.ne.b32 p, %4, 0;\n"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n"
      ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void commit_elected(uint64_t* bar) {
  asm volatile(
      "{\n.reg .pred q;\nelect.sync _|q, 0xffffffff;\n"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}\n" ::"r"(smem_u32(bar)) : "memory");
}

// the wait for loads from tensor memory, which these registers' uses stay behind
__device__ __forceinline__ void tmem_landed(float (&x)[BN]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+f"(x[0]), "+f"(x[1]), "+f"(x[2]), "+f"(x[3]), "+f"(x[4]), "+f"(x[5]), "+f"(x[6]), "+f"(x[7]),
                 "+f"(x[8]), "+f"(x[9]), "+f"(x[10]), "+f"(x[11]), "+f"(x[12]), "+f"(x[13]), "+f"(x[14]), "+f"(x[15]),
                 "+f"(x[16]), "+f"(x[17]), "+f"(x[18]), "+f"(x[19]), "+f"(x[20]), "+f"(x[21]), "+f"(x[22]),
                 "+f"(x[23]), "+f"(x[24]), "+f"(x[25]), "+f"(x[26]), "+f"(x[27]), "+f"(x[28]), "+f"(x[29]),
                 "+f"(x[30]), "+f"(x[31])
               :: "memory");
  asm volatile(""
               : "+f"(x[32]), "+f"(x[33]), "+f"(x[34]), "+f"(x[35]), "+f"(x[36]), "+f"(x[37]), "+f"(x[38]), "+f"(x[39]),
                 "+f"(x[40]), "+f"(x[41]), "+f"(x[42]), "+f"(x[43]), "+f"(x[44]), "+f"(x[45]), "+f"(x[46]),
                 "+f"(x[47]), "+f"(x[48]), "+f"(x[49]), "+f"(x[50]), "+f"(x[51]), "+f"(x[52]), "+f"(x[53]),
                 "+f"(x[54]), "+f"(x[55]), "+f"(x[56]), "+f"(x[57]), "+f"(x[58]), "+f"(x[59]), "+f"(x[60]),
                 "+f"(x[61]), "+f"(x[62]), "+f"(x[63]));
}

struct Tile {
  int req, row_tile, index;    // index: among all row tiles; req < 0: none
  int rows, start, seq;        // the request's
};
// the row tile that a block works on, found by every warp for itself
__device__ __forceinline__ Tile tile_of(const Kv4AttnParams& p, int most_packed, int target) {
  const int lane = threadIdx.x & 31, G = p.heads / p.kv_heads;
  int before = 0;
  for (int r0 = 0; r0 < p.requests; r0 += 32) {
    const int r = r0 + lane;
    int n = 0, rows = 0, start = 0, seq = 0;
    if (r < p.requests) {
      rows = max(0, p.q_len[r]);
      start = p.q_start[r];
      seq = max(0, p.seq_len[r]);
      const long long packed = (long long)rows * G;
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
      return {r0 + who, before + end_who - 1 - target, target, __shfl_sync(0xffffffffu, rows, who),
              __shfl_sync(0xffffffffu, start, who), __shfl_sync(0xffffffffu, seq, who)};
    }
    before += all;
  }
  return {-1, 0, target, 0, 0, 0};
}

__device__ __forceinline__ void tmem_st8_nowait(uint32_t taddr, const uint32_t (&v)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};"
               ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]) : "memory");
}
// what a tile's operands count in
struct alignas(16) Units {
  float key[RECS];             // 2^exponent of a record's keys, negative: no key of it is seen
  int value[RECS];             // exponent of its values, and UNEVEN more where its tokens have units of their own:
  float key_of[BN], value_of[BN];
};

// A row's weights of one tile, one by one: for tiles with uneven records, and for rows whose scores are so far from zero that the
// exponents cannot be added to the maximum.  The same steps as in the kernel's loop below, out of its way and its registers.
// clear: the row sees every place of the tile that holds a key.
struct Weighed {
  float m, shrink, alpha, sum;
  int e;
};
__device__ __noinline__ Weighed weigh_one_by_one(const Units* u, uint32_t s_addr, int ts, int lo, int pos, bool clear, float row_unit, float m_run, int e_run) {
  float s[REC_TOKENS], mx = -INFINITY, most = 0.f;     // most: 2^exponent of the largest values that the row sees
  // units of four tokens, from memory that may hold anything where the record has one (no branch: the loads go ahead together)
  auto four = [](bool own, const float* from, float one, float (&to)[4]) {
    const float4 x = *reinterpret_cast<const float4*>(from);
    to[0] = own ? x.x : one, to[1] = own ? x.y : one, to[2] = own ? x.z : one, to[3] = own ? x.w : one;
  };
  auto scores = [&](int g) {
    const bool own = u->value[g] >= UNEVEN / 2;
    const float key = u->key[g];
    const int at = ts + g * REC_TOKENS;
    tmem_ld16(s_addr + g * REC_TOKENS, s);
#pragma unroll
    for (int c = 0; c < REC_TOKENS; c += 4) {
      float kf[4];
      four(own, u->key_of + g * REC_TOKENS + c, key, kf);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bool see = (clear || (at + c + i <= pos && at + c + i >= lo)) && key > 0.f;
        s[c + i] = see ? s[c + i] * (kf[i] * row_unit) : -INFINITY;
      }
    }
    return own;
  };
#pragma unroll 1
  for (int g = 0; g < RECS; ++g) {
    const bool own = scores(g);
    const float value = pow2(u->value[g]);
#pragma unroll
    for (int c = 0; c < REC_TOKENS; c += 4) {
      float vf[4];
      four(own, u->value_of + g * REC_TOKENS + c, value, vf);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        mx = fmaxf(mx, s[c + i]);
        most = fmaxf(most, s[c + i] != -INFINITY ? vf[i] : 0.f);
      }
    }
  }
  const int e_new = max(e_run, (__float_as_int(most) >> 23) - 127);
  float m_new = fmaxf(m_run, mx);
  if (m_run != -INFINITY && m_new - m_run <= 8.0f) m_new = m_run;
  const float m_use = m_new == -INFINITY ? 0.f : m_new, down = pow2(-e_new);
  float sum = 0.f;
#pragma unroll 1
  for (int g = 0; g < RECS; ++g) {                     // a record's weights take the place of scores that have been read
    const bool own = scores(g);
    const float value = pow2(u->value[g]);
    uint32_t w[REC_TOKENS / 2];
#pragma unroll
    for (int c = 0; c < REC_TOKENS; c += 4) {
      float vf[4];
      four(own, u->value_of + g * REC_TOKENS + c, value, vf);
#pragma unroll
      for (int i = 0; i < 4; i += 2) {
        const float x = ex2(s[c + i] - m_use + ROOM), y = ex2(s[c + i + 1] - m_use + ROOM);
        sum += x + y;
        w[(c + i) / 2] = h2(x * down * vf[i], y * down * vf[i + 1]);
      }
    }
    tmem_st8_nowait(s_addr + g * (REC_TOKENS / 2), w);
  }
  const float shrink = ex2(m_run - m_use);
  return {m_new, shrink, shrink * ex2((float)(e_run - e_new)), sum, e_new};
}

// N words from shared memory, as wide as they come
template <int N>
__device__ __forceinline__ void words(unsigned (&w)[N], const unsigned* p) {
  if constexpr (N == 4) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
  } else if constexpr (N == 2) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    w[0] = v.x, w[1] = v.y;
  } else {
    w[0] = *p;
  }
}

template <int D>
__global__ void __launch_bounds__(THREADS, 1)
kv4_attention_tc5_kernel(Kv4AttnParams p, Tc5Split sp, int* err) {
  constexpr int G = D / GROUP, REC = rec_bytes(D);
  constexpr int Q_BYTES = BM * D * 2, T_BYTES = BN * D * 2;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* base = reinterpret_cast<unsigned char*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  unsigned char* Qs = base;                            // [2 halves][D / 64][128 rows][128 B]
  unsigned char* Ks = Qs + Q_BYTES;                    // [STAGES][D / 64][64 keys][128 B]
  unsigned char* Vs = Ks + STAGES * T_BYTES;           // [STAGES][D rows][64 keys: 128 B]
  unsigned* nums = reinterpret_cast<unsigned*>(Vs + STAGES * T_BYTES);   // [CONV][keys s, lo: 16 tokens x G; values s, lo: 8 pairs x G]
  __shared__ __align__(8) uint64_t full[STAGES], empty[STAGES], s_full[2][2], p_full[2][2], o_ready[2], o_done[2], q_full[2];
  __shared__ Units units[STAGES];
  __shared__ uint32_t tmem_base_smem;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_wait();
  const int KV = p.kv_heads, H = p.heads, HG = H / KV, per_page = p.page_tokens / REC_TOKENS;
  const int split = blockIdx.x % sp.splits, kvh = blockIdx.x / sp.splits % KV;
  const Tile tile = tile_of(p, sp.most_packed, blockIdx.x / sp.splits / KV);
  if (tile.req < 0) return;
  const int r = tile.req;
  const int nq = tile.rows, q0 = tile.start, seq = tile.seq;
  const int packed = nq * HG, pr0 = tile.row_tile * BM, rows_here = min(BM, packed - pr0);
  const int pos0 = seq - nq;
  const int pos_min = pos0 + pr0 / HG, pos_max = pos0 + (pr0 + rows_here - 1) / HG;
  // (rows before the first key see none; a window of 2^31 - 1 taken from their positions would not fit an int)
  const int low_min = p.window > 0 ? max(0, max(0, pos_min) - p.window + 1) : 0, low_max = p.window > 0 ? max(0, pos_max) - p.window + 1 : 0;
  const int tile_lo = low_min / BN, tile_hi = pos_max >= 0 ? pos_max / BN + 1 : 0;
  const int all_tiles = max(0, tile_hi - tile_lo);
  const int t_begin = tile_lo + (int)((long long)all_tiles * split / sp.splits);
  const int n_tiles = tile_lo + (int)((long long)all_tiles * (split + 1) / sp.splits) - t_begin;

  const int halves = rows_here > HALF ? 2 : 1;
  if (threadIdx.x == 0) {
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(&full[i], RECS);
      mbar_init(&empty[i], halves);
    }
    for (int h = 0; h < 2; ++h) {
      mbar_init(&s_full[h][0], 1);
      mbar_init(&s_full[h][1], 1);
      mbar_init(&p_full[h][0], 4);
      mbar_init(&p_full[h][1], 4);
      mbar_init(&o_ready[h], 1);
      mbar_init(&o_done[h], 1);
      mbar_init(&q_full[h], 4);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == MMA_WARP) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                 ::"r"(smem_u32(&tmem_base_smem)), "r"(TMEM_COLS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem_base = tmem_base_smem;

  if (warp >= SOFT && warp < MMA_WARP) {
    // ------------------------------------------------------------ records to operands
    // records q = 4 tile + r of the block's tiles, q = own, own + CONV, ...
    const int own = warp - SOFT, records = n_tiles * RECS;
    unsigned* kn = nums + own * (48 * G);              // keys: [16 tokens][G] s twice, then lo twice
    unsigned* vn = kn + 32 * G;                        // values: [8 pairs][G] s, then lo
    const int32_t* table = p.block_table + (long long)r * p.bt_stride;
    const int page_shift = (per_page & (per_page - 1)) == 0 ? 31 - __clz(per_page) : -1;
    auto page_of = [&](int n) {                        // the page of record n, -1: nothing to be seen
      const int t = t_begin * RECS + n;
      if (n >= records || t * REC_TOKENS > pos_max || t * REC_TOKENS + REC_TOKENS <= low_min) return -1;
      const int blk = page_shift >= 0 ? t >> page_shift : t / per_page;
      return blk < p.table_pages ? table[blk] : -1;
    };
    auto record = [&](int n, int page) -> long long {  // and where it lies
      const int t = t_begin * RECS + n, in_page = page_shift >= 0 ? t & (per_page - 1) : t % per_page;
      return page >= 0 && page < p.num_pages ? ((long long)(page * KV + kvh) * per_page + in_page) * REC : -1;
    };
    // lane's tasks: keys: tokens kt and kt + 8, words j of all groups; values: pairs 4 vc .. 4 vc + 3, r8, half the groups;
    // numbers: four words of one kind and pair
    const int kj = lane & 3, kt = (lane >> 3) + 4 * ((lane >> 2) & 1);
    const int vr = lane & 7, vc = (lane >> 3) & 1, vg = (lane >> 4) * (G / 2);
    const int kind = lane >> 3, np = lane & 7;
    const unsigned k_chunk[2] = {(unsigned)((kj ^ kt) << 4), (unsigned)(((4 + kj) ^ kt) << 4)};     // of 128 swizzled bytes
    struct Words {
      unsigned k[2][G], v[4][G / 2], n[G];
    };
    auto load = [&](Words& to, long long at) {
      if (at < 0) return;
      auto &kw = to.k;
      auto &vw = to.v;
      auto &nw = to.n;
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
    // pages are asked for two records ahead, words one: neither is waited for where it is asked for
    int page_1 = page_of(own + CONV), page_2 = page_of(own + 2 * CONV);
    long long at = record(own, page_of(own));
    Words now, then;
    load(now, at);
    bool ok = true;
#pragma unroll 2
    for (int n = own; n < records; n += CONV) {
      const int j = n / RECS, rec = n % RECS, st = j % STAGES, round = j / STAGES;
      const long long at_then = record(n + CONV, page_1);
      load(then, at_then);
      page_1 = page_2;
      page_2 = page_of(n + 3 * CONV);
      auto &kw = now.k;
      auto &vw = now.v;
      auto &nw = now.n;
      const bool seen = at >= 0;
      const int key = (t_begin * RECS + n) * REC_TOKENS + 2 * np;            // the numbers' two tokens
      // places that hold no key of this row tile may hold anything: their numbers count as zero
      const unsigned keep = !seen ? 0u : (key <= pos_max && key >= low_min ? 0xffffu : 0u) |
                                             (key + 1 <= pos_max && key + 1 >= low_min ? 0xffff0000u : 0u);
      unsigned most[2] = {0, 0};                       // of the two tokens
#pragma unroll
      for (int g = 0; g < G; ++g) {
        nw[g] &= keep;
        most[0] = max(most[0], nw[g] & 0x7fffu);
        most[1] = max(most[1], (nw[g] >> 16) & 0x7fffu);
      }
      // kinds by eights of lanes: lo and s of keys, lo and s of values.  The unit is such that s reaches up to 2^-8 and lo
      // stays within float16
      const int e_own = (int)(max(most[0], most[1]) >> 7) - 127 + (kind & 1 ? 9 : -14);
      const int e = max(-MOST_E, min(MOST_E + 9, lane < 16 ? __reduce_max_sync(0x0000ffffu, e_own) : __reduce_max_sync(0xffff0000u, e_own)));
      // A token whose s is far below the record's largest number would lose its bits to that, and to rows that see no larger one it
      // is all there is: the tokens of such a record have units of their own.  (Within EVEN the shared unit leaves 2^-12 of s * 15.)
      const bool far = (kind & 1) && ((keep & 0xffffu && (int)(most[0] >> 7) - 127 + 9 < e - EVEN) ||
                                      (keep >> 16 && (int)(most[1] >> 7) - 127 + 9 < e - EVEN));
      bool own_units = __any_sync(0xffffffffu, far);
      int e_tok[2] = {e, e};
      if (own_units) {
        // looked at once more with the token's lo: one whose numbers are all zero has nothing to lose
        int e_i[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          e_i[i] = most[i] ? (int)(most[i] >> 7) - 127 + (kind & 1 ? 9 : -14) : NOTHING;
          e_i[i] = max(e_i[i], __shfl_xor_sync(0xffffffffu, e_i[i], 8));
        }
        own_units = __any_sync(0xffffffffu, (e_i[0] != NOTHING && max(-MOST_E, e_i[0]) < e - EVEN) ||
                                                (e_i[1] != NOTHING && max(-MOST_E, e_i[1]) < e - EVEN));
#pragma unroll
        for (int i = 0; i < 2; ++i)
          if (own_units) e_tok[i] = max(-MOST_E, min(MOST_E + 9, e_i[i]));
      }
      const float by[2] = {pow2((kind & 1 ? 24 : 0) - e_tok[0]), pow2((kind & 1 ? 24 : 0) - e_tok[1])};
      unsigned half[G];
#pragma unroll
      for (int g = 0; g < G; ++g)
        half[g] = h2(__uint_as_float(nw[g] << 16) * by[0], __uint_as_float(nw[g] & 0xffff0000u) * by[1]);
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
      ok = ok && mbar_wait(&empty[st], (round & 1) ^ 1, err);
      if (lane == 0) units[st].key[rec] = seen ? pow2(e) : -1.f;
      if (lane == 16) units[st].value[rec] = own_units ? e + UNEVEN : e;
      if (own_units && !(kind & 1))
        *reinterpret_cast<float2*>((kind == K_LO ? units[st].key_of : units[st].value_of) + rec * REC_TOKENS + 2 * np) =
            make_float2(pow2(e_tok[0]), pow2(e_tok[1]));
      __syncwarp();                                    // the numbers are there: each is read by other lanes than its own
      // ---- keys
      // (a record that is not seen, or a place without a key, has numbers that are zero, whatever its codes)
      unsigned char* kd = Ks + st * T_BYTES + rec * (REC_TOKENS * 128) + kt * 128;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        unsigned sc[G], lo[G];
        words<G>(sc, kn + (kt + 8 * i) * G);
        words<G>(lo, kn + 16 * G + (kt + 8 * i) * G);
#pragma unroll
        for (int g = 0; g < G; ++g) {
          unsigned x[4];
          four_pairs(kw[i][g], sc[g], lo[g], x);
          *reinterpret_cast<uint4*>(kd + (g >> 1) * (BN * 128) + i * 1024 + k_chunk[g & 1]) = make_uint4(x[0], x[1], x[2], x[3]);
        }
      }
      // ---- values
      unsigned char* vd = Vs + st * T_BYTES + (32 * vg + vr) * 128 + (((2 * rec + vc) ^ vr) << 4);
      unsigned sc[4][G / 2], lo[4][G / 2];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        words<G / 2>(sc[i], vn + (4 * vc + i) * G + vg);
        words<G / 2>(lo[i], vn + 8 * G + (4 * vc + i) * G + vg);
      }
#pragma unroll
      for (int g = 0; g < G / 2; ++g) {
        unsigned x[4][4];                              // [pair][i]
#pragma unroll
        for (int i = 0; i < 4; ++i) four_pairs(vw[i][g], sc[i][g], lo[i][g], x[i]);
#pragma unroll
        for (int i = 0; i < 4; ++i)
          *reinterpret_cast<uint4*>(vd + (32 * g + 8 * i) * 128) = make_uint4(x[0][i], x[1][i], x[2][i], x[3][i]);
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(&full[st]);
      now = then;
      at = at_then;
    }
    // the commits that release the last tiles arrive whenever the tensor core gets there: not after the block is gone
    if (own == 0 && lane == 0) {
      for (int j = max(0, n_tiles - STAGES); j < n_tiles && ok; ++j) {
        ok = mbar_wait(&empty[j % STAGES], (j / STAGES) & 1, err);
      }
    }
  } else if (warp >= MMA_WARP) {
    const int h = warp - MMA_WARP;
    if (h < halves && n_tiles > 0) {
      // ------------------------------------------------------------ MMA issuer of half h
      const uint32_t idesc_s = idesc_f16(HALF, BN), idesc_o = idesc_f16(HALF, D);
      const uint32_t tmem = __shfl_sync(0xffffffffu, tmem_base, 0) + h * 128;
      bool ok = true;
      // an operand further on is an addition to its descriptor's address field (in units of 16 bytes)
      const uint64_t q_desc = make_desc(smem_u32(Qs) + h * (HALF * D * 2)), k_desc = make_desc(smem_u32(Ks)), v_desc = make_desc(smem_u32(Vs));
      auto scores = [&](int j) {
        const int st = j % STAGES;
        ok = ok && mbar_wait_warp(&full[st], (j / STAGES) & 1, err);
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint64_t b = k_desc + (uint32_t)(st * (T_BYTES / 16));
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks)
          mma_elected(tmem + S_COL + (j & 1) * BN, q_desc + ((ks >> 2) * (HALF * 128 / 16) + (ks & 3) * 2),
                      b + ((ks >> 2) * (BN * 128 / 16) + (ks & 3) * 2), idesc_s, ks > 0 ? 1u : 0u);
        commit_elected(&s_full[h][j & 1]);
      };
      ok = ok && mbar_wait_warp(&q_full[h], 0, err);
      scores(0);
      if (n_tiles > 1) scores(1);
      for (int j = 0; j < n_tiles && ok; ++j) {
        const int st = j % STAGES;
        ok = ok && mbar_wait_warp(&p_full[h][j & 1], (j >> 1) & 1, err);     // P_j written, O rescaled
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint64_t b = v_desc + (uint32_t)(st * (T_BYTES / 16));
#pragma unroll
        for (int ks = 0; ks < BN / 16; ++ks)
          mma_ts_elected(tmem + O_COL, tmem + S_COL + (j & 1) * BN + ks * 8, b + ks * 2, idesc_o, (j > 0 || ks > 0) ? 1u : 0u);
        commit_elected(&o_ready[h]);
        commit_elected(&empty[st]);                    // the keys were multiplied before
        if (j + 1 == n_tiles) commit_elected(&o_done[h]);
        if (j + 2 < n_tiles) scores(j + 2);            // into the buffer that P_j has left: the tensor pipe runs in order
      }
    }
  } else if (warp < 4 * halves) {
    // ---------------------------------------------------------------- softmax, correction, epilogue
    const int h = warp >> 2, row = warp * 32 + lane, pr = pr0 + row;
    const bool row_valid = row < rows_here;
    const int q_row = row_valid ? pr / HG : 0, head = kvh * HG + (row_valid ? pr - q_row * HG : 0);
    const bool held = row_valid && q0 >= 0 && q0 + q_row < p.rows;
    const int pos = row_valid ? pos0 + q_row : -1;
    const int lo = p.window > 0 ? max(0, pos) - p.window + 1 : 0;
    // ---- the warp's 32 rows of queries as float16, each scaled by a power of two so that its largest lies in [1, 2); the lanes
    // load whole rows (a thread loading its own asks for 32 lines an instruction, and the first records wait behind them)
    float row_unit;
    constexpr int LANES = D / 8, ROWS = 32 / LANES;    // lanes a row takes, rows an instruction
    {
      const unsigned own = held ? (unsigned)(((size_t)(q0 + q_row) * H + head) * LANES) : 0xffffffffu;   // in 16 bytes
      const uint4* src = (const uint4*)p.q + lane % LANES;
      uint4 w[32 / ROWS];
#pragma unroll
      for (int i = 0; i < 32 / ROWS; ++i) {
        const unsigned from = __shfl_sync(0xffffffffu, own, i * ROWS + lane / LANES);
        w[i] = from != 0xffffffffu ? src[from] : make_uint4(0, 0, 0, 0);
      }
      int e_row = 0;
#pragma unroll
      for (int i = 0; i < 32 / ROWS; ++i) {
        const unsigned u[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
        unsigned most = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) most = max(most, max(u[k] & 0x7fffu, (u[k] >> 16) & 0x7fffu));
#pragma unroll
        for (int o = 1; o < LANES; o <<= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
        const int e = max(-MOST_E, min(MOST_E, (int)(most >> 7) - 127));
        const int e_there = __shfl_sync(0xffffffffu, e, lane % ROWS * LANES);
        if (lane / ROWS == i) e_row = e_there;
        const float by = pow2(-e);
        unsigned x[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) x[k] = h2(__uint_as_float(u[k] << 16) * by, __uint_as_float(u[k] & 0xffff0000u) * by);
        const int to = (warp & 3) * 32 + i * ROWS + lane / LANES, c = lane % LANES;
        *reinterpret_cast<uint4*>(Qs + h * (HALF * D * 2) + (c >> 3) * (HALF * 128) + swizzled(to, c & 7)) = make_uint4(x[0], x[1], x[2], x[3]);
      }
      row_unit = pow2(e_row) * p.scale * 1.4426950408889634f;
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(&q_full[h]);
    }
    const uint32_t lane_addr = tmem_base + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t s_addr = lane_addr + S_COL + h * 128, o_addr = lane_addr + O_COL + h * 128;
    float m_run = -INFINITY, l_run = 0.f;              // maximum in units of log2
    int e_run = row_valid ? -2 * MOST_E : MOST_E + 9;  // the output's unit: 2^(e_run - ROOM + m_run); rows that are none have the most
    bool ok = true, far = false;                       // far: a row of the warp has its maximum far from zero
    auto is_far = [](float m) { return __any_sync(0xffffffffu, fabsf(m) > FAR && m != -INFINITY) != 0; };
    for (int j = 0; j < n_tiles; ++j) {
      const int st = j & 1, kst = j % STAGES, ts = (t_begin + j) * BN;
      ok = ok && mbar_wait(&s_full[h][st], (j >> 1) & 1, err);
      ok = ok && mbar_wait(&full[kst], (j / STAGES) & 1, err);              // complete, but for the exponents beside it
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const Units& u = units[kst];
      const float l_was = l_run;
      float m_new = m_run, alpha = 1.f;
      int e_new = max(max(u.value[0], u.value[1]), max(u.value[2], u.value[3]));
      // tokens with units of their own, or scores far from zero: a few tiles if any
      bool one_by_one = far || e_new >= UNEVEN / 2;
      if (!one_by_one) {
        float s[BN];
        auto fetch = [&]() {
#pragma unroll
          for (int c = 0; c < BN / 32; ++c) tmem_ld32_nowait(s_addr + st * BN + c * 32, &s[c * 32]);
        };
        fetch();
        float unit[RECS];
        int ev[RECS];
        bool whole = ts + BN - 1 <= pos_min && ts >= low_max;
#pragma unroll
        for (int g = 0; g < RECS; ++g) {
          unit[g] = u.key[g] * row_unit;
          ev[g] = u.value[g];
          whole = whole && unit[g] > 0.f;
        }
        if (!whole) {                                  // of the records that the row sees
          e_new = e_run;
#pragma unroll
          for (int g = 0; g < RECS; ++g) {
            const int first = ts + g * REC_TOKENS;
            if (first <= pos && first + REC_TOKENS > lo) e_new = max(e_new, ev[g]);
          }
        }
        e_new = max(e_run, e_new);
        float sum, most, shrink = 1.f;
        uint32_t w[BN / 2];
        // weights from the scores, against the maximum so far; their sum, in units of 2^(m_new - ROOM), and the largest part of it
        auto weigh = [&]() {
          const float m_use = m_new == -INFINITY ? 0.f : m_new;
          sum = most = 0.f;
#pragma unroll
          for (int g = 0; g < RECS; ++g) {
            const float off = (float)(ROOM + ev[g] - e_new) - m_use;
            const f32x2 unit2 = both(unit[g], unit[g]), off2 = both(off, off);
            f32x2 part = both(0.f, 0.f);
#pragma unroll
            for (int i = g * 16; i < g * 16 + 16; i += 2) {
              float x, y;
              apart(fma2(both(s[i], s[i + 1]), unit2, off2), x, y);
              x = ex2(x);
              y = ex2(y);
              part = add2(part, both(x, y));
              w[i / 2] = h2(x, y);
            }
            float x, y;
            apart(part, x, y);
            most = fmaxf(most, x + y);
            sum = fmaf(x + y, ex2((float)min(e_new - ev[g], 126)), sum);
          }
        };
        auto masked = [&]() {
#pragma unroll
          for (int i = 0; i < BN; ++i) {
            const int key = ts + i;
            if (key > pos || key < lo || !(u.key[i / REC_TOKENS] > 0.f)) s[i] = -INFINITY;
          }
#pragma unroll
          for (int g = 0; g < RECS; ++g) unit[g] = fmaxf(fabsf(unit[g]), 1e-37f);      // times minus infinity: not 0
        };
        tmem_landed(s);
        if (!whole) masked();
        // Weights first, without a look at this tile's maximum: while no sum of 16 passes 2^15 none of them is too large for
        // float16.  Where one does, or none was seen before, or larger values come, the maximum is found and moved (to no more
        // than 2^8 below it) and the weights are made again: a few tiles of a row.
        weigh();
        const bool again = !(most <= 32768.f) || m_run == -INFINITY || e_new > e_run;
        if (__any_sync(0xffffffffu, again)) {
          fetch();
          tmem_landed(s);
          if (!whole) masked();
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
          m_new = fmaxf(m_run, mx);
          if (m_run != -INFINITY && m_new - m_run <= 8.0f) m_new = m_run;
          shrink = ex2(m_run - (m_new == -INFINITY ? 0.f : m_new));
          alpha = shrink * ex2((float)(e_run - e_new));
          one_by_one = far = is_far(m_new);
          weigh();
        }
        l_run = fmaf(l_run, shrink, sum);
        if (!one_by_one) tmem_st32_nowait(s_addr + st * BN, &w[0]);
      }
      if (one_by_one) {
        const Weighed x = weigh_one_by_one(&u, s_addr + st * BN, ts, lo, pos, ts + BN - 1 <= pos_min && ts >= low_max, row_unit,
                                           m_run, e_run);
        m_new = x.m, e_new = x.e, alpha = x.alpha;
        l_run = fmaf(l_was, x.shrink, x.sum);
        far = is_far(m_new);
      }
      // only a rescaled output has to wait for the product before (the scores of tile j came after that of tile j - 2)
      if (j > 0 && __any_sync(0xffffffffu, m_new > m_run || e_new > e_run)) {
        ok = ok && mbar_wait(&o_ready[h], (j - 1) & 1, err);
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
          float v[32];
          tmem_ld32(o_addr + c * 32, v);
          uint32_t x[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) x[i] = __float_as_uint(v[i] * alpha);
          tmem_st32_nowait(o_addr + c * 32, x);
        }
      }
      m_run = m_new;
      e_run = e_new;
      asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full[h][st]);      // by turns: the next tile's may come before this one is waited for
    }
    pdl_launch_dependents();
    if (n_tiles > 0) {
      ok = ok && mbar_wait(&o_done[h], 0, err);        // o_ready may be two products behind: its parity would not tell
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    } else {
      ok = ok && mbar_wait(&q_full[h], 0, err);        // another warp's queries still come to where this one's rows are laid
    }
    // l is in units of 2^(m_run - ROOM), the output in units of 2^e_run more
    const float back = n_tiles > 0 ? pow2(e_run) : 0.f;
    const float inv = sp.splits > 1 ? back : l_run > 0.f ? back / l_run : l_run == 0.f ? 0.f : l_run;
    const size_t part = ((size_t)tile.index * KV + kvh) * sp.splits + split;
    // rows are stored whole too, through shared memory that held queries (all of the half's warps have laid theirs down, and no
    // product reads them any more)
    unsigned char* stage = Qs + h * (HALF * D * 2) + (warp & 3) * (32 * D * 2);        // [32 rows][LANES chunks of 16 bytes]
    auto place = [&](int to, int c) { return stage + (to * LANES + (c ^ (to & 7))) * 16; };
    const unsigned own = held ? (unsigned)(((size_t)(q0 + q_row) * H + head) * LANES) : 0xffffffffu;
    auto flush = [&](auto store) {
      __syncwarp();
#pragma unroll
      for (int i = 0; i < 32 / ROWS; ++i) {
        const int to = i * ROWS + lane / LANES, c = lane % LANES;
        const unsigned at = __shfl_sync(0xffffffffu, own, to);
        const uint4 x = *reinterpret_cast<const uint4*>(place(to, c));
        if (at != 0xffffffffu) store(to, c, at, x);
      }
      __syncwarp();
    };
#pragma unroll
    for (int g = 0; g < G; ++g) {
      float v[32];
      if (n_tiles > 0) {                               // block-uniform: every lane takes part in the load
        tmem_ld32(o_addr + g * 32, v);
      } else {
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = 0.f;
      }
      // column 8 i + r is channel 4 r + i
      if (sp.splits == 1) {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          unsigned w[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int r8 = 2 * c + (k >> 1), i = 2 * (k & 1);
            const __nv_bfloat162 x = __floats2bfloat162_rn(v[8 * i + r8] * inv, v[8 * (i + 1) + r8] * inv);
            w[k] = *reinterpret_cast<const unsigned*>(&x);
          }
          *reinterpret_cast<uint4*>(place(lane, 4 * g + c)) = make_uint4(w[0], w[1], w[2], w[3]);
        }
      } else {
#pragma unroll
        for (int r8 = 0; r8 < 8; ++r8)
          *reinterpret_cast<float4*>(place(lane, (8 * g + r8) % LANES)) =
              make_float4(v[r8] * inv, v[8 + r8] * inv, v[16 + r8] * inv, v[24 + r8] * inv);
        if (g % (G / 2) == G / 2 - 1) {                // half of the channels are there
          const int first = g / (G / 2) * LANES;
          flush([&](int to, int c, unsigned, uint4 x) {
            reinterpret_cast<uint4*>(sp.part_o + (part * BM + (row - lane) + to) * D)[first + c] = x;
          });
        }
      }
    }
    if (sp.splits == 1) {
      flush([&](int, int c, unsigned at, uint4 x) { ((uint4*)p.out)[(size_t)at + c] = x; });
    } else if (held) {
      sp.part_ml[(part * BM + row) * 2] = m_run;
      sp.part_ml[(part * BM + row) * 2 + 1] = l_run;
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  }
  __syncthreads();
  if (warp == MMA_WARP) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(TMEM_COLS) : "memory");
  }
}

// The splits of a row tile and key/value head merged, a warp a row, in MERGE_SLICES blocks.
constexpr int MOST_SPLITS = 32, MERGE_SLICES = 16;
template <int D>
__global__ void __launch_bounds__(256) kv4_tc5_merge_kernel(Kv4AttnParams p, Tc5Split sp) {
  constexpr int C = D / 32;
  pdl_launch_dependents();
  pdl_wait();
  const int KV = p.kv_heads, H = p.heads, HG = H / KV, kvh = blockIdx.x % KV;
  const Tile tile = tile_of(p, sp.most_packed, blockIdx.x / KV);
  if (tile.req < 0) return;
  const int packed = tile.rows * HG, q0 = tile.start, lane = threadIdx.x & 31;
  for (int row = blockIdx.y * 8 + (threadIdx.x >> 5); row < BM; row += gridDim.y * 8) {
    const int pr = tile.row_tile * BM + row, q_row = pr / HG;
    if (pr >= packed || q0 < 0 || q0 + q_row >= p.rows) return;
    const size_t part0 = ((size_t)tile.index * KV + kvh) * sp.splits;
    // a lane's split (there are at most 32): maximum and sum, then its factor
    const float2 ml = lane < sp.splits ? *reinterpret_cast<const float2*>(sp.part_ml + ((part0 + lane) * BM + row) * 2)
                                       : make_float2(-INFINITY, 0.f);
    const float top = warp_max(ml.x), mine = exp2f(ml.x - (top == -INFINITY ? 0.f : top)), sum = warp_sum(mine * ml.y);
    float x[C] = {};
#pragma unroll 8
    for (int s = 0; s < sp.splits; ++s) {
      const float f = __shfl_sync(0xffffffffu, mine, s);
      const float* src = sp.part_o + ((part0 + s) * BM + row) * D + C * lane;
#pragma unroll
      for (int c = 0; c < C; c += 2) {
        const float2 y = *reinterpret_cast<const float2*>(src + c);
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
  const size_t smem = (size_t)BM * D * 2 + 2 * STAGES * (size_t)BN * D * 2 + CONV * 48 * (D / GROUP) * 4 + 1024;
  static OptIn opt_in;
  if (const cudaError_t e = opt_in(smem, kv4_attention_tc5_kernel<D>)) return (int)e;
  launch_k(kv4_attention_tc5_kernel<D>, (unsigned)(tiles * p.kv_heads * sp.splits), THREADS, smem, stream, p, sp, err);
  if (sp.splits > 1) launch_k(kv4_tc5_merge_kernel<D>, dim3(tiles * p.kv_heads, MERGE_SLICES), 256, 0, stream, p, sp);
  return launch_status();
}
}  // namespace

// Requests of more than most_packed packed rows.  tiles: row tiles of 256 packed rows, at least as many as there are.
// workspace (splits > 1): tiles * kv_heads * splits * 256 * (head_dim + 2) floats.
PBE_EXPORT int pbe_kv4_attention_tc5(const Kv4AttnParams* params, float* workspace, int tiles, int splits, int head_dim,
                                     int most_packed, int* err, cudaStream_t stream) {
  const Kv4AttnParams p = *params;
  if (p.requests <= 0 || p.rows <= 0 || tiles <= 0) return 0;
  // (rows of queries and outputs are counted by eight numbers in 32 bits)
  if ((head_dim != 64 && head_dim != 128) || splits < 1 || splits > MOST_SPLITS || !(p.scale > 0.f) ||
      (long long)tiles * p.kv_heads * splits > 0x7fffffffLL || (long long)p.rows * p.heads * (head_dim / 8) >= 0xffffffffLL)
    return (int)cudaErrorInvalidValue;
  Tc5Split sp;
  sp.part_o = workspace;
  sp.part_ml = workspace + (size_t)tiles * p.kv_heads * splits * BM * head_dim;
  sp.most_packed = most_packed;
  sp.splits = splits;
  return head_dim == 64 ? launch<64>(p, sp, tiles, err, stream) : launch<128>(p, sp, tiles, err, stream);
}
