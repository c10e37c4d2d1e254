// Bias, rotary position encoding, and the write of keys and values into 4-bit pages (kv4.cuh), in one pass over the fused
// projection; and the way back, from pages to numbers.
//
// Four neighbouring threads share a group of 32 channels, eight each: minimum and maximum over the four, the group's lo and s,
// and eight codes a thread.  A code is made from the float32 value, not from a bfloat16 of it.
//
// lo is the minimum rounded down to bfloat16 and s = (maximum - lo) / 15 rounded up, so the group's span always lies within
// codes 0..15.  The division is IEEE's, the code the nearest whole number (ties to even).  NaN is kept as 0 and what lies
// beyond 2^120 as 2^120: four bits hold no mark for them, and a cache that held them would hand them to every later row.
//
// The angle position * frequency is formed in 64 bits and brought within a turn before its sine and cosine are taken in 32:
// the float32 product alone is off by up to 0.002 below position 65,536.  (rope_kv.cu takes it as it is.)
#include "common.cuh"
#include "kv4.cuh"
#include "pdl.cuh"

using namespace pbe;
using namespace pbe::kv4;

namespace {
constexpr int ROW_THREADS = 384;        // at most, of a block that keeps rows in registers
constexpr int SMS = 148, ROW_REGS = 65536, ROW_REGS_EACH = 80;

struct WriteParams {
  const void* qkv;
  const float* bias;
  void* q_out;
  unsigned char* pages;
  const int32_t* positions;
  const int32_t* slots;
  const float* inv_freq;
  int rows, heads, kv_heads, head_dim, rotary_dim, page_tokens, interleaved;
  long long places;            // pages * page_tokens
};

constexpr float MOST = 1.329227995784916e36f;          // 2^120
__device__ __forceinline__ float held(float x) {
  if (isnan(x)) return 0.f;
  return fminf(fmaxf(x, -MOST), MOST);
}
// the same of eight, looked at one by one only where something is to be changed
__device__ __forceinline__ void held(float (&x)[8]) {
  bool fine = true;
#pragma unroll
  for (int i = 0; i < 8; ++i) fine = fine && fabsf(x[i]) <= MOST;
  if (!fine) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = held(x[i]);
  }
}
// the nearest bfloat16 that is not above x, as a float (|x| <= 2^121)
__device__ __forceinline__ float down(float x) {
  const unsigned b = __float_as_uint(x);
  return __uint_as_float((x < 0.f ? b + 0xffffu : b) & 0xffff0000u);
}

// Eight channels of one group (four neighbouring lanes hold its 32) -> lo, s and the codes (in the low four bits).
//
// A code is the quotient (x - lo) / s, correctly rounded, to the nearest whole number: with the rounded reciprocal r of s one
// step of the remainder, q + (d - q s) r, gives the rounded quotient (Markstein 1990), which a division instruction each does
// in three times the instructions.  Both are first scaled by the power of two that brings s to 1..2, so nothing under- or
// overflows on the way.  0 <= d / s <= 15, and adding 1.5 * 2^23 leaves the whole number in the low bits.
__device__ __forceinline__ void quantise(const float (&x)[8], float& lo, float& s, unsigned (&code)[8]) {
  float mn = x[0], mx = x[0];
#pragma unroll
  for (int i = 1; i < 8; ++i) {
    mn = fminf(mn, x[i]);
    mx = fmaxf(mx, x[i]);
  }
#pragma unroll
  for (int o = 1; o < 4; o <<= 1) {
    mn = fminf(mn, __shfl_xor_sync(0xffffffffu, mn, o));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  }
  lo = down(mn);
  s = -down(-__fdiv_rn(mx - lo, 15.f));
  const float scale = __uint_as_float((254u - (__float_as_uint(s) >> 23)) << 23), one = s * scale;
  const float r = s > 0.f ? __frcp_rn(one) : 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float d = (x[i] - lo) * scale, q = d * r;
    code[i] = __float_as_uint(fmaf(fmaf(-q, one, d), r, q) + 12582912.f) & 15u;
  }
}

// the numbers and eight codes of a chunk of channels ch.. into its record
__device__ __forceinline__ void put(unsigned char* rec, int D, int tok, int ch, bool value, float lo, float s,
                                    const unsigned (&code)[8]) {
  const int g = ch / GROUP, G = D / GROUP;
  if (!value) {
    unsigned w = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) w |= code[e] << (16 * (e & 1) + 4 * (e >> 1));
    *reinterpret_cast<unsigned*>(rec + tok * (D / 2) + ((ch % GROUP / 8) * G + g) * 4) = w;
  } else {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const unsigned w = code[4 * h] | code[4 * h + 1] << 4 | code[4 * h + 2] << 8 | code[4 * h + 3] << 12;
      const int r = ch % GROUP / 4 + h;
      *reinterpret_cast<unsigned short*>(rec + v_codes(D) + (tok >> 1) * D + (r * G + g) * 4 + 2 * (tok & 1)) = (unsigned short)w;
    }
  }
  if (ch % GROUP == 0) {
    *reinterpret_cast<__nv_bfloat16*>(rec + number_at(D, value ? V_LO : K_LO, tok, g)) = __float2bfloat16_rn(lo);
    *reinterpret_cast<__nv_bfloat16*>(rec + number_at(D, value ? V_S : K_S, tok, g)) = __float2bfloat16_rn(s);
  }
}

// the turn of position `pos` about frequency j: the angle in 64 bits, its sine and cosine in 32
__device__ __forceinline__ void turn(int pos, float freq, float* sine, float* cosine) {
  double a = (double)pos * (double)freq;
  a -= 6.283185307179586 * rint(a * 0.15915494309189535);
  sincosf((float)a, sine, cosine);
}

// eight numbers as they lie in memory
template <typename T>
struct Eight {
  uint4 w[sizeof(T) / 2];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) w[i] = reinterpret_cast<const uint4*>(p)[i];
  }
  __device__ __forceinline__ void to(float (&x)[8]) const {
    if constexpr (sizeof(T) == 2) {
      const unsigned u[4] = {w[0].x, w[0].y, w[0].z, w[0].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[2 * i] = __uint_as_float(u[i] << 16);
        x[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
      }
    } else {
#pragma unroll
      for (int i = 0; i < (int)sizeof(T) / 2; ++i) {
        x[4 * i] = __uint_as_float(w[i].x), x[4 * i + 1] = __uint_as_float(w[i].y);
        x[4 * i + 2] = __uint_as_float(w[i].z), x[4 * i + 3] = __uint_as_float(w[i].w);
      }
    }
  }
};
__device__ __forceinline__ void load8(float (&x)[8], const float* p) {
  Eight<float> e;
  e.load(p);
  e.to(x);
}
__device__ __forceinline__ void store8(float* p, const float (&x)[8]) {
  *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
  *reinterpret_cast<float4*>(p + 4) = make_float4(x[4], x[5], x[6], x[7]);
}
__device__ __forceinline__ void store8(__nv_bfloat16* p, const float (&x)[8]) {
  alignas(16) __nv_bfloat162 w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
  *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(w);
}

// Rows in registers: a thread has eight channels of each half of one head, the same in every row that its block takes, so that a
// rotation of whole halves (HALVES), or of neighbouring channels, needs no other thread's channels, four neighbouring threads
// hold two groups, and the bias is read once.  The next row is on its way and its sines are worked out while one is written.
// 2,048 rows of 36 heads of 128 in bfloat16 (34 MB): 15.7 us, 2.1 TB/s; the form through shared memory below takes 28.5 and a
// block a row, with its bias read and heads found anew, 18 to 20.  What is left is 300 instructions a warp and row (a third of
// them sines) beside loads that 18 warps a multiprocessor wait for.  8 rows: 2.6 us, the chain of one row's loads.
template <typename T, bool HALVES>
__global__ void __launch_bounds__(ROW_THREADS) kv4_write_rows_kernel(WriteParams p) {
  extern __shared__ __align__(16) float smem[];        // two rows' [2][half]
  pdl_launch_dependents();
  pdl_wait();
  const int H = p.heads, KV = p.kv_heads, D = p.head_dim, half = p.rotary_dim / 2, per_head = D / 16;
  const int items = (H + 2 * KV) * per_head, at = blockIdx.y * blockDim.x + threadIdx.x, item = min(at, items - 1);
  const bool own = at < items;                         // no lane leaves: a group's lanes exchange
  const int head = item / per_head, ch = (item - head * per_head) * 8, far = ch + D / 2;
  const bool stored = __any_sync(0xffffffffu, own && head >= H), value = head >= H + KV;
  const int kv = max(0, value ? head - H - KV : head - H);
  const T* in = (const T*)p.qkv + (size_t)head * D + ch;
  const size_t width = (size_t)(H + 2 * KV) * D;
  Eight<T> u, v;
  int t = blockIdx.x, slot = -1, pos = 0;
  auto ask = [&](int row) {
    u.load(in + row * width);
    v.load(in + row * width + D / 2);
    if (p.slots) slot = p.slots[row];
    pos = p.positions[row];
  };
  auto turns = [&](float* trig) {
    for (int j = threadIdx.x; j < half; j += blockDim.x) turn(pos, p.inv_freq[j], &trig[half + j], &trig[j]);
  };
  ask(t);
  float a[8] = {}, b[8] = {};
  if (p.bias) {
    load8(a, p.bias + head * D + ch);
    load8(b, p.bias + head * D + far);
  }
  float *trig = smem, *other = smem + 2 * half;
  turns(trig);
  for (; t < p.rows; t += gridDim.x) {
    float x[8], y[8];
    u.to(x);
    v.to(y);
    const int to = slot;
    const bool more = t + (int)gridDim.x < p.rows;
    if (more) ask(t + gridDim.x);
    __syncthreads();                                   // this row's sines are there, the last row's are read
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] += a[i], y[i] += b[i];
    if (head < H + KV) {
      if (HALVES) {
        float c[8], s[8];
        load8(c, trig + ch);
        load8(s, trig + half + ch);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float left = x[i], right = y[i];
          x[i] = left * c[i] - right * s[i];
          y[i] = right * c[i] + left * s[i];
        }
      } else {
        auto pairs = [&](float (&z)[8], int from) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int j = from / 2 + i;
            if (j >= half) continue;
            const float left = z[2 * i], right = z[2 * i + 1], c = trig[j], s = trig[half + j];
            z[2 * i] = left * c - right * s;
            z[2 * i + 1] = right * c + left * s;
          }
        };
        pairs(x, ch);
        pairs(y, far);
      }
    }
    if (own && head < H) {
      T* out = (T*)p.q_out + ((size_t)t * H + head) * D + ch;
      store8(out, x);
      store8(out + D / 2, y);
    }
    if (stored && p.pages != nullptr && to >= 0 && to < p.places) {
      const int page = to / p.page_tokens, off = to - page * p.page_tokens;
      unsigned char* rec = p.pages + record_at(page, kv, off, KV, p.page_tokens, D);
      float lo, s;
      unsigned code[8];
      held(x);
      held(y);
      quantise(x, lo, s, code);
      if (own && head >= H) put(rec, D, off % REC_TOKENS, ch, value, lo, s, code);
      quantise(y, lo, s, code);
      if (own && head >= H) put(rec, D, off % REC_TOKENS, far, value, lo, s, code);
    }
    if (more) turns(other);
    float* swap = trig;
    trig = other;
    other = swap;
  }
}

// The rotation of the first rotary_dim < D channels by halves, whose pairs lie anywhere: turned through shared memory, a block
// a row.
template <typename T>
__global__ void kv4_write_kernel(WriteParams p) {
  extern __shared__ float smem[];
  pdl_launch_dependents();
  pdl_wait();
  const int t = blockIdx.x;
  const int H = p.heads, KV = p.kv_heads, D = p.head_dim, half = p.rotary_dim / 2;
  float* trig = smem;                                  // [2][half]
  float* kv = smem + 2 * half;                         // [2 KV][D]: keys, then values
  const T* in = (const T*)p.qkv + (size_t)t * (H + 2 * KV) * D;
  const int slot = p.slots ? p.slots[t] : -1;
  const bool write = p.pages != nullptr && slot >= 0 && slot < p.places;
  for (int j = threadIdx.x; j < half; j += blockDim.x) {
    turn(p.positions[t], p.inv_freq[j], &trig[half + j], &trig[j]);
  }
  __syncthreads();
  auto at = [&](int col) { return to_float(in[col]) + (p.bias ? p.bias[col] : 0.f); };
  const int per_head = half + (D - p.rotary_dim);
  const int turned = (H + (write ? KV : 0)) * per_head;
  for (int item = threadIdx.x; item < turned; item += blockDim.x) {
    const int head = item / per_head, j = item - head * per_head, base = head * D;
    int i0, i1;
    float a, b = 0.f;
    if (j < half) {
      i0 = p.interleaved ? 2 * j : j;
      i1 = p.interleaved ? 2 * j + 1 : j + half;
      const float u = at(base + i0), v = at(base + i1), c = trig[j], s = trig[half + j];
      a = u * c - v * s;
      b = v * c + u * s;
    } else {
      i0 = i1 = p.rotary_dim + (j - half);
      a = at(base + i0);
    }
    if (head < H) {
      T* dst = (T*)p.q_out + (size_t)t * H * D + base;
      dst[i0] = from_float<T>(a);
      if (i1 != i0) dst[i1] = from_float<T>(b);
    } else {
      float* dst = kv + (head - H) * D;
      dst[i0] = held(a);
      if (i1 != i0) dst[i1] = held(b);
    }
  }
  if (!write) return;
  for (int e = threadIdx.x; e < KV * D; e += blockDim.x) kv[KV * D + e] = held(at((H + KV) * D + e));
  __syncthreads();
  const int chunks = 2 * KV * (D / 8);                 // of eight channels
  const long long page = slot / p.page_tokens;
  const int off = slot % p.page_tokens, tok = off % REC_TOKENS;
  for (int c0 = 0; c0 < chunks; c0 += blockDim.x) {
    const int c = c0 + threadIdx.x, cc = min(c, chunks - 1);       // no lane leaves: a group's lanes exchange
    const int row = cc / (D / 8), ch = (cc % (D / 8)) * 8;
    const bool value = row >= KV;
    const int head = value ? row - KV : row;
    float x[8], lo, s;
    unsigned code[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = kv[row * D + ch + i];
    quantise(x, lo, s, code);
    if (c < chunks) put(p.pages + record_at(page, head, off, KV, p.page_tokens, D), D, tok, ch, value, lo, s, code);
  }
}

// a thread takes eight channels of a key and of its value (2,048 rows of 4 heads of 128: 5.4 us, 11 with outputs stored one
// by one)
template <typename T>
__global__ void kv4_read_kernel(const unsigned char* pages, const int32_t* slots, T* k, T* v, int rows, int kv_heads,
                                int head_dim, int page_tokens, long long places) {
  pdl_launch_dependents();
  pdl_wait();
  const int D = head_dim, G = D / GROUP, per_row = kv_heads * (D / 8), row = blockIdx.x * blockDim.y + threadIdx.y;
  if (row >= rows) return;
  const int slot = slots[row];
  for (int rest = threadIdx.x; rest < per_row; rest += blockDim.x) {
    const int head = rest / (D / 8), ch = rest % (D / 8) * 8, g = ch / GROUP;
    float a[8] = {}, b[8] = {};
    if (slot >= 0 && slot < places) {
      const int off = slot % page_tokens, tok = off % REC_TOKENS;
      const unsigned char* rec = pages + record_at(slot / page_tokens, head, off, kv_heads, page_tokens, D);
      auto number = [&](int kind) { return __bfloat162float(*reinterpret_cast<const __nv_bfloat16*>(rec + number_at(D, kind, tok, g))); };
      const float klo = number(K_LO), ks = number(K_S), vlo = number(V_LO), vs = number(V_S);
      const unsigned w = *reinterpret_cast<const unsigned*>(rec + tok * (D / 2) + ((ch % GROUP / 8) * G + g) * 4);
#pragma unroll
      for (int e = 0; e < 8; ++e) a[e] = fmaf(ks, (float)(w >> (16 * (e & 1) + 4 * (e >> 1)) & 15u), klo);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const unsigned u = *reinterpret_cast<const unsigned short*>(rec + v_codes(D) + (tok >> 1) * D +
                                                                    ((ch % GROUP / 4 + h) * G + g) * 4 + 2 * (tok & 1));
#pragma unroll
        for (int i = 0; i < 4; ++i) b[4 * h + i] = fmaf(vs, (float)(u >> (4 * i) & 15u), vlo);
      }
    }
    T* ko = k + (size_t)row * kv_heads * D + head * D + ch;
    T* vo = v + (size_t)row * kv_heads * D + head * D + ch;
    store8(ko, a);
    store8(vo, b);
  }
}
}  // namespace

PBE_EXPORT int pbe_kv4_write(const void* qkv, const float* bias, void* q_out, void* pages, const int32_t* positions,
                             const int32_t* slots, const float* inv_freq, int rows, int heads, int kv_heads, int head_dim,
                             int rotary_dim, int page_tokens, int interleaved, long long num_pages, int dtype,
                             cudaStream_t stream) {
  if (rows <= 0) return 0;
  if (heads < 1 || kv_heads < 1 || rotary_dim < 0 || rotary_dim > head_dim || (rotary_dim & 1) || head_dim % GROUP != 0 ||
      page_tokens % REC_TOKENS != 0)
    return (int)cudaErrorInvalidValue;
  WriteParams p{qkv, bias, q_out, (unsigned char*)pages, positions, slots, inv_freq, rows, heads, kv_heads, head_dim,
                rotary_dim, page_tokens, interleaved, num_pages * page_tokens};
  const bool halves = !interleaved && rotary_dim == head_dim;
  if ((halves || interleaved || rotary_dim == 0) && head_dim % 64 == 0) {
    const int items = (heads + 2 * kv_heads) * (head_dim / 16), slices = (items + ROW_THREADS - 1) / ROW_THREADS;
    const int threads = ((items + slices - 1) / slices + 31) / 32 * 32;
    const int most = max(1, SMS * max(1, ROW_REGS / (ROW_REGS_EACH * threads)) / slices), rounds = (rows + most - 1) / most;
    const dim3 grid((rows + rounds - 1) / rounds, slices);
    const size_t trig = 2 * (size_t)rotary_dim * sizeof(float);
    if (dtype == PBE_F32)
      launch_k(halves ? kv4_write_rows_kernel<float, true> : kv4_write_rows_kernel<float, false>, grid, threads, trig, stream, p);
    else
      launch_k(halves ? kv4_write_rows_kernel<__nv_bfloat16, true> : kv4_write_rows_kernel<__nv_bfloat16, false>, grid, threads,
               trig, stream, p);
    return launch_status();
  }
  const size_t smem = (size_t)(rotary_dim + 2 * kv_heads * head_dim) * sizeof(float);
  if (smem > 48 * 1024) return (int)cudaErrorInvalidValue;
  if (dtype == PBE_F32) launch_k(kv4_write_kernel<float>, rows, 256, smem, stream, p);
  else launch_k(kv4_write_kernel<__nv_bfloat16>, rows, 256, smem, stream, p);
  return launch_status();
}

PBE_EXPORT int pbe_kv4_read(const void* pages, const int32_t* slots, void* k, void* v, int rows, int kv_heads, int head_dim,
                            int page_tokens, long long num_pages, int dtype, cudaStream_t stream) {
  if (rows <= 0) return 0;
  if (kv_heads < 1 || head_dim < GROUP || head_dim % GROUP != 0 || page_tokens < 1 || page_tokens % REC_TOKENS != 0)
    return (int)cudaErrorInvalidValue;
  const int across = kv_heads * (head_dim / 8) < 128 ? kv_heads * (head_dim / 8) : 128;
  const dim3 threads(across, 128 / across);
  const unsigned blocks = (unsigned)((rows + threads.y - 1) / threads.y);
  const long long places = num_pages * page_tokens;
  if (dtype == PBE_F32)
    launch_k(kv4_read_kernel<float>, blocks, threads, 0, stream, (const unsigned char*)pages, slots, (float*)k, (float*)v,
             rows, kv_heads, head_dim, page_tokens, places);
  else
    launch_k(kv4_read_kernel<__nv_bfloat16>, blocks, threads, 0, stream, (const unsigned char*)pages, slots,
             (__nv_bfloat16*)k, (__nv_bfloat16*)v, rows, kv_heads, head_dim, page_tokens, places);
  return launch_status();
}
