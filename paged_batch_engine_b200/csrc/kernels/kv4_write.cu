// Bias, rotary position encoding, and the write of keys and values into 4-bit pages (kv4.cuh), in one pass over the fused
// projection; and the way back, from pages to numbers.
//
// A block takes one row.  Its threads turn queries (stored at once) and keys, and lay keys and values down in shared memory in
// float32; then four neighbouring threads share a group of 32 channels, eight each: minimum and maximum over the four, the
// group's lo and s, and eight codes a thread.  A code is made from the float32 value, not from a bfloat16 of it.
//
// lo is the minimum rounded down to bfloat16 and s = (maximum - lo) / 15 rounded up, so the group's span always lies within
// codes 0..15.  The division is IEEE's, the code the nearest whole number (ties to even).  NaN is kept as 0 and what lies
// beyond 2^120 as 2^120: four bits hold no mark for them, and a cache that held them would hand them to every later row.
//
// The angle position * frequency is formed in 64 bits and brought within a turn before its sine and cosine are taken in 32:
// the float32 product alone is off by 0.004 at position 65,536.
#include "common.cuh"
#include "kv4.cuh"
#include "pdl.cuh"

using namespace pbe;
using namespace pbe::kv4;

namespace {
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

__device__ __forceinline__ float held(float x) {
  if (isnan(x)) return 0.f;
  constexpr float most = 1.329227995784916e36f;        // 2^120
  return fminf(fmaxf(x, -most), most);
}
// the nearest bfloat16 that is not above x, as a float (|x| <= 2^121)
__device__ __forceinline__ float down(float x) {
  const unsigned b = __float_as_uint(x);
  return __uint_as_float((x < 0.f ? b + 0xffffu : b) & 0xffff0000u);
}

// eight channels of one group (four neighbouring lanes hold its 32) -> lo, s and the codes
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
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float c = s > 0.f ? rintf(__fdiv_rn(x[i] - lo, s)) : 0.f;
    code[i] = (unsigned)fminf(fmaxf(c, 0.f), 15.f);
  }
}

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
    double a = (double)p.positions[t] * (double)p.inv_freq[j];
    a -= 6.283185307179586 * rint(a * 0.15915494309189535);
    sincosf((float)a, &trig[half + j], &trig[j]);
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
    const int head = value ? row - KV : row, g = ch / GROUP, G = D / GROUP;
    float x[8], lo, s;
    unsigned code[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = kv[row * D + ch + i];
    quantise(x, lo, s, code);
    if (c >= chunks) continue;
    unsigned char* rec = p.pages + record_at(page, head, off, KV, p.page_tokens, D);
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
}

template <typename T>
__global__ void kv4_read_kernel(const unsigned char* pages, const int32_t* slots, T* k, T* v, int rows, int kv_heads,
                                int head_dim, int page_tokens, long long places) {
  pdl_launch_dependents();
  pdl_wait();
  const int D = head_dim, G = D / GROUP, per_row = kv_heads * (D / 8);
  const long long items = (long long)rows * per_row;
  for (long long item = (long long)blockIdx.x * blockDim.x + threadIdx.x; item < items; item += (long long)gridDim.x * blockDim.x) {
    const int row = (int)(item / per_row), rest = (int)(item % per_row), head = rest / (D / 8), ch = rest % (D / 8) * 8;
    const int slot = slots[row], g = ch / GROUP;
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
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      ko[i] = from_float<T>(a[i]);
      vo[i] = from_float<T>(b[i]);
    }
  }
}
}  // namespace

PBE_EXPORT int pbe_kv4_write(const void* qkv, const float* bias, void* q_out, void* pages, const int32_t* positions,
                             const int32_t* slots, const float* inv_freq, int rows, int heads, int kv_heads, int head_dim,
                             int rotary_dim, int page_tokens, int interleaved, long long num_pages, int dtype,
                             cudaStream_t stream) {
  if (rows <= 0) return 0;
  if (rotary_dim < 0 || rotary_dim > head_dim || (rotary_dim & 1) || head_dim % GROUP != 0 || page_tokens % REC_TOKENS != 0)
    return (int)cudaErrorInvalidValue;
  WriteParams p{qkv, bias, q_out, (unsigned char*)pages, positions, slots, inv_freq, rows, heads, kv_heads, head_dim,
                rotary_dim, page_tokens, interleaved, num_pages * page_tokens};
  const size_t smem = (size_t)(rotary_dim + 2 * kv_heads * head_dim) * sizeof(float);
  if (smem > 48 * 1024) return (int)cudaErrorInvalidValue;
  if (dtype == PBE_F32) launch_k(kv4_write_kernel<float>, rows, 256, smem, stream, p);
  else launch_k(kv4_write_kernel<__nv_bfloat16>, rows, 256, smem, stream, p);
  return launch_status();
}

PBE_EXPORT int pbe_kv4_read(const void* pages, const int32_t* slots, void* k, void* v, int rows, int kv_heads, int head_dim,
                            int page_tokens, long long num_pages, int dtype, cudaStream_t stream) {
  if (rows <= 0) return 0;
  if (head_dim % GROUP != 0 || page_tokens % REC_TOKENS != 0) return (int)cudaErrorInvalidValue;
  const long long items = (long long)rows * kv_heads * (head_dim / 8);
  long long blocks = (items + 255) / 256;
  if (blocks > 148 * 8) blocks = 148 * 8;
  const long long places = num_pages * page_tokens;
  if (dtype == PBE_F32)
    launch_k(kv4_read_kernel<float>, (unsigned)blocks, 256, 0, stream, (const unsigned char*)pages, slots, (float*)k, (float*)v,
             rows, kv_heads, head_dim, page_tokens, places);
  else
    launch_k(kv4_read_kernel<__nv_bfloat16>, (unsigned)blocks, 256, 0, stream, (const unsigned char*)pages, slots,
             (__nv_bfloat16*)k, (__nv_bfloat16*)v, rows, kv_heads, head_dim, page_tokens, places);
  return launch_status();
}
