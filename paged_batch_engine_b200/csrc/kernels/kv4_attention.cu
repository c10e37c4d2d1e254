// Causal attention of every row over 4-bit pages (kv4.cuh).
//
// A warp takes one row of one head and walks over its keys one by one: the dot product over the lanes, the running maximum and
// sum of the softmax, and each lane's channels of the output in float32.
#include "common.cuh"
#include "kv4.cuh"
#include "pdl.cuh"

using namespace pbe;
using namespace pbe::kv4;

namespace {
struct Kv4AttnParams {
  const void* q;
  const unsigned char* pages;
  void* out;
  const int32_t* q_start;
  const int32_t* q_len;
  const int32_t* seq_len;
  const int32_t* block_table;
  long long bt_stride;
  int table_pages, num_pages, requests, rows, heads, kv_heads, page_tokens, window;
  float scale;
};

template <typename T, int D>
__global__ void kv4_attention_kernel(Kv4AttnParams p) {
  pdl_wait();
  constexpr int E = D / 32, G = D / GROUP;
  const int r = blockIdx.x, lane = threadIdx.x & 31, H = p.heads, head = blockIdx.y, kvh = head / (H / p.kv_heads);
  const int n = p.q_len[r], seq = p.seq_len[r], q0 = p.q_start[r];
  for (int i = blockIdx.z * (blockDim.x >> 5) + (threadIdx.x >> 5); i < n; i += gridDim.z * (blockDim.x >> 5)) {
    if (q0 + i >= p.rows) return;
    const int pos = seq - n + i;
    const size_t at = ((size_t)(q0 + i) * H + head) * D;
    float q[E], o[E] = {}, m = -INFINITY, l = 0.f;
    for (int e = 0; e < E; ++e) q[e] = to_float(((const T*)p.q)[at + e * 32 + lane]);
    for (int key = p.window > 0 ? max(0, pos - p.window + 1) : 0; key <= pos; ++key) {
      const int blk = key / p.page_tokens, off = key % p.page_tokens, tok = off % REC_TOKENS;
      const int page = blk < p.table_pages ? p.block_table[r * p.bt_stride + blk] : -1;
      if (page < 0 || page >= p.num_pages) continue;
      const unsigned char* rec = p.pages + record_at(page, kvh, off, p.kv_heads, p.page_tokens, D);
      auto number = [&](int kind, int g) { return __bfloat162float(*reinterpret_cast<const __nv_bfloat16*>(rec + number_at(D, kind, tok, g))); };
      float dot = 0.f, v[E];
      for (int g = 0; g < E; ++g) {                    // the lane's channel of each group
        const int kb = 32 * ((tok * 4 + lane / 8) * G + g) + 16 * (lane & 1) + 4 * (lane % 8 >> 1);
        const int vb = 32 * ((tok / 2 * 8 + lane / 4) * G + g) + 16 * (tok & 1) + 4 * (lane & 3);
        dot = fmaf(q[g], fmaf(number(K_S, g), (float)(rec[kb / 8] >> (kb & 7) & 15), number(K_LO, g)), dot);
        v[g] = fmaf(number(V_S, g), (float)(rec[v_codes(D) + vb / 8] >> (vb & 7) & 15), number(V_LO, g));
      }
      const float s = warp_sum(dot) * p.scale, m2 = fmaxf(m, s), a = expf(m - m2), w = expf(s - m2);
      l = l * a + w;
      m = m2;
      for (int g = 0; g < E; ++g) o[g] = o[g] * a + w * v[g];
    }
    for (int e = 0; e < E; ++e) ((T*)p.out)[at + e * 32 + lane] = from_float<T>(l > 0.f ? o[e] / l : 0.f);
  }
}
}  // namespace

PBE_EXPORT int pbe_kv4_attention(const Kv4AttnParams* params, int head_dim, int most_rows, int dtype, cudaStream_t stream) {
  const Kv4AttnParams p = *params;
  if (p.requests <= 0 || p.rows <= 0) return 0;
  const dim3 grid(p.requests, p.heads, most_rows > 128 ? 32 : most_rows > 1 ? 4 : 1);
  if (dtype == PBE_F32) {
    if (head_dim == 64) launch_k(kv4_attention_kernel<float, 64>, grid, 128, 0, stream, p);
    else launch_k(kv4_attention_kernel<float, 128>, grid, 128, 0, stream, p);
  } else {
    if (head_dim == 64) launch_k(kv4_attention_kernel<__nv_bfloat16, 64>, grid, 128, 0, stream, p);
    else launch_k(kv4_attention_kernel<__nv_bfloat16, 128>, grid, 128, 0, stream, p);
  }
  return launch_status();
}
