// A key/value cache in four bits: where things lie in it.
//
// The channels of a key or a value of one head are cut into groups of 32.  A group keeps two bfloat16 numbers, lo and s, and a
// code of 0..15 for each channel, and stands for lo + s * code: lo is the smallest channel rounded down, s the span above it
// over 15, rounded up, so that every channel lies within the codes and is off by at most s / 2.  1.25 bytes hold what a
// bfloat16 cache takes 4 for (key and value of a channel): 3.2 times less to read and 3.2 times the tokens in a pool.
//
// A page of one head is page_tokens / 16 records of 16 tokens, 20 D bytes each, keys and values together, so that a tile of 16
// keys is one contiguous read:
//   0       keys' codes    [16 tokens][4 j][G] words: channels 32 g + 8 j + e of a token, e at bit 16 (e & 1) + 4 (e >> 1)
//   8 D     values' codes  [8 pairs][8 r][G] words: channels 32 g + 4 r + i of tokens 2 p and 2 p + 1, at bit 16 (t & 1) + 4 i
//   16 D    numbers        [4: lo of keys, s of keys, lo of values, s of values][8 pairs][G][2 tokens] bfloat16
// (G = D / 32).  The order is that of the tensor cores' fragments (mma.sync m16n8k16): a lane's operands are whole words of
// its token (keys, pairs of channels) or of its pair of tokens (values, pairs of tokens), and one AND takes two of them out.
#pragma once
#include <stdint.h>

namespace pbe {
namespace kv4 {
constexpr int GROUP = 32;
constexpr int REC_TOKENS = 16;
enum { K_LO = 0, K_S = 1, V_LO = 2, V_S = 3 };

__host__ __device__ constexpr int rec_bytes(int d) { return 20 * d; }
__host__ __device__ constexpr int v_codes(int d) { return 8 * d; }
__host__ __device__ constexpr int numbers(int d) { return 16 * d; }
// byte offset of a number within its record
__host__ __device__ constexpr int number_at(int d, int kind, int tok, int g) {
  return numbers(d) + kind * d + (((tok >> 1) * (d / GROUP) + g) * 2 + (tok & 1)) * 2;
}
// byte offset of the record that holds place `off` of a page, for one head
__device__ __forceinline__ long long record_at(long long page, int head, int off, int kv_heads, int page_tokens, int d) {
  return ((page * kv_heads + head) * (page_tokens / REC_TOKENS) + off / REC_TOKENS) * (long long)rec_bytes(d);
}
}  // namespace kv4
}  // namespace pbe
