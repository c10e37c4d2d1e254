// What both kernels of attention over 4-bit pages are given; mirrored in ops.py.
#pragma once
#include <stdint.h>

struct Kv4AttnParams {
  const void* q;               // [rows, heads * D]
  const unsigned char* pages;  // [num_pages][kv_heads][page_tokens / 16] records
  void* out;
  const int32_t* q_start;      // [requests]
  const int32_t* q_len;
  const int32_t* seq_len;
  const int32_t* block_table;  // [requests][bt_stride], table_pages of them
  long long bt_stride;
  int table_pages, num_pages, requests, rows, heads, kv_heads, page_tokens, window;
  int settled;                 // lengths, table and the keys before the requests' rows are older than the launch before this one
  float scale;
};
