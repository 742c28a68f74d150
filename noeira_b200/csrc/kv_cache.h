// Parameter blocks of the paged 8-bit cache kernels (kv_cache.cu) and of the attention over it (kv_attention.cu).
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

// status code: a row found no free block, no room in its table or none in the token buffers
#define NB_ST_CACHE_FULL 5u

struct KvPlan {
  const int *lengths, *new_lens;
  int* tables;
  const int *free_ids, *free_count;
  int *free_count_out, *starts, *ends, *row_of, *positions, *slots;
  int rows, width, block_log, free_size, tokens;
  int blocks;                                   // of the cache: an id from here on is none
  int limit;                                    // tokens that a row may hold: no more than its line of the table has room for
  unsigned int* status;
};

struct KvAppend {
  const void *k, *v;
  uint8_t* codes;
  float* scale;
  const int* slots;
  int tokens, heads, block_log, blocks, limit, window, k_vec, v_vec;
  long long k_token, k_head, v_token, v_head;   // element strides of the inputs
  long long kv_stride;                          // bytes from the keys' codes to the values'
};

struct KvReorder {
  uint8_t* codes;
  float* scale;
  const int *tables, *lengths, *parents, *spare;
  int *tables_out, *lengths_out, *spare_out;
  int blocks, heads, block, dim, rows, beams, width, planes;
  long long plane;                              // bytes of one layer's keys or values
  unsigned int* status;
};

struct KvAttn {
  const void* q;                                // bf16 [T, Hq, D], element strides q_token, q_head
  void* out;                                    // bf16 [T, Hq, D], element strides o_token, o_head
  const uint8_t* codes;                         // [2, N, H, bs, D]
  const float* scale;                           // [2, N, H]
  const int *tables, *starts, *ends;
  int rows, tokens, hq, hk, group, block_log, blocks, width;
  unsigned group_mul, hk_mul;                   // 2^32 / group and / hk, rounded up
  int kv_rows;                                  // blocks * hk * block
  int q_vec, o_vec, o_vec16;                    // 16-byte loads of q, 8- and 16-byte stores of out are aligned
  int few;                                      // rows of the batch with at most this many query rows per head are done here
  uint8_t* far;                                 // all of them, if a CTA of the kernel of prompts said so: a byte each, far_size of them
  int far_size;
  int tile;                                     // query rows of a tile
  int pieces, team;                             // warps; every tile is one block's
  long long q_token, q_head, o_token, o_head;
  long long kv_stride, s_stride;                // from the keys' codes / scales to the values'
  float scale_log2;
  float *part_o, *part_ml;                      // partial outputs, (maximum, sum)
  int4* part_job;                               // of each piece: the job that it begins and does not end
  unsigned int* status;
};

// Codes as [2][blocks * heads * block rows][dim bytes], boxes of 16 rows, with the operand swizzle of the row's width or none.
int kv_code_map(CUtensorMap* map, const KvAttn& p, int dim, int swizzled);
// Rows of the batch with more than p.few query rows, on the tensor cores (kv_attention_prompt_tcgen05.cu).
int kv_launch_prompts(const KvAttn& p, int dim, int units, cudaStream_t s);
