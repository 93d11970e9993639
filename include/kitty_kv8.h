/*
 * kitty_kv8.h - C ABI of the 8-bit paged KV cache and of the per-head norm with
 * rotary embedding (libkitty_kv8.so, sm_100a).
 *
 * The conventions are those of kitty_b200.h: plain C, pointers, sizes and element
 * strides; every entry point validates its arguments on the host, launches
 * asynchronously on the given CUDA stream (cudaStream_t as void*) of the current
 * device, allocates nothing, and returns 0 or one of the KITTY_ERR_* codes there
 * (1 invalid argument, 2 unsupported, 3 CUDA error, 4 workspace), with a message in
 * kitty_kv8_last_error() (thread-local).
 *
 * Cache layout.  P pages, H KV heads, G tokens per page (a multiple of 32, at most
 * 256), D channels per head (a multiple of 16, at most 256):
 *   key_codes, value_codes   [P][H][G][D]       8-bit codes, e4m3 or int8
 *   key_scale, value_scale   [P][H]             float32, one per block of G tokens and head
 *   tail_k, tail_v           [slots][H][G][D]   fp16 or bf16
 *   block_table              [slots][max_pages] int32 page numbers
 *   lengths                  [slots]            int32 tokens
 * Token t of a slot with `len` tokens is in page block_table[slot][t / G] when
 * (t / G + 1) * G <= len and in row t % G of the slot's tail otherwise: a block is
 * quantised when its last token arrives, and until then its rows stay 16-bit.
 * The value of a code is code * scale.  With a = max(max|x|, 2^-100) over the block of
 * one head and Q = 448 (e4m3) or 127 (int8), scale = a * (1 / Q) and code = x * (1 / a * Q)
 * rounded to nearest even and saturated (int8 to -127..127); each operation is one
 * float32 operation.  A NaN in a block makes its scale NaN; an infinity makes its scale
 * infinite and its values NaN.
 *
 * Errors that only device data shows skip what they concern, never touch memory out
 * of bounds, and set a sticky bit (kitty_kv8_error_flags):
 *   bit 1  a page number outside the pool, or a block past the block table's row
 *   bit 2  row offsets, those of padding entries included, that decrease, are negative or
 *          pass the rows of the call
 *   bit 3  a slot past the cache, or a slot repeated in one write
 *   bit 4  a negative length, a length past the block table's row, or tokens read past it
 *   bit 5  a position past the rotary table
 */
#ifndef KITTY_KV8_H_
#define KITTY_KV8_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#if defined(__GNUC__)
#pragma GCC visibility push(default) /* the library exports these functions only */
#endif

#define KITTY_KV8_ABI_VERSION 1

#define KITTY_KV8_F16 0   /* 16-bit type of a call */
#define KITTY_KV8_BF16 1
#define KITTY_KV8_E4M3 0  /* code type of a cache */
#define KITTY_KV8_INT8 1

int kitty_kv8_abi_version(void);
const char* kitty_kv8_last_error(void);

/* sizeof() of the argument structs: 0 KittyKv8Cache, 1 KittyKv8WriteArgs,
 * 2 KittyKv8ReadArgs, 3 KittyKv8AttentionArgs, 4 KittyQkNormRopeArgs; 0 otherwise. */
size_t kitty_kv8_args_size(int kind);

/* Sticky error bits of the current device (above); synchronises with it.
 * clear != 0 resets them after reading. */
int kitty_kv8_error_flags(uint32_t* flags, int clear);

/* The cache arrays of one layer (device memory, contiguous except for the row stride
 * of the block table). */
typedef struct KittyKv8Cache {
  void* key_codes;             /* 16-byte aligned */
  void* value_codes;
  float* key_scale;
  float* value_scale;
  void* tail_k;                /* 16-byte aligned */
  void* tail_v;
  const int32_t* block_table;
  const int32_t* lengths;      /* [slots]; for a write: the tokens before it */
  int64_t bt_s_slot;           /* elements between block-table rows */
  int64_t pages;               /* P */
  int32_t slots, max_pages;    /* rows of tail / block_table / lengths; entries of a row */
  int32_t num_heads, head_dim, page_size;
  int32_t code, dtype;         /* KITTY_KV8_E4M3 / INT8; KITTY_KV8_F16 / BF16 (tails and rows) */
} KittyKv8Cache;

/* Append rows to n slots: entry i gets rows row_offsets[i] .. row_offsets[i+1] - 1 of
 * key / value (row r, head h, channel c at base + r*s_row + h*s_head + c; 16-byte
 * aligned rows) behind the lengths[slot] tokens that it has, slot = seq_map[i] (NULL:
 * i).  row_offsets NULL: one row each, n == rows.  Rows behind the last offset are
 * ignored, and so are entries of a negative slot (padding).  Blocks that fill are
 * quantised into their pages, which block_table must hold; the rest goes to the tail.
 * `lengths` is not changed: the caller adds the new tokens before it reads the cache.
 * One launch.  A slot given twice keeps its first entry. */
typedef struct KittyKv8WriteArgs {
  KittyKv8Cache cache;
  const void* key;
  const void* value;
  int64_t k_s_row, k_s_head, v_s_row, v_s_head;
  const int32_t* row_offsets;  /* [n + 1] or NULL */
  const int32_t* seq_map;      /* [n] or NULL */
  int32_t n, rows;
} KittyKv8WriteArgs;

int kitty_kv8_write(const KittyKv8WriteArgs* args, void* stream);

/* Read tokens back to 16 bits: entry i's rows row_offsets[i] .. row_offsets[i+1] - 1 of
 * key / value ([rows][H][D], contiguous, 16-byte aligned) receive tokens first[i] ..
 * (NULL: from 0) of slot seq_map[i] (NULL: i).  Rows behind the last offset, and rows
 * whose token the slot does not have, are left as they were, as are those of a negative
 * slot (padding).  One launch. */
typedef struct KittyKv8ReadArgs {
  KittyKv8Cache cache;
  void* key;
  void* value;
  const int32_t* row_offsets;  /* [n + 1] */
  const int32_t* first;        /* [n] or NULL */
  const int32_t* seq_map;      /* [n] or NULL */
  int32_t n, rows;
} KittyKv8ReadArgs;

int kitty_kv8_read(const KittyKv8ReadArgs* args, void* stream);

/* Decode attention: out[b][qh] = softmax(sm_scale * q[b][qh] . k) . v over the
 * lengths[slot] tokens of slot seq_map[b] (NULL: b), KV head qh / (Hq / H); zeros for
 * an empty slot and for a negative one (padding).  q and out have the cache's 16-bit
 * type (out may be q itself, with the same strides); sums and softmax statistics are
 * float32; the weights that multiply the values are off by at most 2^-22 of themselves,
 * or 2^-31 of the largest.  bf16 values may be as large as 2^128 / tokens (a float32 sum
 * of weights of at most 1).  The workspace (16-byte aligned) holds the partial results
 * of sequences that several warps share; calls that overlap must not share one. */
typedef struct KittyKv8AttentionArgs {
  KittyKv8Cache cache;
  const void* q;
  int64_t q_s_seq, q_s_head;   /* elements; rows 16-byte aligned */
  void* out;
  int64_t out_s_seq, out_s_head;
  const int32_t* seq_map;      /* [batch] or NULL */
  int32_t batch, num_q_heads;
  float sm_scale;
  void* workspace;
  size_t workspace_bytes;
} KittyKv8AttentionArgs;

/* Bytes of workspace that kitty_kv8_attention needs for these arguments (it depends on
 * the shapes alone, not on the lengths). */
int kitty_kv8_attention_workspace_size(const KittyKv8AttentionArgs* args, size_t* bytes);
int kitty_kv8_attention(const KittyKv8AttentionArgs* args, void* stream);

/* RMS norm of every query and key head and the rotary embedding, in one pass:
 *   y = x * rsqrt(mean(x^2) + eps) * weight   (weight NULL: y = x)
 *   (y_a, y_b) <- (y_a c - y_b s, y_b c + y_a s), i < rot / 2,
 *   c = table[pos][i], s = table[pos][rot / 2 + i],
 *   (a, b) = (i, i + rot / 2), or (2i, 2i + 1) when interleaved;
 * channels from rot on are normalised only.  float32 throughout, rounded once.
 * Outputs may be the inputs themselves (same pointer and strides).  A row with a
 * negative position is padding and is left as it was. */
typedef struct KittyQkNormRopeArgs {
  const void* q;               /* [rows][num_q_heads][head_dim], 16-byte aligned rows */
  const void* k;               /* [rows][num_k_heads][head_dim] */
  void* q_out;
  void* k_out;
  int64_t q_s_row, q_s_head, k_s_row, k_s_head;
  int64_t qo_s_row, qo_s_head, ko_s_row, ko_s_head;
  const void* q_weight;        /* [head_dim] or NULL (both or neither) */
  const void* k_weight;
  const void* positions;       /* [rows] int32 or int64 */
  const float* table;          /* [table_rows][rot], 16-byte aligned */
  int64_t table_rows;
  int32_t rows, num_q_heads, num_k_heads, head_dim, rot;
  int32_t interleaved, positions64, weight_f32; /* weight_f32: weights float32, else dtype */
  int32_t dtype;
  float eps;
} KittyQkNormRopeArgs;

int kitty_qk_norm_rope(const KittyQkNormRopeArgs* args, void* stream);

#if defined(__GNUC__)
#pragma GCC visibility pop
#endif

#ifdef __cplusplus
}
#endif

#endif /* KITTY_KV8_H_ */
