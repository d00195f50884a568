/*
 * b200_layer.h - the operators around paged attention in one decoder layer of a serving model:
 *
 *   b200_skip_rms_norm            residual addition + RMS norm, 16-bit or fp8 e4m3 output
 *   b200_rotary_append            rotary embedding (one to four position axes) of new queries and
 *                                 keys; the keys and values go straight into the paged caches
 *   b200_shared_prefix_attention  causal attention over paged caches for a batch whose sequences
 *                                 share one prefix; the prefix is attended once for all of them
 *
 * The conventions are those of b200_paged.h: device pointers on the current device (each aligned to
 * its elements, workspaces as stated there; anything else is refused), `stream` a
 * cudaStream_t as void*, a B200_* status code as the result, the message in b200_last_error(),
 * no exception leaves the library.  The calls are asynchronous and allocate nothing; they can be
 * captured in a CUDA graph.
 */
#ifndef B200_LAYER_H
#define B200_LAYER_H

#include <stddef.h>
#include <stdint.h>

#include "b200_paged.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---- residual addition + RMS norm ------------------------------------------------------- */

/* Widest row, and the group sizes of a grouped fp8 output. */
#define B200_SKIP_RMS_NORM_MAX_HIDDEN 32768
#define B200_SKIP_RMS_NORM_MIN_GROUP 32
#define B200_SKIP_RMS_NORM_MAX_GROUP 1024

/*
 * For every row: s = x + residual in fp32, residual_out = s rounded to T, and
 * y = s / sqrt(mean(s^2) + epsilon) * weight in fp32 (of the unrounded s).
 *   out_dtype T:             out = y rounded to T
 *   out_dtype FLOAT8E4M3FN:  per row (group_size 0) or per group of group_size channels (the last
 *                            group may be short): scale = max(max|y|, 1e-12) / 448 and
 *                            out = e4m3(y / scale), so out * scale stands for y.  Scale and
 *                            quotient are within a few units in the last place of fp32 (products
 *                            with reciprocals), so a y next to the middle of two codes may take
 *                            either.  A NaN in a group makes its scale NaN.
 * out and residual_out may be x or residual themselves (each row is read before it is written).
 */
typedef struct B200SkipRmsNormParams {
  int32_t rows;
  int32_t hidden;            /* <= B200_SKIP_RMS_NORM_MAX_HIDDEN                               */
  int32_t dtype;             /* T of x, residual, weight, residual_out: FLOAT16 or BFLOAT16    */
  int32_t out_dtype;         /* T or FLOAT8E4M3FN                                              */
  int32_t group_size;        /* fp8: 0 = one scale per row, or a power of two from 32 to 1024  */
  float epsilon;             /* >= 0                                                           */
  int64_t x_row_stride;      /* elements between rows; 0 = hidden                              */
  int64_t residual_row_stride;
  int64_t out_row_stride;
  int64_t residual_out_row_stride;
  const void* x;             /* [rows, hidden]                                                 */
  const void* residual;      /* [rows, hidden] or NULL (s = x)                                 */
  const void* weight;        /* [hidden]                                                       */
  void* out;                 /* [rows, hidden] in out_dtype                                    */
  float* scales;             /* fp8: [rows, ceil(hidden / group_size)] ([rows, 1] per row)     */
  void* residual_out;        /* [rows, hidden] or NULL (not written)                           */
} B200SkipRmsNormParams;

B200_API int b200_skip_rms_norm(const B200SkipRmsNormParams* p, void* stream);

/* ---- rotary embedding + KV append ------------------------------------------------------- */

#define B200_MAX_ROTARY_AXES 4
/* Calls of more tokens than this need a workspace (duplicate slots are resolved in a table). */
#define B200_ROTARY_APPEND_SCAN_TOKENS 8192

/*
 * Channels [rotary_offset, rotary_offset + rotary_dim) of every query and key head are rotated in
 * fp32 and rounded once; rotary pair i (of rotary_dim / 2) turns by row position[axis(i)][token],
 * column i of the cos / sin tables, and consists of channels (i, i + rotary_dim / 2) or, when
 * rotary_interleaved, (2 i, 2 i + 1).  Axis a owns axis_pairs[a] consecutive pairs.  Rotated
 * queries go to `output`, rotated keys and plain values to cache slot slot_mapping[token]
 * (slot = block * block_size + row; -1 = the token is not cached, its query still is rotated).
 * Of several tokens with one slot the last one is stored.  fp8 caches hold
 * e4m3(x / scale[block, kv head]), saturating.
 * A slot outside [-1, num_blocks * block_size) is not written and a position outside the tables
 * leaves its pairs unrotated; both set a bit of *device_status.
 */
typedef struct B200RotaryAppendParams {
  int32_t num_heads, kv_num_heads, head_size;
  int32_t rotary_dim;          /* even, <= head_size - rotary_offset                            */
  int32_t rotary_offset;
  int32_t rotary_interleaved;
  int32_t rotary_positions;    /* rows of the cos / sin tables                                  */
  int32_t axes;                /* 1..B200_MAX_ROTARY_AXES                                       */
  int32_t axis_pairs[B200_MAX_ROTARY_AXES]; /* pairs per axis; they sum to rotary_dim / 2       */
  int32_t act_dtype;           /* FLOAT16 or BFLOAT16 (T)                                       */
  int32_t cache_dtype;         /* T or FLOAT8E4M3FN                                             */
  int32_t table_dtype;         /* of cos / sin: T or FLOAT                                      */
  int32_t position_dtype;      /* INT32 or INT64                                                */
  int32_t num_tokens, num_blocks, block_size;
  int64_t query_row_stride;    /* elements between tokens; 0 = dense                            */
  int64_t key_row_stride, value_row_stride;
  int64_t output_row_stride;
  int64_t position_axis_stride;  /* elements between axes                                       */
  int64_t position_token_stride; /* elements between tokens; 0 = 1                              */
  const void* query;           /* [num_tokens, num_heads * head_size]                           */
  const void* key;             /* [num_tokens, kv_num_heads * head_size]                        */
  const void* value;
  void* output;                /* [num_tokens, num_heads * head_size] in T; may be `query`      */
  void* key_cache;             /* [num_blocks, block_size, kv_num_heads, head_size]             */
  void* value_cache;
  const void* position_ids;    /* [axes, num_tokens]                                            */
  const void* cos_cache;       /* [rotary_positions, rotary_dim / 2]                            */
  const void* sin_cache;
  const int32_t* slot_mapping; /* [num_tokens]                                                  */
  const float* k_scale;        /* fp8 caches: [num_blocks, kv_num_heads]                        */
  const float* v_scale;
  void* workspace;             /* >= b200_rotary_append_workspace_size() bytes, aligned to 4;
                                  NULL when that is 0                                           */
  size_t workspace_bytes;
  int32_t* device_status;      /* see b200_layer_read_status; NULL = not reported               */
} B200RotaryAppendParams;

B200_API int b200_rotary_append_workspace_size(const B200RotaryAppendParams* p, size_t* bytes);
B200_API int b200_rotary_append(const B200RotaryAppendParams* p, void* stream);

/* ---- attention over a shared prefix ------------------------------------------------------ */

#define B200_SHARED_PREFIX_MAX_HEAD_SIZE 256

/*
 * Every sequence's keys are the prefix_length keys of prefix_block_table (shared by the whole
 * batch) followed by its own past_seqlens[b] + n_b keys in row b of block_table, with
 * n_b = cumulative_sequence_length[b + 1] - cumulative_sequence_length[b] new tokens.  New token i
 * sees the whole prefix and its own keys [0, past_seqlens[b] + i].  All keys, the new tokens' own
 * included, are read from the caches (b200_rotary_append or b200_kv_append first).
 * Scores are scale * q.k, soft-capped as softcap * tanh(score / softcap) when softcap > 0; the
 * optional head_sink adds exp(sink[h]) to each softmax denominator.  Softmax and sums are fp32.
 * For their product with the values the weights are rounded to fp16 or carried as two bf16 parts; the
 * values enter as they are stored, whatever their magnitude.
 * Pages may hold anything in slots past a sequence's (or the prefix's) last key.  A NaN in a query or
 * in a key makes the rows that see it NaN, and no others.  The values of a call's new tokens should be
 * finite: hidden ones are multiplied with a weight of zero, so an infinity or NaN in the value of a new
 * token can reach earlier tokens of the same sequence in the call.
 * Head sizes 64 and 128 with a block_size that is a multiple of 16, at most 128 query heads per kv head
 * and 16-byte aligned rows run on the tensor cores; everything else, up to head size 256, runs in a
 * plain kernel that reads the prefix again for every token and head.
 * Invalid metadata (lengths, table capacity, block ids) sets bits of *device_status; the rows it
 * concerns are unspecified, nothing outside the tensors is read or written.
 */
typedef struct B200SharedPrefixParams {
  int32_t num_heads, kv_num_heads, head_size;
  float scale;                 /* 0 = 1 / sqrt(head_size)                                       */
  float softcap;               /* 0 = none                                                      */
  int32_t act_dtype;           /* T of query, caches, head_sink, output: FLOAT16 or BFLOAT16    */
  int32_t num_tokens;          /* packed new tokens                                             */
  int32_t batch;               /* positive, or 0 without tokens                                 */
  int32_t num_blocks, block_size;
  int32_t max_blocks_per_seq;  /* columns of block_table                                        */
  int32_t prefix_length;       /* keys of the prefix, >= 0                                      */
  int32_t prefix_blocks;       /* entries of prefix_block_table                                 */
  int32_t num_sms;             /* 0 = query the device; at most 1024                            */
  int64_t query_row_stride;    /* elements between tokens; 0 = num_heads * head_size            */
  int64_t output_row_stride;
  const void* query;           /* [num_tokens, num_heads * head_size]                           */
  const void* key_cache;       /* [num_blocks, block_size, kv_num_heads, head_size]             */
  const void* value_cache;
  const int32_t* cumulative_sequence_length; /* [batch + 1]                                     */
  const int32_t* past_seqlens;               /* [batch]                                         */
  const int32_t* block_table;                /* [batch, max_blocks_per_seq]                     */
  const int32_t* prefix_block_table;         /* [prefix_blocks]; may be NULL without a prefix   */
  const void* head_sink;       /* [num_heads] in T or NULL                                      */
  void* output;                /* [num_tokens, num_heads * head_size]                           */
  void* workspace;             /* >= b200_shared_prefix_attention_workspace_size() bytes,
                                  aligned to 16                                                 */
  size_t workspace_bytes;
  int32_t* device_status;      /* see b200_layer_read_status; NULL = not reported               */
} B200SharedPrefixParams;

/* Bytes of device workspace (shapes and prefix_length only).  A workspace serves one call in
 * flight.  Most of it holds fp32 partial outputs: num_tokens * num_heads * (head_size + 2) floats for the
 * own keys and for each range that the prefix is split into (up to 64 with few tokens, one or two with
 * many), 15 to 29 MB for cut own keys, and for bf16 calls of many tokens an fp16 copy of the prefix's
 * values. */
B200_API int b200_shared_prefix_attention_workspace_size(const B200SharedPrefixParams* p, size_t* bytes);
B200_API int b200_shared_prefix_attention(const B200SharedPrefixParams* p, void* stream);

/* ---- status ------------------------------------------------------------------------------ */

/* Synchronise `stream`, read a status word that calls of this header were given as device_status (zero
 * it once before its first use; the calls only set bits) and clear the bits that it held.  B200_ERR_FAIL
 * for invalid metadata, B200_ERR_DEVICE for a device wait that ran out.  A report does not say which call
 * made it: give streams, and graphs that are replayed elsewhere, a word each. */
B200_API int b200_layer_read_status(int32_t* device_status, void* stream);

/* sizeof of the parameter structs (0 skip RMS norm, 1 rotary append, 2 shared prefix), for binding
 * layout checks. */
B200_API size_t b200_layer_struct_size(int32_t which);

#ifdef __cplusplus
}
#endif

#endif /* B200_LAYER_H */
