/*
 * jfb paged KV cache: the kernels of a cache kept in pages instead of one
 * contiguous slot per sequence (jfb_kv_slot of jfb_kernels.h): rotary
 * positions with the append to the pages, attention of a chunk of new tokens
 * over them, the attention weight every cached key received, and the eviction
 * of the keys that received least.
 *
 * Conventions are those of jfb_kernels.h: device pointers unless a name ends
 * in _host, shapes validated on the host, a jfb_status instead of exceptions,
 * `stream` a cudaStream_t, nothing allocated here. The calls are ordered on
 * their stream and can be captured into a graph; they read the lengths, the
 * page table and the positions on the device, so a captured call serves later
 * steps whose arrays hold other values.
 *
 * Values met on the device that the host cannot check never lead to an access
 * outside the given arrays. They are counted as errors in *error_flag (may be
 * NULL; device memory, never cleared by these calls): bit 0 is set when a page
 * id, a length, a slot or a row range is outside its array (the effect is
 * stated per call), bit 1 when a bounded wait inside a kernel gave up and the
 * outputs are incomplete.
 *
 * Calls without rows or without sequences are allowed, with NULL for the
 * arrays that are then empty. Without rows the accumulated weight still carries
 * mass_in over to mass_out; the others do nothing.
 *
 * The reference keeps one contiguous cache per session
 * (qwen2_architecture.cpp:1072-1079) and has no counterpart of these calls.
 */
#ifndef JFB_PAGED_H
#define JFB_PAGED_H

#include <stddef.h>
#include <stdint.h>

#include "jfb/jfb_status.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef enum jfb_dtype {
    JFB_DTYPE_F32 = 0,
    JFB_DTYPE_F16 = 1,
    JFB_DTYPE_BF16 = 2,
} jfb_dtype;

#define JFB_PAGED_ERROR_RANGE 1
#define JFB_PAGED_ERROR_TIMEOUT 2

/* Most sequences of one call. */
#define JFB_PAGED_MAX_SEQUENCES 4096

/* One layer's pools. Element (page, token, kv head, d) of K is
 * k[page * page_stride + token * token_stride + head * head_stride + d], and
 * the same for V: [pages][page_size][kv_heads][head_dim] and
 * [pages][kv_heads][page_size][head_dim] are both expressed by the strides.
 * k and v are 16-byte aligned, the strides (in elements) positive multiples
 * of 8, no two elements share an address; page_size is a power of two from 8
 * to 1024; head_dim a multiple of 8 up to 128; dtype F16 or BF16. */
typedef struct jfb_paged_cache {
    void * k;
    void * v;
    uint64_t page_stride;
    uint64_t token_stride;
    uint64_t head_stride;
    uint32_t dtype;
    uint32_t pages;
    uint32_t page_size;
    uint32_t kv_heads;
    uint32_t head_dim;
    uint32_t reserved;
} jfb_paged_cache;

/* The sequences of one call. Rows q_start[b] .. q_start[b + 1] - 1 of the
 * call's row arrays are sequence b's new tokens (possibly none), in order; its
 * keys are slots 0 .. kv_len[b] - 1, slot j lying in page
 * page_table[b * table_stride + j / page_size]. kv_len counts the new tokens:
 * they hold the last slots, so new token i of n has slot kv_len - n + i. A
 * length beyond the table, or beyond 2^31 - 1024, is cut to it. Page ids beyond
 * the last used one are not read. Sequences may share pages that no call writes
 * (a common prefix). Rows at and behind q_start[sequences] belong to no
 * sequence: nothing of theirs is used or written. The arrays must not change
 * while a call that was given them runs. */
typedef struct jfb_paged_batch {
    const int32_t * q_start;     /* [sequences + 1] */
    const int32_t * kv_len;      /* [sequences] */
    const int32_t * page_table;  /* [sequences][table_stride], table_width used */
    uint64_t table_stride;
    uint32_t sequences;
    uint32_t table_width;
} jfb_paged_batch;

/* Scaling of rotary frequencies for contexts beyond the trained one. */
typedef enum jfb_rope_scaling {
    JFB_ROPE_SCALING_NONE = 0,
    JFB_ROPE_SCALING_LINEAR = 1, /* every frequency / factor (position interpolation) */
    JFB_ROPE_SCALING_NTK = 2,    /* base * factor^(d / (d - 2)) (NTK-aware) */
    JFB_ROPE_SCALING_YARN = 3,   /* YaRN: low frequencies / factor, high ones kept, a ramp between */
    JFB_ROPE_SCALING_BANDS = 4,  /* wavelength bands: long waves / factor, short ones kept, a blend between */
} jfb_rope_scaling;

/* freq_host[rope_dims / 2] = radians per position of each pair under the
 * scaling, in double, and *factor_host what cos and sin are multiplied by
 * (1 except for YaRN: 0.1 ln(factor) + 1). Base frequency i is
 * base^(-2i / rope_dims). `trained` is the context the model was trained on
 * (YaRN and bands). low and high: for YaRN the numbers of turns over `trained`
 * below which a frequency is divided and above which it is kept (commonly 1
 * and 32); for bands the divisors of `trained` that bound the blended
 * wavelengths (commonly 1 and 4). */
jfb_status jfb_rope_frequencies_host(double * freq_host, double * factor_host, uint32_t rope_dims, double base,
                                     uint32_t scaling, double factor, double trained, double low, double high);

/* Rotation of the first rope_dims of each head; the rest pass through.
 * Pair i is elements (i, i + rope_dims / 2), or (2i, 2i + 1) when interleaved;
 * its angle is pos * freq[i], formed in double. */
typedef struct jfb_rope {
    const double * freq;  /* [rope_dims / 2] */
    uint32_t rope_dims;   /* even, 2 .. head_dim */
    uint32_t interleaved;
    float factor;         /* multiplies cos and sin */
    uint32_t reserved;
} jfb_rope;

/* q_out = rotated q, and the new tokens' rotated k and their v appended to the
 * cache. Row r of q is heads x head_dim values of in_dtype at q + r * q_stride
 * (elements), k and v kv_heads x head_dim at their strides, q_out heads x
 * head_dim of the cache's dtype at q_out + r * q_out_stride. Arithmetic is in
 * f32; each value is rounded once. q_out may be q itself (same dtype and
 * stride). pos[r] is row r's rotary position, any int32: after an eviction a
 * token's position is no longer its slot. A row whose slot is negative or
 * beyond the table, or whose page id is outside the pool, gets its q_out but
 * appends nothing (error bit 0). Two rows of one call must not share a slot. */
jfb_status jfb_rope_paged_append(const void * q, const void * k, const void * v, uint32_t in_dtype, uint64_t q_stride,
                                 uint64_t k_stride, uint64_t v_stride, uint32_t rows, uint32_t heads,
                                 const int32_t * pos, const jfb_rope * rope, const jfb_paged_cache * cache,
                                 const jfb_paged_batch * batch, void * q_out, uint64_t q_out_stride,
                                 int32_t * error_flag, void * stream);

/* Workspace of jfb_paged_attention on the current device: one size for every
 * shape. Zero-filled before its first use; every call that completes leaves
 * it ready for the next, after error bit 1 it is zero-filled again. Calls that
 * overlap on the GPU need one each. */
uint64_t jfb_paged_attention_workspace_bytes(void);

/* Attention of the batch's rows over their sequences' keys. Row r of sequence
 * b at slot p sees the slots j <= p, with window > 0 only j > p - window:
 *     x_j = scale * q . k_j,   out = sum_j exp(x_j - lse) v_j,
 *     lse = log sum_j exp(x_j).
 * scale is positive, up to 1e38. Query head h reads kv head
 * h / (heads / kv_heads). q and out do not overlap (refused); they have the
 * cache's dtype, rows of heads x head_dim at their strides (elements,
 * multiples of 8, 16-byte aligned pointers); lse (may be NULL) is f32
 * [rows][heads]. Scores, the softmax's maximum and sum and the output sums are
 * f32; the exponentials are rounded to the cache's dtype for the second
 * product, where F16 leaves out those below 2^-32 of the row's largest. |x_j|
 * is meant to stay below 2^26: from there the steps of f32 are 8 and more. A
 * row that sees no key gets zeros and lse = -inf. Slots behind kv_len and
 * before every row's window are never used, whatever they hold; a key that one
 * row of a sequence's chunk sees must hold finite values of v (a non-finite one
 * may reach rows of the chunk that do not see it). A page id outside the pool
 * reads as zeros, a length beyond the table is cut to it (error bit 0). Results
 * do not depend on timing: partial sums are joined in a fixed order. One kernel
 * is chosen for all sequences of the call, by the mean of their rows and the
 * width of the table: single tokens and long chunks are faster in calls of
 * their own. */
jfb_status jfb_paged_attention(const void * q, uint64_t q_stride, uint32_t rows, uint32_t heads, float scale,
                               uint32_t window, const jfb_paged_cache * cache, const jfb_paged_batch * batch,
                               void * out, uint64_t out_stride, float * lse, void * workspace,
                               uint64_t workspace_bytes, int32_t * error_flag, void * stream);

/* The weight the batch's rows gave each key, summed over the rows and the
 * query heads of its kv head:
 *     mass_out[b][h][j] = before + sum_r exp(scale * q_r . k_j - lse_r),
 * over the rows that see slot j; lse is jfb_paged_attention's. `before` is
 * mass_in[b][h][j] for the slots the sequence held before this call, and 0
 * for its new tokens' slots or when mass_in is NULL. Both are f32
 * [sequences][kv_heads][mass_stride]; mass_in may be mass_out. Slots at and
 * behind kv_len are left as they were. Sums are f32, in a fixed order; a weight
 * below 2^-126 counts as zero. A length beyond mass_stride or the table is cut
 * to it, a page id outside the pool reads as zeros (error bit 0). The kernel is
 * chosen as for the attention. */
jfb_status jfb_paged_attention_mass(const void * q, uint64_t q_stride, uint32_t rows, uint32_t heads, float scale,
                                    uint32_t window, const float * lse, const jfb_paged_cache * cache,
                                    const jfb_paged_batch * batch, const float * mass_in, float * mass_out,
                                    uint64_t mass_stride, int32_t * error_flag, void * stream);

/* Cuts every sequence to at most `budget` keys, for each kv head by itself:
 * the last `recent` slots stay, and of the others those of the largest mass
 * (ties to the lowest slot; a NaN counts as the least). Kept keys keep their
 * order and move to slots 0, 1, ... of page_table_out [sequences]
 * [table_out_stride] (table_out_width * page_size >= budget); their masses to
 * mass_out [sequences][kv_heads][mass_out_stride] (>= budget). keep
 * [sequences][kv_heads][budget] receives the kept slots in order, -1 behind
 * them, and kv_len_out [sequences] the new lengths, min(kv_len, budget).
 * page_table_out is either the batch's own page_table, the same address (the
 * compaction is in place; mass_out may be mass, kv_len_out kv_len), or shares
 * no page with it; either way no page stands in it twice. A copy of the batch's
 * table is neither: a sequence whose first page stays its own keeps its rows
 * where they are (error bit 0 if it is cut).
 * A length beyond the table or mass_stride is cut to it; a kept row with a
 * page id outside the pool on either side is not moved (error bit 0). The
 * batch's q_start is not read. */
jfb_status jfb_paged_evict(const float * mass, uint64_t mass_stride, const jfb_paged_cache * cache,
                           const jfb_paged_batch * batch, uint32_t budget, uint32_t recent, int32_t * keep,
                           int32_t * kv_len_out, float * mass_out, uint64_t mass_out_stride,
                           const int32_t * page_table_out, uint64_t table_out_stride, uint32_t table_out_width,
                           int32_t * error_flag, void * stream);

#ifdef __cplusplus
}
#endif

#endif
