/*
 * tllm_b200_cache4.h -- a key/value cache held in 4 bits: rotary positions, append, read back and
 * attention for sequences of different lengths in one call.
 *
 * No counterpart in the reference, whose cache is FP16 with one start position for all sequences
 * (include/kernels.cuh:50-76; tllm_b200_layer.h has those operators).  At a head size of 128 a position
 * takes 72 bytes of a key or value head instead of 256.
 *
 * Cache.  Codes uint8 [batch, kv_heads, rows, dim / 2] and params half [batch, kv_heads, rows, dim / 64, 2],
 * for keys and for values.  64 neighbouring values share (s, l): value = s c + l, c = 0..15.  Eight
 * neighbouring values lie in 32 bits: value 2 i in nibble i, value 2 i + 1 in nibble i + 4.  Position p of
 * sequence b is row p of entry b.  A cache that a caller fills may have scales of either sign; its params are
 * finite and s c + l of every code within FP16's range, as append leaves them, or a key's are NaN, which marks its
 * position.  (Attention of many rows holds s c + l as FP16: beyond 65504 it would be infinite there alone.)
 *
 * Sequences of a call.  Activations are [tokens, heads, dim]; sequence b has their rows first[b] ..
 * first[b + 1] - 1 (int [batch + 1] on the device, rising) and holds lens[b] positions (int [batch] on the
 * device) with them: they sit at its last positions.  A sequence without rows takes no part.  Rows before
 * first[0] and from first[batch] on are left alone.  A row whose position would be negative is padding:
 * nothing is written for it, and its attention is 0.  first that does not rise or leaves 0..tokens, or
 * lens outside 0..rows, is cut to those limits and raises TLLM_ERR_SHAPE at the next
 * tllm_b200_check_device_errors; nothing outside the tensors is read or written.  (Where first falls,
 * attention writes nothing, and a row belongs to the first sequence that ends behind it for the others.)
 *
 * Activations: consecutive heads of a row lie behind one another, rows are ld elements apart, on 16-byte
 * boundaries.  All calls may be captured into graphs (once the library has been used on the device) and keep
 * no state between calls; calls on different streams do not disturb one another.
 */
#ifndef TLLM_B200_CACHE4_H
#define TLLM_B200_CACHE4_H

#include <stddef.h>

#include "tllm_b200.h"

#ifdef __cplusplus
extern "C" {
#endif

#define TLLM_CACHE4_GROUP 64
#define TLLM_CACHE4_LIMIT 61440.0f /* values are limited to this size before they are rounded to 4 bits */

enum { TLLM_FP16 = 0, TLLM_BF16 = 1, TLLM_FP32 = 2 }; /* activation types */
enum { TLLM_ROTARY_PLAIN = 0, TLLM_ROTARY_LINEAR = 1, TLLM_ROTARY_NTK = 2, TLLM_ROTARY_YARN = 3, TLLM_ROTARY_LLAMA3 = 4 };

/* Frequencies of long contexts.  LINEAR: f / factor.  NTK: base * factor^(rot / (rot - 2)).  YARN: f / factor
 * for pairs that turn less than `low` times over the original length, f for those that turn more than `high`
 * times, a ramp over the pairs between, results times 0.1 ln(factor) + 1.  LLAMA3: the same with a ramp over
 * the turns and without that factor. */
typedef struct tllm_b200_rotary_scaling {
    int type;
    double factor, original, low, high;
} tllm_b200_rotary_scaling;

/* Angles a position of the rot_dim / 2 pairs, and the factor of the result.  On the host. */
int tllm_b200_rotary_frequencies(int rot_dim, double base, const tllm_b200_rotary_scaling* scaling, double* frequencies_host,
                                 float* amplitude_host);
/* The same in turns, as 64-bit fractions: what the kernels multiply with a position.  On the host. */
int tllm_b200_rotary_turns(const double* frequencies_host, int pairs, unsigned long long* turns_host);

typedef struct tllm_b200_rotary_table {
    const unsigned long long* turns; /* device, [rot_dim / 2] */
    int rot_dim;                     /* the first rot_dim entries of a head turn, an even number */
    int half_layout;                 /* pairs (i, i + rot_dim / 2); 0: (2 i, 2 i + 1) */
    float amplitude;
} tllm_b200_rotary_table;

typedef struct tllm_b200_cache4 {
    void *k_codes, *k_params, *v_codes, *v_params;
    int batch, kv_heads, rows, dim; /* dim 64 or 128 */
} tllm_b200_cache4;

/* Activations [tokens, heads, dim]: rows `ld` elements apart. */
typedef struct tllm_b200_heads {
    void* p;
    long long ld;
} tllm_b200_heads;

/* (x1, x2) -> a (x1 cos - x2 sin, x2 cos + x1 sin) with the angles of positions[row]; `inverse` turns the
 * other way (the gradient of this operator).  k and k_out may be NULL (kv_heads 0).  An output may be its
 * own input, else outputs must not overlap anything.  dim: a multiple of 8 (FP32: of 4) up to 512. */
int tllm_b200_rotary(int type, const tllm_b200_rotary_table* table, const int* positions, int tokens, const tllm_b200_heads* q,
                     const tllm_b200_heads* q_out, int heads, const tllm_b200_heads* k, const tllm_b200_heads* k_out, int kv_heads, int dim,
                     int inverse, void* stream);

/* Rotates q into q_out (may be q; both NULL: no queries) and k, rounds both to the activation type, and
 * writes k and v (which are only read) to the cache.  table NULL: nothing turns.  FP16 or BF16.
 * Of 64 values limited to +-61440: l = half(min), s = half((max - l) / 15), c = rint((x - l) / s) within 0..15,
 * 0 where s = 0.  A NaN in a key or a value makes the params of that position's key NaN: rows that see the
 * position become NaN.  NaN values themselves are written as 0. */
int tllm_b200_cache4_append(const tllm_b200_cache4* cache, int type, const tllm_b200_rotary_table* table, const int* first, const int* lens,
                            int tokens, const tllm_b200_heads* q, const tllm_b200_heads* q_out, int heads, const tllm_b200_heads* k,
                            const tllm_b200_heads* v, void* stream);

/* Keys and values at the rows' positions as the cache holds them; k or v may be NULL.  Padding rows: 0. */
int tllm_b200_cache4_read(const tllm_b200_cache4* cache, int type, const int* first, const int* lens, int tokens, const tllm_b200_heads* k,
                          const tllm_b200_heads* v, void* stream);

/* out = softmax(scale q . k) v over the positions up to the row's own, heads / kv_heads query heads to a
 * key/value head.  FP16 or BF16.  max_new: about the most rows of a sequence (0: not known, then as many as
 * they have on the average), which chooses the way of the work, not the result's meaning.  max_len: no sequence
 * holds more positions (0: the cache's rows); lens above it is cut and raises TLLM_ERR_SHAPE as lens above rows
 * does.  workspace: device memory of tllm_b200_cache4_workspace bytes on a 128-byte boundary, for this call
 * alone. */
int tllm_b200_cache4_attention(const tllm_b200_cache4* cache, int type, const int* first, const int* lens, int tokens,
                               const tllm_b200_heads* q, const tllm_b200_heads* out, int heads, float scale, int max_new, int max_len,
                               void* workspace, size_t workspace_bytes, void* stream);
int tllm_b200_cache4_workspace(const tllm_b200_cache4* cache, int tokens, int heads, int max_new, int max_len, size_t* bytes);

#ifdef __cplusplus
}
#endif
#endif /* TLLM_B200_CACHE4_H */
