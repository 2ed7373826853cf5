/*
 * Shared plain-C types of the dranzer-b200 C ABI (dz_host.h, dz_cuda.h).
 * No C++ or CUDA types cross this boundary: plain pointers, sizes and status codes.
 */
#ifndef DZ_TYPES_H
#define DZ_TYPES_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Status codes: 0 or negative. Mapping to the reference's dranzer_status_t
 * (src/include/dranzer.h:30-41): DZ_E_INVALID -> DRANZER_INVALID_ARGUMENT,
 * DZ_E_IO -> DRANZER_IO_ERROR, DZ_E_FORMAT -> DRANZER_FORMAT_ERROR,
 * DZ_E_CHECKSUM -> DRANZER_CHECKSUM_ERROR, DZ_E_NOMEM -> DRANZER_OUT_OF_MEMORY,
 * DZ_E_UNSUPPORTED -> DRANZER_UNSUPPORTED, DZ_E_DEVICE / DZ_E_TIMEOUT ->
 * DRANZER_MODEL_ERROR, DZ_E_NOT_BUNDLE -> DRANZER_FORMAT_ERROR. */
enum {
    DZ_OK = 0,
    DZ_E_INVALID = -1,
    DZ_E_IO = -2,
    DZ_E_FORMAT = -3,
    DZ_E_CHECKSUM = -4,
    DZ_E_NOMEM = -5,
    DZ_E_UNSUPPORTED = -6,
    DZ_E_DEVICE = -7,
    DZ_E_TIMEOUT = -8,
    DZ_E_NOT_BUNDLE = -9
};

/* Quantization granularity, src/include/core/quantize.h:41-56. */
enum { DZ_GRAN_TENSOR = 0, DZ_GRAN_ROW = 1, DZ_GRAN_COLUMN = 2 };

/* Parameter kinds, src/include/core/model_params.h:20-38. */
enum { DZ_KIND_PROJECTION = 0, DZ_KIND_EMBEDDING = 1, DZ_KIND_BIAS = 2, DZ_KIND_NORM = 3 };

/* Element type of the activations of the 4-bit and 8-bit operators (and of the
 * scales of a group-scaled matrix). No counterpart in the reference, which is fp32. */
enum { DZ_TYPE_F32 = 0, DZ_TYPE_F16 = 1, DZ_TYPE_BF16 = 2 };

/* Model shape: the six bundle header dimensions (src/core/bundle.c:452-458)
 * minus the derived parameter count, plus the v3 architecture flags
 * (src/include/core/model_types.h:26-36). */
typedef struct {
    size_t vocab_size;
    size_t embedding_dim;
    size_t num_heads;
    size_t num_layers;
    size_t max_seq_len;
    uint32_t architecture_flags;
} dz_model_desc_t;

/* One parameter tensor in model_param_tensors() order
 * (src/core/model_params.c:39-103). Either `f32` (bits == 0) or `scales` +
 * `packed` in the reference's storage form: codes biased by qmax, packed
 * least-significant bit first at bit offset i*bits of the row-major k x n
 * tensor (src/core/quantize.c:213-270). */
typedef struct {
    uint32_t kind;
    size_t rows;
    size_t cols;
    int bits;
    int granularity;
    const float *scales;
    size_t scale_count;
    const uint8_t *packed;
    size_t packed_size;
    const float *f32;
} dz_tensor_blob_t;

/* A rows x cols (k x n, row-major) matrix of 4-bit codes with one scale per
 * `group` consecutive rows of a column: value(k, n) = scales[k / group][n] *
 * (code(k, n) - 7). `group` is 32, 64 or 128; the last group may be short.
 * Codes 0..14, packed as quantize_pack packs 4-bit codes (code i = k * cols + n
 * at bit offset 4 i, least-significant bit first). scales: [ceil(rows /
 * group)][cols], DZ_TYPE_F32 or DZ_TYPE_F16, finite and >= 0. */
typedef struct {
    size_t rows;
    size_t cols;
    size_t group;
    const uint8_t *packed;
    size_t packed_size;
    const void *scales;
    size_t scale_count;
    int scale_type;
} dz_grouped_blob_t;

/* Ring caches of keys and values in 4 bits for `batch` sequences of one layer:
 * device buffers that the caller owns.
 *   codes  [batch][kv_heads][capacity][head_dim / 2] bytes, element e of a row
 *          in the low half of byte e / 2 when e is even, else in its high half
 *   scales [batch][kv_heads][capacity][head_dim / 64] fp32, one per 64 elements
 * value = scale * (code - 7), the scale of either sign (a NaN marks 64 elements
 * that hold none). head_dim is 64 or 128. Position p of a sequence
 * lives in slot p while p < sinks (the first tokens, which stay), else in slot
 * sinks + (p - sinks) % (capacity - sinks): the newest capacity - sinks later
 * positions are retained. sinks < capacity <= 2^31 - 64. Code buffers start on 16-byte
 * boundaries, scale buffers on 8-byte ones; k and v buffers do not overlap. */
typedef struct {
    int device;
    uint8_t *k_codes;
    uint8_t *v_codes;
    float *k_scales;
    float *v_scales;
    size_t batch;
    size_t kv_heads;
    size_t head_dim;
    size_t capacity;
    size_t sinks;
} dz_kv4_t;

/* How a head's elements pair up for the rotation: (2p, 2p + 1) as the
 * reference does (src/core/transformer.c:24-54), or (p, p + head_dim / 2). */
enum { DZ_ROPE_PAIRS = 0, DZ_ROPE_HALVES = 1 };

/* One call of dz_cuda_kv4_append. Row r = b * n_tokens + j is token j of
 * sequence b; element e of head h of row r is at base[r * stride + h *
 * head_dim + e] (strides in elements, no alignment asked). */
typedef struct {
    int type;              /* DZ_TYPE_* of q, k, v and the outputs */
    size_t q_heads;        /* 0: no queries */
    const void *q, *k, *v;
    size_t q_stride, k_stride, v_stride;
    void *q_out;           /* normed and rotated queries */
    size_t q_out_stride;
    void *k_out, *v_out;   /* the new rows as the cache now holds them, or NULL */
    size_t k_out_stride, v_out_stride;
    const float *q_gain;   /* [head_dim] gains of the norm, or NULL: no norm */
    const float *k_gain;
    double eps;
    double rope_base;      /* 0: no rotation */
    int rope_pairing;      /* DZ_ROPE_* */
} dz_kv4_append_t;

/* One call of dz_cuda_kv4_attention. */
typedef struct {
    int type;              /* DZ_TYPE_* of q and out */
    size_t q_heads;        /* a multiple of kv_heads: q_heads / kv_heads share a key head */
    const void *q;
    size_t q_stride;
    void *out;
    size_t out_stride;
    float scale;           /* scores are scale * (q . k) */
    size_t window;         /* 0: every retained token; else the newest `window` and the sinks */
} dz_kv4_attention_t;

/* One call of dz_cuda_norm_q8: rows of `width` elements, element e of row r at
 * base[r * stride + e] (strides in elements, no alignment asked). */
typedef struct {
    int device;
    int type;                /* DZ_TYPE_* of x, residual and sum_out */
    const void *x;
    size_t x_stride;
    const void *residual;    /* added to x, or NULL */
    size_t residual_stride;
    void *sum_out;           /* x + residual rounded to `type`, or NULL */
    size_t sum_stride;
    const float *gain;       /* [width], or NULL: 1 */
    int norm;                /* 1: the root-mean-square norm, 0: the rows as they are */
    double eps;
    int8_t *codes;           /* row r at codes + r * codes_stride */
    size_t codes_stride;
    float *scales;           /* [rows] */
} dz_norm_q8_t;

/* Keys and values of `batch` sequences of one layer in 8 bits, on a pool of
 * pages that the sequences share: device buffers that the caller owns.
 *   codes  [pages][kv_heads][page][head_dim] int8, -127..127
 *   scales [pages][kv_heads] fp32, one per page and head (a NaN marks a page that
 *          holds no values)
 *   table  [batch][table_pages] int32: the page that holds the tokens [j * page,
 *          (j + 1) * page) of sequence b is table[b * table_pages + j]
 * value = scale * code. `page` is 32 or 64 tokens, head_dim 64 or 128. An entry
 * outside 0..pages-1 names no page: tokens there are neither stored nor seen,
 * nor are those at table_pages * page and after. Several entries may name one
 * page for attention (sequences that share a prefix); an append writes to every
 * page that its new tokens fall in, which then has to be named once. table_pages
 * * page <= 2^31 - 64. Code buffers start on 16-byte boundaries; k and v
 * buffers do not overlap. */
typedef struct {
    int device;
    int8_t *k_codes;
    int8_t *v_codes;
    float *k_scales;
    float *v_scales;
    size_t pages;
    size_t page;
    size_t kv_heads;
    size_t head_dim;
    const int32_t *table;
    size_t batch;
    size_t table_pages;
} dz_kv8_t;

/* One call of dz_cuda_kv8_append: the fields of a 4-bit cache's. */
typedef dz_kv4_append_t dz_kv8_append_t;

/* One call of dz_cuda_kv8_attention. */
typedef struct {
    int type;              /* DZ_TYPE_* of q and out */
    size_t q_heads;        /* a multiple of kv_heads: q_heads / kv_heads share a key head */
    const void *q;
    size_t q_stride;
    void *out;
    size_t out_stride;
    float scale;           /* scores are scale * (q . k) */
    size_t window;         /* 0: every token; else the newest `window` */
    size_t longest;        /* 0, or a hint: about the most tokens that a sequence holds. It
                            * shapes the launch, results hold whatever it is */
} dz_kv8_attention_t;

#ifdef __cplusplus
}
#endif

#endif
