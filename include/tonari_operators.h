/*
 * tonari_operators.h - C ABI of the operators that an atomistic transformer
 * runs next to a neighbor list (libtonari_hip.so, beside tonari_hip.h): rows
 * of a table by species, attention within the structures of a batch, and
 * attention along the pairs of a neighbor list, each with its gradients.
 * They have no counterpart in the reference.
 *
 * The conventions are those of tonari_hip.h: pointers are device pointers,
 * every launch goes on `stream` on the current HIP device, the library
 * allocates nothing, keeps no state and does not wait.  Return codes are
 * TNR_OK, TNR_INPUT_ERROR and TNR_DEVICE_ERROR with a message in `err`.
 *
 * What only the device can see (a species outside the table, a batch_ptr
 * that does not rise from 0 to the number of atoms, a list whose sources do not
 * lie together or that names atoms that do not exist) is not refused, since a call does not
 * wait for the device: the results that it touches are NaN, and no access
 * goes by it.
 *
 * Tensors are contiguous unless a stride is given.  Strides are in elements;
 * q, k and v have contiguous channels, and their addresses and strides are
 * multiples of 16 bytes.
 */
#ifndef TONARI_OPERATORS_H
#define TONARI_OPERATORS_H

#include "tonari_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Version of this header's structs and functions. */
#define TNR_OPERATORS_VERSION 2

/* Types besides TNR_FLOAT32. */
#define TNR_BFLOAT16 2
#define TNR_FLOAT16 3

int tnr_operators_version(void);

/* ------------------------------------------------------------- embedding */

/* out[n] = scale * weight[species[n]] for atoms n, rows of `channels`. */
typedef struct tnr_embedding {
    int32_t dtype;          /* of weight, out and their gradients */
    int32_t index_bytes;    /* 4 or 8: species are int32 or int64 */
    int64_t n_atoms;        /* below 2^31 - 1 */
    int64_t n_species;      /* rows of the table, below 2^24 */
    int64_t channels;       /* up to 2^18 */
    const void* species;    /* [n_atoms]; outside [0, n_species): a row of NaN, no gradient */
    const void* weight;     /* T[n_species][channels] */
    float scale;
    void* out;              /* T[n_atoms][channels] */
    const void* grad_out;   /* backward: T[n_atoms][channels] */
    void* grad_weight;      /* backward: T[n_species][channels], written whole */
} tnr_embedding;

int tnr_embedding_forward(const tnr_embedding* req, void* stream, char* err, size_t err_len);

/* Device scratch of the backward (256-byte aligned). */
size_t tnr_embedding_workspace_size(const tnr_embedding* req);

/* grad_weight[z] = scale * the sum of grad_out over the atoms of species z, in
 * 32 bits and in an order that the inputs alone fix. */
int tnr_embedding_backward(const tnr_embedding* req, void* workspace, size_t workspace_bytes,
                           void* stream, char* err, size_t err_len);

/* --------------------------------------------------- structure attention */

/* Every query atom of a structure attends to all key atoms of the same
 * structure (query_ptr and key_ptr give each structure's rows).  For a query
 * at distance r from a key, with x = scale q.k and u = softcap tanh(x /
 * softcap) (u = x where softcap is 0), the score is u - slopes[head] r; the
 * output is the softmax-weighted sum of the values, and 0 where a structure
 * has no keys.  Query head h reads key and value head h * kv_heads / heads. */
typedef struct tnr_structure_attention {
    int32_t dtype;                  /* of q, k, v, out and their gradients */
    int32_t heads, kv_heads, dim;   /* dim: a multiple of 8, 8 to 128 */
    int64_t n_structures, n_queries, n_keys;  /* below 2^30 (backward: together below
                                                 1.4 * 10^9); rows of all heads below 2^31 */
    const int64_t* query_ptr;       /* [n_structures + 1] */
    const int64_t* key_ptr;         /* [n_structures + 1] (may be query_ptr) */
    const void* q;                  /* T[n_queries][heads][dim] */
    const void* k;                  /* T[n_keys][kv_heads][dim] */
    const void* v;
    int64_t q_stride[2], k_stride[2], v_stride[2];  /* atom, head */
    const float* query_positions;   /* [n_queries][3]; NULL: the queries are the keys' atoms, at
                                       positions (n_queries == n_keys), or there are none */
    const float* positions;         /* [n_keys][3] */
    const float* slopes;            /* [heads] */
    float scale, softcap;
    void* tiles;                    /* tnr_structure_tiles_size() bytes, 256-byte aligned: the batch
                                       as the forward cuts it up; the backward reads it */
    void* out;                      /* T[n_queries][heads][dim] */
    float* out32;                   /* the same in 32 bits for the backward; NULL: not wanted
                                       (with TNR_FLOAT32 the backward reads out) */
    float* lse;                     /* [heads][n_queries]: what the backward needs; NULL: not wanted */
    /* backward: tiles, out, out32 and lse of the forward, and */
    const void* grad_out;           /* T[n_queries][heads][dim] */
    void* grad_q;                   /* contiguous, like q, k and v; written whole */
    void* grad_k;
    void* grad_v;
    float* grad_query_positions;    /* NULL: not wanted */
    float* grad_positions;          /* NULL: not wanted; holds the queries' share too where
                                       query_positions is NULL */
    float* grad_slopes;             /* [heads]; NULL: not wanted */
} tnr_structure_attention;

size_t tnr_structure_tiles_size(const tnr_structure_attention* req);
size_t tnr_structure_forward_workspace_size(const tnr_structure_attention* req);
int tnr_structure_forward(const tnr_structure_attention* req, void* workspace,
                          size_t workspace_bytes, void* stream, char* err, size_t err_len);
size_t tnr_structure_backward_workspace_size(const tnr_structure_attention* req);
int tnr_structure_backward(const tnr_structure_attention* req, void* workspace,
                           size_t workspace_bytes, void* stream, char* err, size_t err_len);

/* ---------------------------------------------------- neighbor attention */

/* A neighbor list laid out for neighbor attention.  `rows` holds
 * tnr_neighbor_rows_size() bytes written by tnr_neighbor_rows; rows of a list of
 * other sizes give NaN.  The first 32-bit word is 0 for a valid list. */
typedef struct tnr_neighbor_list {
    int64_t n_pairs;                        /* up to 2^31 - 4097 */
    int64_t n_sources, n_targets;           /* up to 2^26 - 4 */
    const int64_t* sources;                 /* i: int64[n_pairs], those of an atom together */
    const int64_t* targets;                 /* j: int64[n_pairs] */
    int32_t transpose;                      /* 1: also by target, which the backward needs */
    void* rows;
} tnr_neighbor_list;

size_t tnr_neighbor_rows_size(const tnr_neighbor_list* list);
size_t tnr_neighbor_rows_workspace_size(const tnr_neighbor_list* list);
int tnr_neighbor_rows(const tnr_neighbor_list* list, void* workspace, size_t workspace_bytes,
                      void* stream, char* err, size_t err_len);

/* Attention of each source atom over its pairs in the list, scores as in
 * structure attention with the pair's distance d for r.  A source without
 * pairs gives 0. */
typedef struct tnr_neighbor_attention {
    int32_t dtype;
    int32_t heads, kv_heads, dim;   /* dim: a multiple of 8, 8 to 128 */
    tnr_neighbor_list list;         /* sources and targets are not read */
    const void* q;                  /* T[n_sources][heads][dim] */
    const void* k;                  /* T[n_targets][kv_heads][dim] */
    const void* v;
    int64_t q_stride[2], k_stride[2], v_stride[2];
    const float* distances;         /* d: [n_pairs] */
    const float* slopes;            /* [heads] */
    float scale, softcap;
    void* out;                      /* T[n_sources][heads][dim] */
    float* out32;                   /* the same in 32 bits for the backward; NULL: not wanted
                                       (with TNR_FLOAT32 the backward reads out) */
    float* lse;                     /* [n_sources][heads]; NULL: not wanted */
    const void* grad_out;           /* T[n_sources][heads][dim] */
    void* grad_q;                   /* contiguous; written whole */
    void* grad_k;
    void* grad_v;
    float* grad_distances;          /* [n_pairs] */
    float* grad_slopes;             /* [heads] */
} tnr_neighbor_attention;

int tnr_neighbor_forward(const tnr_neighbor_attention* req, void* stream, char* err,
                         size_t err_len);
size_t tnr_neighbor_backward_workspace_size(const tnr_neighbor_attention* req);
int tnr_neighbor_backward(const tnr_neighbor_attention* req, void* workspace,
                          size_t workspace_bytes, void* stream, char* err, size_t err_len);

#ifdef __cplusplus
}
#endif

#endif /* TONARI_OPERATORS_H */
