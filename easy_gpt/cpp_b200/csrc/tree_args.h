/* What the operators of drafted trees are given: blocks of 8-byte fields, so that a caller in another language packs one in one go.  Pointers are to the
 * device's memory. */
#ifndef EASY_GPT_TREE_ARGS_H
#define EASY_GPT_TREE_ARGS_H

/* eg_attention_tree (attention_tree.cu) */
typedef struct eg_attention_tree_args {
    const void* q;                  /* [>= rows, ldq], num_heads * head_dim columns */
    const void* k_cache;            /* [num_pages][num_kv_heads][page_size][head_dim], strides of pages and heads in elements */
    const void* v_cache;            /* the same */
    const int* block_table;         /* [entries, table_pages], row stride table_stride */
    const int* entry_starts;        /* [entries + 1] */
    const int* context;             /* [entries] */
    const int* parents;             /* [rows] */
    void* out;                      /* [>= rows, ldo] */
    int* status;
    long long dtype, ldq, ldo, page_stride, head_stride, table_stride, table_pages, num_pages, rows, entries, num_heads, num_kv_heads, head_dim, page_size;
    long long window;               /* 0: none */
    long long max_context;          /* the most keys an entry has, cached and its own, as far as known: how the work is split follows it */
    long long row_tile, max_parts, part_tiles;      /* a plan (eg_attention_tree_plan); row_tile below 0: made by the call */
    double scale;                   /* above 0 in 32 bits, below 2e38 */
} eg_attention_tree_args;

/* eg_tree_accept (tree_step.cu) */
typedef struct eg_tree_accept_args {
    const int* tokens;              /* [rows] */
    const int* targets;             /* [rows] */
    const int* entry_starts;        /* [entries + 1] */
    const int* parents;             /* [rows] */
    int* path;                      /* [entries, longest] */
    int* accepted;                  /* [entries] */
    int* emitted;                   /* [entries, longest] */
    int* status;
    long long entries, rows, longest;
} eg_tree_accept_args;

/* eg_cache_keep (tree_step.cu) */
typedef struct eg_cache_keep_args {
    void* kv;                       /* [layers][num_pages][2][kv_heads][page_size][head_dim], strides of the first four in elements */
    const int* block_table;         /* [entries, table_pages], row stride table_stride */
    const int* context;             /* [entries] */
    const int* path;                /* [entries, longest] */
    const int* accepted;            /* [entries] */
    int* status;
    long long element_size;         /* 2 or 4 bytes */
    long long layers, num_pages, kv_heads, page_size, head_dim, layer_stride, page_stride, plane_stride, head_stride, table_stride, table_pages, entries, longest;
} eg_cache_keep_args;

#endif
