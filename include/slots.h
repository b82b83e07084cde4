/*
 * slots.h -- C ABI of the slot operators in librwkv7_hip.so (gfx950): copies (forks), compaction and freeing of the slots of
 * several cache tensors at once, for states, token shifts, penalty counts and whatever else a served sequence holds.
 *
 * A cache has `layers` layers of slots; a slot's row in a layer is `row_bytes` contiguous bytes.  Indices are int64 on the
 * device.  A negative index leaves its entry out; one past the slots does too and is reported in `status`.
 * Return codes are the WKV7_* codes of wkv7.h.  No call allocates or synchronises; all can be recorded into a HIP graph.
 */
#ifndef RWKV_NEXT_AMD_SLOTS_H
#define RWKV_NEXT_AMD_SLOTS_H

#include <stddef.h>
#include <stdint.h>

#include "wkv7.h"

#ifdef __cplusplus
extern "C" {
#endif

#define SLOTS_MAX_CACHES 16      /* tensors of one call */
#define SLOTS_MAX_PAIRS 1024     /* copies of one call */
#define SLOTS_MAX_COMPACT 8192   /* slots of caches that are compacted */

/* Bit of *status: an index past the slots */
#define SLOTS_STATUS_SLOT 1024

typedef struct slots_cache {
    const void *from;           /* row of layer 0, slot 0 that copies read (slots_copy) */
    void *to;                   /* row of layer 0, slot 0 that is written */
    int64_t from_layer_stride;  /* bytes */
    int64_t from_slot_stride;
    int64_t to_layer_stride;
    int64_t to_slot_stride;
    int64_t row_bytes;
    int64_t layers;
} slots_cache;

/* sizeof(slots_cache) as compiled into the library (bindings check their struct layout against it). */
size_t slots_cache_size(void);

/* to[layer][dst[i]] = from[layer][src[i]] for every layer of every cache and i < n, as if all sources were read before any
 * destination is written (swaps and chains are exact where to == from); of several entries with one destination the last one
 * counts.  from and to are the same tensor or apart.  to_slots and from_slots bound dst and src. */
int slots_copy(const slots_cache *caches, int32_t num_caches, const int64_t *src, const int64_t *dst, int32_t n,
               int64_t from_slots, int64_t to_slots, int32_t *status, void *stream);

/* to[layer][idx[i]] = 0. */
int slots_free(const slots_cache *caches, int32_t num_caches, const int64_t *idx, int32_t n, int64_t slots, int32_t *status,
               void *stream);

/* With k the number of live slots (live[s] != 0): those at k and behind move, in their order, to the free ones before k, in
 * theirs.  where[s] = the slot's place after, -1 for a free one; *count = k.  Rows that nothing moves to are left as they are.
 * where (slots entries) and count (one) may be NULL.  `from` is not used. */
int slots_compact(const slots_cache *caches, int32_t num_caches, const uint8_t *live, int64_t slots, int64_t *where,
                  int32_t *count, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* RWKV_NEXT_AMD_SLOTS_H */
