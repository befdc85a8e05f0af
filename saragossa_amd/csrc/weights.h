// The weights that cached rows get from queries (kernels_weights.hip) and the eviction by them (kernels_evict.hip): what their launchers take.
#pragma once

#include "skv_internal.h"

namespace skv {

// Queries are those of the cache's last rows; a slot is a (query, head of the kv head's group) pair, slot / gqa its query.
struct WeightsArgs {
    const float *q; // [n_queries][q_heads * head_dim]
    const uint16_t *k_pool;
    const int32_t *table;
    float *weights; // [kv_heads][stride], rows 0 .. len - 1 added to
    long stride;
    int len;
    int n_queries;
    int n_slots; // of a kv head
    float qscale; // log2(e) / sqrt(head_dim or what stands for it)
    int q_vec;    // queries may be read 16 bytes at a time (set by the launcher)
    int rows16;   // len rounded up to whole pages
    // few slots: scores kept, [kv_heads][n_slots][rows16], a split's maxima and sums [kv_heads][n_slots][splits]
    float *scores;
    float *part_m;
    float *part_l;
    int splits;
    // many slots: queries as operands, [kv_heads][tiles of 16 slots][..]; maximum and 1 / sum of each slot, [kv_heads][tiles * 16]; sums of a split
    // of the slots, [sum_splits][kv_heads][rows16]
    uint4 *q_ops;
    float2 *stats;
    float *part_sum;
    int tiles;
    int sum_splits;
    Geom g;
};
// Of the queries of `left` rows behind `before` others as many as one plan_weights takes within 256 MiB of scores (few slots; at least a query's) or
// 128 MiB of operands
size_t weights_at_once(const Geom &g, size_t before, size_t left);
// Fills in how the launches divide their work and returns the scratch bytes they want; place_weights points them at it.
size_t plan_weights(WeightsArgs &a);
void place_weights(WeightsArgs &a, void *scratch);
hipError_t launch_weights(const WeightsArgs &a, hipStream_t s);

struct Mover {
    int row, held; // where it is: in the cache, and in the pools (page * 16 + row of it)
    float weight;
};
struct EvictArgs {
    uint16_t *k_pool;
    uint16_t *v_pool;
    const int32_t *table;
    float *weights; // [kv_heads][stride]
    long stride;
    int len, keep, first, last;
    int32_t *kept; // [kv_heads][keep]: the old row of each new one (null = nowhere, until place_evict)
    // scratch. Up to 16384 rows: where each new row's numbers come from, as `held` below, -1 = it stays, [kv_heads][keep]. More:
    // the rows from `keep` on that stay, in order, [kv_heads][len - keep]; how many weights of a stretch of `per` rows begin
    // with each eleven bits, [kv_heads][stretches][2048] (one stretch: null)
    int32_t *from;
    Mover *moved;
    int32_t *counts;
    int stretches, per;
    bool few; // no more rows can move than the workgroup that chooses moves itself (no scratch)
    Geom g;
};
// Fills in how the launches divide the rows and returns the scratch bytes they want; place_evict points them at it.
size_t plan_evict(EvictArgs &a, bool lists_kept);
void place_evict(EvictArgs &a, void *scratch);
hipError_t launch_evict(const EvictArgs &a, hipStream_t s);

} // namespace skv
