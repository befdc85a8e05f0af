// Host side of eviction by attention weight: argument checks, the scratch, and what an eviction leaves of a layer.
#include <algorithm>
#include <cmath>
#include <string>

#include "layer.h"
#include "weights.h"

using namespace skv;

extern "C" {

int32_t skv_attention_weights_device(skv_layer *L, skv_stream stream, const float *q_dev, size_t n_rows, float attn_scalar, float *weights_dev) try {
    if (!L || !q_dev || !weights_dev) return fail(SKV_ERR_DEVICE, "attention weights: pointeur nul");
    if (L->window > 0) return fail(SKV_ERR_CONFIG, "attention weights: couche à fenêtre glissante");
    if (n_rows == 0) return fail(SKV_ERR_DIMENSION, "attention weights attend seq > 0");
    if (n_rows > L->len)
        return fail(SKV_ERR_DIMENSION, "attention weights: " + std::to_string(n_rows) + " requêtes pour " + std::to_string(L->len) + " lignes");
    if (!(attn_scalar == 0.0f || (std::isfinite(attn_scalar) && attn_scalar > 0.0f)))
        return fail(SKV_ERR_CONFIG, "scalaire d'attention invalide: " + std::to_string(attn_scalar));
    if ((reinterpret_cast<uintptr_t>(q_dev) | reinterpret_cast<uintptr_t>(weights_dev)) & 3)
        return fail(SKV_ERR_DIMENSION, "attention weights: pointeur non aligné f32");
    const Geom &g = L->g;
    const uintptr_t q0 = reinterpret_cast<uintptr_t>(q_dev), w0 = reinterpret_cast<uintptr_t>(weights_dev);
    if (q0 < w0 + (size_t)g.kv_heads * L->capacity * sizeof(float) && w0 < q0 + n_rows * (size_t)g.q_heads * g.head_dim * sizeof(float))
        return fail(SKV_ERR_DIMENSION, "attention weights: poids sur les requêtes");
    if (n_rows * (size_t)g.gqa > (size_t)1 << 21) // (the grid of the widest heads' kernel then has 32768 workgroups along its last dimension)
        return fail(SKV_ERR_DIMENSION, "attention weights: trop de requêtes");
    WeightsArgs a{};
    a.k_pool = L->k_pool;
    a.table = L->table_dev;
    a.weights = weights_dev;
    a.stride = (long)L->capacity;
    a.qscale = (1.0f / std::sqrt(attn_scalar > 0.0f ? attn_scalar : (float)g.head_dim)) * 1.4426950408889634f;
    a.g = g;
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    for (size_t first = 0; first < n_rows;) { // queries whose scratch stays within bounds at a time: those of the last rows but the ones behind them
        const size_t len = L->len - (n_rows - first), n = weights_at_once(g, len, n_rows - first);
        a.q = q_dev + first * (size_t)g.q_heads * g.head_dim;
        a.len = (int)(len + n);
        a.n_queries = (int)n;
        a.n_slots = (int)(n * (size_t)g.gqa);
        a.rows16 = (a.len + 15) / 16 * 16;
        StreamScratch::Lease lease;
        void *scratch = nullptr;
        const int32_t rc = stream_scratch(L->ctx, s, plan_weights(a), lease, &scratch, "attention weights");
        if (rc) return rc;
        place_weights(a, scratch);
        SKV_HIP(launch_weights(a, s));
        first += n;
    }
    return SKV_OK;
} catch (...) {
    return skv::fail_exception();
}

int32_t skv_evict_device(skv_layer *L, skv_stream stream, float *weights_dev, size_t keep_rows, size_t first_rows, size_t last_rows,
                         int32_t *kept_dev) try {
    if (!L || !weights_dev) return fail(SKV_ERR_DEVICE, "evict: pointeur nul");
    if (L->window > 0) return fail(SKV_ERR_CONFIG, "evict: couche à fenêtre glissante");
    if (keep_rows == 0) return fail(SKV_ERR_DIMENSION, "evict attend au moins une ligne gardée");
    if (keep_rows > L->len)
        return fail(SKV_ERR_DIMENSION, "evict: " + std::to_string(keep_rows) + " lignes à garder de " + std::to_string(L->len));
    if (first_rows > keep_rows || last_rows > keep_rows - first_rows)
        return fail(SKV_ERR_DIMENSION, "evict: " + std::to_string(first_rows) + " premières et " + std::to_string(last_rows) +
                                           " dernières lignes pour " + std::to_string(keep_rows) + " gardées");
    if ((reinterpret_cast<uintptr_t>(weights_dev) | reinterpret_cast<uintptr_t>(kept_dev)) & 3)
        return fail(SKV_ERR_DIMENSION, "evict: pointeur non aligné");
    const Geom &g = L->g;
    const size_t kvh = (size_t)g.kv_heads;
    const uintptr_t w0 = reinterpret_cast<uintptr_t>(weights_dev), k0 = reinterpret_cast<uintptr_t>(kept_dev);
    if (kept_dev && w0 < k0 + kvh * keep_rows * sizeof(int32_t) && k0 < w0 + kvh * L->capacity * sizeof(float))
        return fail(SKV_ERR_DIMENSION, "evict: lignes gardées sur les poids");
    EvictArgs a{};
    a.k_pool = L->k_pool;
    a.v_pool = L->v_pool;
    a.table = L->table_dev;
    a.weights = weights_dev;
    a.stride = (long)L->capacity;
    a.len = (int)L->len;
    a.keep = (int)keep_rows;
    a.first = (int)first_rows;
    a.last = (int)last_rows;
    a.g = g;
    a.kept = kept_dev;
    StreamScratch::Lease lease;
    void *scratch = nullptr;
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    const size_t need = plan_evict(a, kept_dev != nullptr);
    if (need > 0) {
        const int32_t rc = stream_scratch(L->ctx, s, need, lease, &scratch, "evict");
        if (rc) return rc;
    }
    place_evict(a, scratch);
    const bool leaves = keep_rows < L->len;
    if (leaves) { // (what may fail for want of memory before anything is queued)
        mark_moved(L, 0);
        if (stream_captured(s) && std::find(L->captured_evictions.begin(), L->captured_evictions.end(), keep_rows) == L->captured_evictions.end())
            L->captured_evictions.push_back(keep_rows);
    }
    SKV_HIP(launch_evict(a, s));
    if (leaves) {
        L->written = std::max(L->written, L->len);
        L->len = keep_rows;
        L->evicted = keep_rows;
        mark_moved(L, keep_rows);
    }
    return SKV_OK;
} catch (...) {
    return skv::fail_exception();
}

size_t skv_evicted_rows(const skv_layer *L) { return L ? L->evicted : 0; }

} // extern "C"
