// Internal (C++) launchers of the rotary and key/value-cache operators.
// Arguments are validated by kv_abi.hip before any of these is called.
#pragma once
#include <cmath>

#include "q4k_launch.hpp"

namespace mgq {

struct KvView;

hipError_t rope_table_launch(float *table, int n_pos, int first, int rot_dim, const mgq_rope_scaling &s,
                             hipStream_t stream);
hipError_t rope_launch(const float *x, float *y, const int *pos, const mgq_rope &r, int n_tokens, int heads, int dim,
                       int64_t x_stride, int64_t y_stride, hipStream_t stream);

hipError_t rope_axes_launch(const float *x, float *y, const mgq_rope_axes &axes, const mgq_rope &r, int n_tokens,
                            int heads, int dim, int64_t x_stride, int64_t y_stride, hipStream_t stream);
// How the kernels see several axes (kv_rope.hip); all of it checked.
struct RopeMany;
RopeMany rope_many(const mgq_rope &r, const mgq_rope_axes &axes);

// k and v rows `kv_stride` floats apart; rope null: stored as they come; q
// null: no queries. Queries are rotated from q to q_out.
struct KvAppend {
    const float *k, *v;
    int64_t kv_stride;
    const float *q;
    float *q_out;
    int64_t q_stride, q_out_stride;
    int hq;
};
hipError_t kv_append_launch(const KvView &c, int dim, int fmt, const mgq_rope *rope, const mgq_rope_axes *axes,
                            const KvAppend &a, hipStream_t stream);
hipError_t kv_dequant_launch(const KvView &c, int dim, int fmt, const int *pages, int n, float *k_out, float *v_out,
                             hipStream_t stream);

struct KvAttn {
    const float *q;
    void *out;
    int64_t q_stride, out_stride;
    int hq, out_f16;
    float scale, softcap;
    int window, sinks;
    float *ws;
    int shared_tokens;  // 0: no shared prefix
};
// Whether this many query rows of a kv head take kv_attn_wide.hip.
bool kv_attn_is_wide(int dim, int64_t rows);
size_t kv_attn_workspace(int dim, int hq, int hkv, int n_seqs, int max_new, int64_t capacity);
size_t kv_attn_shared_workspace(int dim, int fmt, int hq, int hkv, int n_seqs, int n_tokens, int max_new, int64_t capacity,
                                int shared_tokens);
// Whether one launch counts the join of a call that reads every sequence by itself.
bool kv_attn_join_fits(int dim, int group, int hkv, int n_seqs, int max_new, int64_t capacity, int window, int sinks);
// How a call behind a shared prefix is gone about: mgq_kv_shared_plan.
typedef mgq_kv_shared_plan SharedPlan;
SharedPlan kv_attn_shared_plan(int dim, int fmt, int out_f16, int hq, int hkv, int n_seqs, int n_tokens, int max_new,
                               int64_t capacity, int shared_tokens);
hipError_t kv_attn_launch(const KvView &c, int dim, int fmt, const KvAttn &a, hipStream_t stream);

}  // namespace mgq
