// fa_decode_stream.h — launch interface of decode attention over a part of the sequences' keys (fa_decode_stream_sm100.cu).
#pragma once
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "../../include/fa_sm120.h"

namespace fa_sm100 {

// One new token of every sequence against an e4m3 cache.  Sequence b of length n sees
//   shared_lens == nullptr   keys [0, sinks) and [n - window, n) (window 0: all);
//   otherwise                keys [min(shared_lens[b], n), n); in the place of O and LSE their states are left, for whoever adds up what the keys before give: own_o
//                            [batch * q_heads][hd] (sums of weighted values) and own_ml [batch * q_heads][2] (maximum in log2 units, sum of weights).
struct StreamArgs {
    const void *q, *k_cache, *v_cache;
    void* o;
    float* lse;
    const int* seq_lens;
    int batch, q_heads, kv_heads, hd, s_max, seq_len;
    int window, sinks;
    float scale, v_descale;
    const float *scale_q_dev, *scale_k_dev, *scale_v_dev;
    const int* block_table;
    int page_size, max_pages, num_pages;
    cudaStream_t stream;
    const int* shared_lens;
    float *own_o, *own_ml;
    void* workspace;        // stream_workspace_bytes() bytes
    uint32_t* arrivals;     // stream_arrivals() words that are zero; the launch leaves them zero
};
// The checks of fa_decode and of what these kernels want besides.
fa_status_t check_stream(fa_ctx_t* ctx, const char* who, const fa_decode_args_t* args, int& s_max);
StreamArgs stream_args(const fa_decode_args_t& g, int s_max);   // of a checked call; window, sinks and what belongs to a prefix are zero
size_t stream_workspace_bytes(const StreamArgs& a);
size_t stream_arrivals(const StreamArgs& a);
cudaError_t launch_stream(const StreamArgs& a);
fa_status_t launch_stream_call(fa_ctx_t* ctx, const char* who, const StreamArgs& a);   // with scratch of the context

int sms_of_current_device();

// Where a kernel of this library leaves the code of a wait that ran out, on the current device.
uint32_t* status_word();

}  // namespace fa_sm100
