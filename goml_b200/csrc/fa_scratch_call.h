// fa_scratch_call.h — what entry points of libfa_sm120.so that lie outside fa_api.cu use of a context: its message, its device and its scratch.
#pragma once
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "../../include/fa_sm120.h"

namespace fa_sm100 {

// Scratch of one call: `workspace` is written before it is read; `zeros` are words that the call finds zero and leaves zero.
struct CallScratch {
    void* workspace;
    uint32_t* zeros;
};

// Leaves "<who>: <text>" as the context's message and returns `status`.
fa_status_t refuse(fa_ctx_t* ctx, const char* who, fa_status_t status, const char* text);
// FA_OK where the context serves this GPU and its device is the calling thread's current one.
fa_status_t usable(fa_ctx_t* ctx, const char* who);
// The checks of a decode call over an e4m3 cache: FA_OK, and the keys that a sequence's row of the cache or of the table holds; q must be aligned to q_align bytes.
fa_status_t check_decode(fa_ctx_t* ctx, const char* who, const fa_decode_args_t* args, int q_align, int& s_max);
// On the current device, what calls keep between them is as a first call finds it: behind a wait that ran out.
void clear_kept_words();
// Takes the scratch, calls launch(args, scratch), which queues the call's kernels on `stream`, and gives the scratch back behind them.
fa_status_t call_with_scratch(fa_ctx_t* ctx, const char* who, cudaStream_t stream, size_t workspace_bytes, size_t zero_words,
                              cudaError_t (*launch)(const void* args, const CallScratch& scratch), const void* args);

}  // namespace fa_sm100
