// Internal interface between the C-ABI core (ms_api.cu), the file loader
// (ms_loader.cu) and the operators beside the token loop (ms_ops.cu).  Nothing
// here is exported from the library.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

#include "../../include/mojostream_cuda.h"

// Record a failure in the context's last-error message and return s.
ms_status ms_fail_(ms_ctx* c, ms_status s, const char* msg);
cudaStream_t ms_stream_(ms_ctx* c);
int ms_device_(const ms_ctx* c);
// Device-resident BOS embedding: token id `bos_id` embeds as bos (hidden
// floats, device) instead of its lm_head column.
ms_status ms_model_set_bos_(ms_ctx* c, ms_model* m, const float* bos, int bos_id);
void ms_set_load_stats_(ms_ctx* c, double seconds, uint64_t bytes);
int ms_sm_count_(const ms_ctx* c);
// Device word of the error bits that bounded waits leave for ms_sync.
int* ms_err_word_(ms_ctx* c);
// At least `bytes` of device workspace for one call on `s`: the stream's own, or
// that of the graph which the stream is being captured into (ms_ws.h).
// MS_ERR_STATE in a capture that asks for more than any call before it.
ms_status ms_workspace_(ms_ctx* c, cudaStream_t s, size_t bytes, void** out);
