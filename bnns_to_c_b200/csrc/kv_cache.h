// kv_cache.h - the handle of the block-scaled key/value cache, shared by its
// write and read (kv_cache.cu) and the attention (kv_attend.cu).
#pragma once
#include <cuda_runtime.h>

#include "lowbit.h"

struct bnn_kv_cache {
    int device;
    int type;
    int sms;  // of the device
    bnn::lowbit::KvGeo geo;
    void* base;  // one allocation:
    uint8_t *kc, *vc;   // codes of keys, of values
    uint16_t *ks, *vs;  // their scales
    size_t bytes;
};

namespace bnn {
namespace lowbit {
// sets what the attention kernels of such a cache need on the current device
cudaError_t attend_setup(const KvGeo& g);
}  // namespace lowbit
}  // namespace bnn
