// kv_cache.h - the handle of the block-scaled key/value cache, shared by its
// write and read (kv_cache.cu) and the attention (kv_attend.cu).
#pragma once
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
