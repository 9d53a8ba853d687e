// kv_cache.h -- the F16 KV cache handle (NewKVCacheF16 model.go:1396).
#pragma once

#include <stdint.h>

struct gllm_hip_kv {
    int layers, kv_dim_k, kv_dim_v, max_len;
    uint16_t** k;  // host array of device pointers
    uint16_t** v;
    int device;
};
