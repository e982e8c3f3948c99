// The paged cache as its kernels see it (kvpool.cu) and as the attention that reads it does (treeattn.cu).
#pragma once

#include <memory>

#include "common.cuh"

namespace lokal {

struct PoolArgs {
    int32_t* table;  // [n_slots][max_pages]
    int32_t* lens;   // [n_slots]
    int32_t* refs;   // [n_pages]
    void** stores;   // device array of n_stores base addresses
    int* work;       // scratch of the plans
    unsigned* err_word;
    unsigned page_rows, page_shift, n_pages, n_slots, max_pages, n_stores;
    size_t row_bytes;
};

}  // namespace lokal

struct lokal_kv_pool {
    int device = 0;
    bool vec16 = false;  // rows and stores allow 16-byte accesses
    void* block = nullptr;
    std::unique_ptr<void*[]> stores;  // the same addresses, for the host
    lokal::PoolArgs a{};
};
