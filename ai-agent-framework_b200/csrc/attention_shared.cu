// Attention of rows that share a prefix of a paged KV cache.
#include <cuda_runtime.h>

#include "paged.h"

namespace b2 {

size_t attention_shared_scratch(int batch, int nh, int nkv, int hd, int sms) {
    return attention_paged_scratch(batch, nh, nkv, hd, sms);
}

int launch_attention_shared(const b2_paged_kv& kv, const b2_paged_attn_opts& o, const void* q, const int32_t* table,
                            const int32_t* lens, const int32_t* req, int batch, const int32_t* starts,
                            const int32_t* prefix, int n_groups, void* out, float* lse, void* scratch, cudaStream_t s,
                            std::string* err) {
    (void)starts, (void)prefix, (void)n_groups;
    return launch_attention_paged(kv, o, q, table, lens, req, batch, out, lse, scratch, s, err);
}

}  // namespace b2
