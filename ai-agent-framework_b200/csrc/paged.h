// Kernels of a paged serving step: block tables and slot maps (page_plan.cu),
// rotary positions and cache writes (rope.cu), attention over the paged cache
// (attention_paged.cu), log probabilities (logprobs.cu).  Each launch_*
// function works on `s` and returns a B2_* code; the exported entry points
// check the arguments first.
#pragma once
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include <string>

#include "../../include/b2decode.h"

namespace b2 {

constexpr int kPlanMaxReq = 16384;   // requests of one b2_page_plan (its prefix sums live in shared memory)
constexpr int kLogprobMaxTop = 64;   // alternatives of one b2_logprobs row
constexpr int kPagedMaxHd = 256;     // head dimension of the paged cache

struct PagePlanArgs {
    const int32_t* cached;     // [n_req]
    const int32_t* fresh;      // [n_req]
    const int32_t* free_pages; // [*n_free]
    const int32_t* n_free;
    int32_t* table;            // [n_req][table_stride]
    int64_t table_stride;
    int32_t* lens;             // [n_req]
    int32_t* starts;           // [n_req + 1]
    int64_t* slots;            // [max_tokens]
    int32_t* positions;        // [max_tokens]
    int32_t* token_req;        // [max_tokens]
    int32_t* info;             // [4]
    int32_t n_req, page_size, max_pages, max_tokens;
    // set by launch_page_plan: division by the page size
    uint32_t page_mul;
    int32_t page_shift;
};

int launch_page_plan(const PagePlanArgs& a, cudaStream_t s, std::string* err);

// k_out null: k and v go to the cache at slots; kv null: k goes to k_out.
int launch_rope(const b2_rope_rows& d, const b2_paged_kv* kv, const double* freqs, const int32_t* positions,
                const int64_t* slots, int n_tok, const void* q, const void* k, const void* v, void* q_out, void* k_out,
                cudaStream_t s, std::string* err);

size_t attention_paged_scratch(int batch, int nh, int nkv, int hd, int sms);
int launch_attention_paged(const b2_paged_kv& kv, const b2_paged_attn_opts& o, const void* q, const int32_t* table,
                           const int32_t* lens, const int32_t* req, int batch, void* out, float* lse, void* scratch,
                           cudaStream_t s, std::string* err);

int launch_logprobs(const void* logits, int dtype, int n, int rows, int64_t ld, const int32_t* ids, int m,
                    float* logprob, float* entropy, int k, int32_t* top_ids, float* top_logprob, cudaStream_t s,
                    std::string* err);

// The current device's SM count, looked up once per device; 0 without one.
int current_sms(std::string* err);

// A pointer argument: its name in messages and its alignment (a power of two).
struct DevicePtr {
    const char* name;
    const void* p;
    size_t align;
};
// B2_OK when every pointer is null or on its alignment; B2_ERR_BAD_ARG
// otherwise.
int check_alignment(const DevicePtr* p, int n, std::string* err);
// B2_OK when every pointer is null or memory that kernels on the current
// device may address (its own, or managed); B2_ERR_BAD_ARG otherwise, for host
// memory and another device's among them.
int check_device_pointers(const DevicePtr* p, int n, std::string* err);

// The message of a failed CUDA call; returns B2_ERR_CUDA.
int cuda_failed(const char* what, cudaError_t e, std::string* err);

}  // namespace b2
