// Kernels of a paged serving step: block tables and slot maps (page_plan.cu),
// rotary positions and cache writes (rope.cu), attention over the paged cache
// (attention_paged.cu), log probabilities (logprobs.cu); and of a beam search
// over that cache: choice and reordering (beam.cu), pages that rows share
// (page_pool.cu), attention of shared prefixes (attention_shared.cu).  Each launch_*
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
constexpr int kBeamMaxWidth = 64;    // beams of a request

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

size_t beam_select_scratch(int n, int rows, int k);
int launch_beam_select(const void* logits, int dtype, int n, int n_groups, int width, int64_t ld, const float* scores,
                       int k, int eos, int32_t* parent, int32_t* token, float* score, float* eos_score, void* scratch,
                       cudaStream_t s, std::string* err);
int launch_beam_reorder(const void* src, int n_src, int64_t src_stride, void* dst, int n_dst, int64_t dst_stride,
                        int64_t words, const int32_t* parent, const int32_t* lens, const int32_t* token,
                        int32_t* new_lens, cudaStream_t s, std::string* err);

struct PageForkArgs {
    const int32_t* parent;      // [n_req]
    const int32_t* table;       // [n_src][table_stride]
    const int32_t* lens;        // [n_src]
    const int32_t* refs;        // [n_pages] or null
    const int32_t* free_pages;  // [*n_free]
    const int32_t* n_free;
    int32_t* new_table;         // [n_req][new_stride]
    int32_t* new_lens;          // [n_req]
    int32_t* pairs;             // [n_req][3]
    int32_t* info;              // [4]
    int64_t table_stride, new_stride;
    int32_t n_req, n_src, page_size, n_pages, max_pages;
};
int launch_page_fork(const PageForkArgs& a, cudaStream_t s, std::string* err);
int launch_page_copy(const b2_paged_kv& kv, int layers, int64_t layer_stride, const int32_t* pairs, const int32_t* n_pairs,
                     int max_pairs, cudaStream_t s, std::string* err);
size_t page_pool_scratch(int n_pages);
int launch_page_pool(const int32_t* table, int64_t table_stride, const int32_t* lens, int n_req, int page_size,
                     int max_pages, int32_t* refs, int n_pages, int32_t* free_pages, int32_t* n_free, void* scratch,
                     cudaStream_t s, std::string* err);
size_t page_compact_scratch(int n_pages);
int launch_page_compact(int32_t* table, int64_t table_stride, const int32_t* lens, int n_req, int page_size,
                        int max_pages, const int32_t* refs, int n_pages, int32_t* pairs, int max_pairs, int32_t* info,
                        void* scratch, cudaStream_t s, std::string* err);

size_t attention_shared_scratch(int batch, int nh, int nkv, int hd, int sms);
int launch_attention_shared(const b2_paged_kv& kv, const b2_paged_attn_opts& o, const void* q, const int32_t* table,
                            const int32_t* lens, const int32_t* req, int batch, const int32_t* starts,
                            const int32_t* prefix, int n_groups, void* out, float* lse, void* scratch, cudaStream_t s,
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
