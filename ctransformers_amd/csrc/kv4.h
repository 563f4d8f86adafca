// Launches of the 4-bit paged KV cache (kernels_kv4.h, kernels_kvpages.h): what the C entry points (include/ctransformers_amd_ops.h) and the engine share.
// All of them are asynchronous on `stream` of the current device and return false, with a message, without having launched anything if an argument is refused.
#pragma once
#include "kernels_kv4.h"
#include "kernels_kvpages.h"

namespace ctamd {

// groups of 32 dims that a head takes (5 and 7 take the room of 6 and 8); 0: not supported
int kv4_groups(int head_dim);
long long kv4_page_bytes(int n_head_kv, int head_dim, int page_tokens);   // 0: not supported
// fills groups and bshift from the head's size and the page's; checks the rest
bool kv4_check(Kv4Cache& c, int page_tokens, const char*& err);
bool kv4_append(Kv4Append& a, int max_rows, hipStream_t stream, const char*& err);
bool kv4_read(Kv4Append& a, int max_rows, hipStream_t stream, const char*& err);
// floats of workspace that kv4_attention wants for these arguments; 0: none
long long kv4_attention_plan(Kv4Attn& a, int max_rows);
bool kv4_attention(Kv4Attn& a, int max_rows, long long ws_floats, hipStream_t stream, const char*& err);
long long kv_pages_ws_ints(const KvPages& a);
bool kv_fork(const KvPages& a, hipStream_t stream, const char*& err);
bool kv_reserve(const KvPages& a, hipStream_t stream, const char*& err);
bool kv_compact(const KvPages& a, hipStream_t stream, const char*& err);

}  // namespace ctamd
