// dcn_token_api.cu -- the token operators' entry points of include/dcn_b200.h: their checks, then
// one launcher each.  Launches are asynchronous on the caller's stream; nothing here allocates
// device memory or reads it.
#include "dcn_tokens.cuh"

using namespace dcn;

namespace {

constexpr int64_t kMaxStride = int64_t{1} << 40;  // elements; offsets inside an allocation then fit 63 bits
constexpr int32_t kMaxHeads = 4096;  // of one tensor

size_t element_bytes(int dtype) { return dtype == DCN_DTYPE_F32 ? 4 : 2; }

bool valid_dtype(int dtype) {
    return dtype == DCN_DTYPE_F32 || dtype == DCN_DTYPE_F16 || dtype == DCN_DTYPE_BF16;
}

bool aligned_to(const void *p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

bool valid_stride(int64_t s) { return s >= 0 && s < kMaxStride; }

// A null or misaligned tensor, or a stride out of range.
dcn_status check_heads(const dcn_heads *h, int dtype) {
    if (h == nullptr || h->data == nullptr || !aligned_to(h->data, element_bytes(dtype)) ||
        !valid_stride(h->token_stride) || !valid_stride(h->head_stride))
        return DCN_ERR_INVALID_ARGUMENT;
    return DCN_OK;
}

dcn_status check_rotation(const dcn_rotation *r, int32_t head_dim) {
    if (r == nullptr) return DCN_ERR_INVALID_ARGUMENT;
    int64_t pairs = 0;
    for (int32_t n : r->pairs) {
        if (n < 0) return DCN_ERR_INVALID_SHAPE;
        pairs += n;
    }
    if (2 * pairs > head_dim) return DCN_ERR_INVALID_SHAPE;
    if (r->interleaved != 0 && r->interleaved != 1) return DCN_ERR_INVALID_ARGUMENT;
    if (pairs > 0 && (r->frequencies == nullptr || r->positions == nullptr || !aligned_to(r->frequencies, 8) ||
                      !aligned_to(r->positions, 4)))
        return DCN_ERR_INVALID_ARGUMENT;
    return DCN_OK;
}

dcn_status check_cache(const dcn_paged_cache *c) {
    if (c == nullptr || !valid_dtype(c->dtype) || c->reserved != 0) return DCN_ERR_INVALID_ARGUMENT;
    if (c->pages <= 0 || c->page_size <= 0 || c->heads <= 0 || c->heads > kMaxHeads || c->head_dim <= 0 ||
        c->streams < 0 || c->streams > 65535 || c->table_columns < 0)
        return DCN_ERR_INVALID_SHAPE;
    const int64_t strides[] = {c->key_page_stride,   c->key_slot_stride,   c->key_head_stride,  c->value_page_stride,
                               c->value_slot_stride, c->value_head_stride, c->table_stride};
    for (int64_t s : strides)
        if (!valid_stride(s)) return DCN_ERR_INVALID_ARGUMENT;
    if (c->keys == nullptr || c->values == nullptr || !aligned_to(c->keys, element_bytes(c->dtype)) ||
        !aligned_to(c->values, element_bytes(c->dtype)))
        return DCN_ERR_INVALID_ARGUMENT;
    if (c->starts == nullptr || !aligned_to(c->starts, 4)) return DCN_ERR_INVALID_ARGUMENT;
    if (c->streams > 0 && (c->lengths == nullptr || !aligned_to(c->lengths, 4) ||
                           (c->table_columns > 0 && (c->table == nullptr || !aligned_to(c->table, 4)))))
        return DCN_ERR_INVALID_ARGUMENT;
    return DCN_OK;
}

dcn_status check_attention(const dcn_paged_cache *c, const dcn_token_attention_args *a) {
    dcn_status st = check_cache(c);
    if (st != DCN_OK) return st;
    if (a == nullptr || a->reserved != 0) return DCN_ERR_INVALID_ARGUMENT;
    if (a->tokens < 0 || a->tokens >= (int64_t{1} << 31) || a->q_heads <= 0 || a->q_heads > kMaxHeads || a->q_heads % c->heads != 0 ||
        a->tokens * a->q_heads >= (int64_t{1} << 31) || a->max_q < 0 || a->max_kv < 0)
        return DCN_ERR_INVALID_SHAPE;
    if (a->window < 1 || a->sinks < 0 || a->frame < 1 || !(a->scale == a->scale)) return DCN_ERR_INVALID_ARGUMENT;
    if (c->head_dim > 256) return DCN_ERR_UNSUPPORTED;
    return DCN_OK;
}

// Whether a 16-bit tensor's rows start on 16 bytes.
bool packs(const dcn_heads &h) {
    return aligned_to(h.data, 16) && h.token_stride % 8 == 0 && h.head_stride % 8 == 0;
}

HeadCopy copy_of(const dcn_heads &src, const dcn_heads &dst, int32_t heads, bool rotate) {
    HeadCopy c{};
    c.src = src.data;
    c.dst = dst.data;
    c.src_token = src.token_stride;
    c.src_head = src.head_stride;
    c.dst_token = dst.token_stride;
    c.dst_head = dst.head_stride;
    c.heads = heads;
    c.rotate = rotate;
    return c;
}

}  // namespace

extern "C" {

dcn_status dcn_token_rotary(dcn_dtype dtype, int64_t tokens, int32_t heads, int32_t head_dim,
                            const dcn_rotation *rotation, const dcn_heads *x, const dcn_heads *out,
                            dcn_stream stream) {
    if (!valid_dtype(dtype)) return DCN_ERR_INVALID_ARGUMENT;
    if (tokens < 0 || tokens >= (int64_t{1} << 31) || heads <= 0 || heads > kMaxHeads || head_dim <= 0 ||
        head_dim % 2 != 0)
        return DCN_ERR_INVALID_SHAPE;
    if (head_dim > 512) return DCN_ERR_UNSUPPORTED;
    if (tokens == 0) return DCN_OK;
    dcn_status st = check_rotation(rotation, head_dim);
    if (st == DCN_OK) st = check_heads(x, dtype);
    if (st == DCN_OK) st = check_heads(out, dtype);
    if (st != DCN_OK) return st;
    LaunchDevice dev;
    if ((st = launch_device(&dev)) != DCN_OK) return st;
    RotateParams p{};
    p.part[0] = copy_of(*x, *out, heads, true);
    p.parts = 1;
    p.head_dim = head_dim;
    p.tokens = tokens;
    p.rotation = *rotation;
    return status_from_cuda(launch_token_rotate(dtype, p, dev.err_word, reinterpret_cast<cudaStream_t>(stream)));
}

dcn_status dcn_token_append(const dcn_paged_cache *cache, int64_t tokens, const dcn_rotation *rotation,
                            const dcn_heads *keys, const dcn_heads *values, int32_t q_heads, const dcn_heads *q,
                            const dcn_heads *q_out, dcn_stream stream) {
    dcn_status st = check_cache(cache);
    if (st != DCN_OK) return st;
    if (tokens < 0 || tokens >= (int64_t{1} << 31) || q_heads < 0 || q_heads > kMaxHeads) return DCN_ERR_INVALID_SHAPE;
    if (cache->head_dim > 512) return DCN_ERR_UNSUPPORTED;
    if (tokens == 0) return DCN_OK;
    if (rotation != nullptr && (st = check_rotation(rotation, cache->head_dim)) != DCN_OK) return st;
    if ((st = check_heads(keys, cache->dtype)) != DCN_OK) return st;
    if ((st = check_heads(values, cache->dtype)) != DCN_OK) return st;
    if (q_heads > 0) {
        if ((st = check_heads(q, cache->dtype)) != DCN_OK) return st;
        if ((st = check_heads(q_out, cache->dtype)) != DCN_OK) return st;
    }
    LaunchDevice dev;
    if ((st = launch_device(&dev)) != DCN_OK) return st;
    RotateParams p{};
    const bool rotate = rotation != nullptr;
    if (rotate) p.rotation = *rotation;
    const dcn_heads key_pages{cache->keys, 0, cache->key_head_stride};
    const dcn_heads value_pages{cache->values, 0, cache->value_head_stride};
    HeadCopy k = copy_of(*keys, key_pages, cache->heads, rotate);
    k.to_cache = true;
    k.dst_page = cache->key_page_stride;
    k.dst_slot = cache->key_slot_stride;
    HeadCopy v = copy_of(*values, value_pages, cache->heads, false);
    v.to_cache = true;
    v.dst_page = cache->value_page_stride;
    v.dst_slot = cache->value_slot_stride;
    if (q_heads > 0) p.part[p.parts++] = copy_of(*q, *q_out, q_heads, rotate);
    if (cache->streams > 0) {
        p.part[p.parts++] = k;
        p.part[p.parts++] = v;
    }
    if (p.parts == 0) return DCN_OK;
    p.head_dim = cache->head_dim;
    p.tokens = tokens;
    p.table = cache->table;
    p.starts = cache->starts;
    p.lengths = cache->lengths;
    p.table_stride = cache->table_stride;
    p.streams = cache->streams;
    p.table_columns = cache->table_columns;
    p.pages = cache->pages;
    p.page_size = cache->page_size;
    return status_from_cuda(launch_token_rotate(static_cast<dcn_dtype>(cache->dtype), p, dev.err_word,
                                                reinterpret_cast<cudaStream_t>(stream)));
}

size_t dcn_token_attention_workspace_bytes(const dcn_paged_cache *cache, const dcn_token_attention_args *args) {
    if (check_attention(cache, args) != DCN_OK || !token_attention_tensor(*cache, *args)) return 0;
    return token_attention_tensor_workspace(*cache, *args);
}

dcn_status dcn_token_attention(const dcn_paged_cache *cache, const dcn_token_attention_args *args, const dcn_heads *q,
                               const dcn_heads *out, void *workspace, size_t workspace_bytes, dcn_stream stream) {
    dcn_status st = check_attention(cache, args);
    if (st != DCN_OK) return st;
    if (args->tokens == 0 || cache->streams == 0) return DCN_OK;
    if ((st = check_heads(q, cache->dtype)) != DCN_OK) return st;
    if ((st = check_heads(out, cache->dtype)) != DCN_OK) return st;
    const size_t need = dcn_token_attention_workspace_bytes(cache, args);
    if (need > 0 && (workspace == nullptr || !aligned_to(workspace, 16) || workspace_bytes < need))
        return DCN_ERR_INVALID_ARGUMENT;
    const bool tensor = token_attention_tensor(*cache, *args) && packs(*q) && packs(*out);
    LaunchDevice dev;
    if ((st = launch_device(&dev, tensor ? KernelSet::kTokenAttention : KernelSet::kNone)) != DCN_OK) return st;
    AttentionParams p{*cache, *args, *q, *out};
    if (tensor)
        return status_from_cuda(launch_token_attention_tensor(p, workspace, dev.sm_count, dev.err_word,
                                                              reinterpret_cast<cudaStream_t>(stream)));
    return status_from_cuda(launch_token_attention_direct(p, reinterpret_cast<cudaStream_t>(stream)));
}

dcn_status dcn_token_norm(const dcn_token_norm_args *args, dcn_stream stream) {
    if (args == nullptr || !valid_dtype(args->dtype)) return DCN_ERR_INVALID_ARGUMENT;
    const dcn_token_norm_args &a = *args;
    if (a.rows < 0 || a.rows >= (int64_t{1} << 31) || a.width <= 0 || a.group <= 0) return DCN_ERR_INVALID_SHAPE;
    if (a.width > 8192) return DCN_ERR_UNSUPPORTED;
    if ((a.kind != DCN_NORM_RMS && a.kind != DCN_NORM_LAYER) || (a.post != 0 && a.post != 1) ||
        !(a.epsilon >= 0.0f) || !(a.residual_scale == a.residual_scale))
        return DCN_ERR_INVALID_ARGUMENT;
    if (a.rows == 0) return DCN_OK;
    if (a.x == nullptr || (a.hidden == nullptr && a.out == nullptr)) return DCN_ERR_INVALID_ARGUMENT;
    if (a.residual == nullptr && (a.post != 0 || a.gate != nullptr || a.hidden != nullptr))
        return DCN_ERR_INVALID_ARGUMENT;
    if (a.post == 0 && (a.post_weight != nullptr || a.post_bias != nullptr)) return DCN_ERR_INVALID_ARGUMENT;
    const void *pointers[] = {a.x, a.residual, a.post_weight, a.post_bias, a.weight, a.bias,
                              a.gate, a.scale, a.shift, a.hidden, a.out};
    for (const void *p : pointers)
        if (!aligned_to(p, element_bytes(a.dtype))) return DCN_ERR_INVALID_ARGUMENT;
    const int64_t strides[] = {a.x_stride, a.residual_stride, a.hidden_stride, a.out_stride,
                               a.gate_stride, a.scale_stride, a.shift_stride};
    for (int64_t s : strides)
        if (!valid_stride(s)) return DCN_ERR_INVALID_ARGUMENT;
    LaunchDevice dev;
    const dcn_status st = launch_device(&dev, KernelSet::kTokenNorm);
    if (st != DCN_OK) return st;
    return status_from_cuda(launch_token_norm(a, dev.err_word, reinterpret_cast<cudaStream_t>(stream)));
}

}  // extern "C"
