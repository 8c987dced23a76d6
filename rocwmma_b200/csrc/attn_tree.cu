// Attention of drafted tokens over a paged cache: the entry point b200wmma_attn_tree.
#include "attn_common.cuh"

namespace b200wmma
{
    namespace attn_tree
    {
        using attn::from_f32;
        using attn::LOG2E;
        using attn::tanh_of;
        using attn::to_f32;
        constexpr uint32_t CHUNK      = 128;
        constexpr uint32_t MAX_DRAFTS = 64;

        struct Params
        {
            uint32_t batch, heads_q, heads_kv, dim, drafts, num_pages, page_size, ld_table;
            float    scale, cap;
            const float*    slopes;
            const int32_t * block_table, *lens, *n_drafts, *depths;
            const uint64_t* tree;
            attn::Strides   q, k, v, o;
        };

        // One block to a drafted token of one head: 128 scores at a time, then each thread adds up one column of o.
        template <typename T>
        __global__ void __launch_bounds__(CHUNK) tree_kernel(const Params p, const T* q, const T* k, const T* v, T* o)
        {
            __shared__ float   w[CHUNK], buf[8];
            __shared__ int64_t rows[CHUNK];
            const uint32_t     d = blockIdx.x % p.drafts, h = blockIdx.x / p.drafts % p.heads_q, b = blockIdx.x / p.drafts / p.heads_q;
            const uint32_t     g = h / (p.heads_q / p.heads_kv), t = threadIdx.x;
            const int64_t      cap_tokens = int64_t(p.ld_table) * p.page_size;
            const int64_t      len        = max(p.lens[b], 0);
            const uint32_t     n_drafts   = p.n_drafts ? min(uint32_t(max(p.n_drafts[b], 0)), p.drafts) : p.drafts;
            if(d >= n_drafts)
                return;
            const int64_t  end  = min(len + n_drafts, cap_tokens);
            const uint64_t bits = p.tree ? p.tree[size_t(b) * p.drafts + d] : (uint64_t(2) << d) - 1;
            const int64_t  at   = len + (p.depths ? p.depths[size_t(b) * p.drafts + d] : int32_t(d));
            const float    slope = p.slopes ? p.slopes[h] : 0.0f;
            const T*       qr    = q + b * p.q.batch + d * p.q.token + h * p.q.head;
            float          top = -INFINITY, sum = 0.0f, acc = 0.0f;
            for(int64_t j0 = 0; j0 < end; j0 += CHUNK)
            {
                const int64_t j   = j0 + t;
                float         s   = -INFINITY;
                int64_t       row = -1;
                if(j < end)
                {
                    const int32_t page = p.block_table[size_t(b) * p.ld_table + j / p.page_size];
                    if(page >= 0 && uint32_t(page) < p.num_pages && (j < len || (bits >> (j - len) & 1)))
                    {
                        row = page;
                        const T* kr  = k + row * p.k.batch + (j % p.page_size) * p.k.token + g * p.k.head;
                        float    dot = 0.0f;
                        for(uint32_t c = 0; c < p.dim; ++c)
                            dot = fmaf(to_f32(qr[c]), to_f32(kr[c]), dot);
                        s = dot * p.scale;
                        if(p.cap > 0.0f)
                            s = p.cap * tanh_of(s / p.cap);
                        const int64_t where = j < len ? j : len + (p.depths ? p.depths[size_t(b) * p.drafts + (j - len)] : int32_t(j - len));
                        s -= slope * fabsf(static_cast<float>(at - where));
                    }
                }
                float m2 = s, add;
                for(int x = 16; x > 0; x >>= 1)
                    m2 = fmaxf(m2, __shfl_xor_sync(0xFFFFFFFFu, m2, x));
                __syncthreads();
                if((t & 31) == 0)
                    buf[t >> 5] = m2;
                __syncthreads();
                m2 = fmaxf(top, fmaxf(fmaxf(buf[0], buf[1]), fmaxf(buf[2], buf[3])));
                if(m2 == -INFINITY)
                    continue;
                const float f = exp2f((top - m2) * LOG2E);
                add = w[t] = exp2f((s - m2) * LOG2E);
                rows[t]    = row;
                for(int x = 16; x > 0; x >>= 1)
                    add += __shfl_xor_sync(0xFFFFFFFFu, add, x);
                if((t & 31) == 0)
                    buf[4 + (t >> 5)] = add;
                __syncthreads();
                sum = sum * f + ((buf[4] + buf[5]) + (buf[6] + buf[7]));
                acc *= f;
                for(uint32_t c = 0; c < CHUNK; ++c)
                    if(t < p.dim && w[c] != 0.0f)
                        acc += w[c] * to_f32(v[rows[c] * p.v.batch + ((j0 + c) % p.page_size) * p.v.token + g * p.v.head + t]);
                top = m2;
            }
            if(t < p.dim)
                o[b * p.o.batch + d * p.o.token + h * p.o.head + t] = from_f32<T>(sum > 0.0f ? acc / sum : 0.0f);
        }
    } // namespace attn_tree
} // namespace b200wmma

using namespace b200wmma;

extern "C" size_t b200wmma_attn_tree_workspace_bytes(uint32_t, uint32_t, uint32_t, uint32_t, uint32_t, uint32_t)
{
    return 0;
}

extern "C" int b200wmma_attn_tree(const b200wmma_attn_args* a, uint32_t drafts, const void* q, const void* k_cache, const void* v_cache,
                                  uint32_t num_pages, uint32_t page_size, const int32_t* block_table, uint32_t ld_table,
                                  const int32_t* lens, const int32_t* n_drafts, const uint64_t* tree, const int32_t* depths, void* o,
                                  void* workspace, size_t workspace_bytes, void* stream)
{
    clear_error();
    static const char* const who = "attn_tree";
    if(int e = attn::check_common(who, a))
        return e;
    B200_REQUIRE(!a->len_q && !a->len_kv && !a->causal && !a->prefix && !a->doc_q && !a->doc_kv, B200WMMA_ERR_INVALID_ARG,
                 "%s: len_q, len_kv, causal, prefix and documents belong to attn_fwd and must be zero", who);
    B200_REQUIRE(drafts >= 1 && drafts <= attn_tree::MAX_DRAFTS, B200WMMA_ERR_UNSUPPORTED, "%s: drafts must be 1 to %u", who,
                 attn_tree::MAX_DRAFTS);
    B200_REQUIRE(num_pages && page_size && ld_table, B200WMMA_ERR_INVALID_ARG, "%s: num_pages, page_size and ld_table must be non-zero", who);
    B200_REQUIRE(num_pages < (1u << 31) && uint64_t(ld_table) * page_size < (uint64_t(1) << 31), B200WMMA_ERR_UNSUPPORTED,
                 "%s: num_pages and ld_table x page_size must be below 2^31", who);
    B200_REQUIRE(block_table && lens, B200WMMA_ERR_INVALID_ARG, "%s: block_table and lens must be non-null", who);
    B200_REQUIRE(uint64_t(a->batch) * a->heads_q * drafts < (uint64_t(1) << 31), B200WMMA_ERR_UNSUPPORTED,
                 "%s: batch x heads_q x drafts must be below 2^31", who);
    attn_tree::Params p{};
    if(int e = attn::check_strides(who, "q", q, a->q, a->batch, drafts, a->heads_q, &p.q))
        return e;
    if(int e = attn::check_strides(who, "k_cache", k_cache, a->k, num_pages, page_size, a->heads_kv, &p.k))
        return e;
    if(int e = attn::check_strides(who, "v_cache", v_cache, a->v, num_pages, page_size, a->heads_kv, &p.v))
        return e;
    if(int e = attn::check_strides(who, "o", o, a->o, a->batch, drafts, a->heads_q, &p.o))
        return e;
    B200_REQUIRE(attn::disjoint(p.o, a->batch, drafts, a->heads_q, a->head_dim), B200WMMA_ERR_INVALID_ARG, "%s: rows of o overlap", who);
    if(int e = require_sm100())
        return e;
    p.batch = a->batch, p.heads_q = a->heads_q, p.heads_kv = a->heads_kv, p.dim = a->head_dim, p.drafts = drafts, p.num_pages = num_pages;
    p.page_size = page_size, p.ld_table = ld_table, p.scale = a->scale, p.cap = a->cap, p.slopes = a->slopes, p.block_table = block_table;
    p.lens = lens, p.n_drafts = n_drafts, p.depths = depths, p.tree = tree;
    const uint32_t grid = p.batch * p.heads_q * p.drafts;
    if(a->data_type == B200WMMA_OUT_F16)
        attn_tree::tree_kernel<__half><<<grid, attn_tree::CHUNK, 0, as_stream(stream)>>>(
            p, static_cast<const __half*>(q), static_cast<const __half*>(k_cache), static_cast<const __half*>(v_cache), static_cast<__half*>(o));
    else
        attn_tree::tree_kernel<__nv_bfloat16><<<grid, attn_tree::CHUNK, 0, as_stream(stream)>>>(
            p, static_cast<const __nv_bfloat16*>(q), static_cast<const __nv_bfloat16*>(k_cache), static_cast<const __nv_bfloat16*>(v_cache),
            static_cast<__nv_bfloat16*>(o));
    B200_CHECK_CUDA(cudaGetLastError());
    return B200WMMA_OK;
}
