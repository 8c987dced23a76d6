// Attention, forward and backward: the entry points b200wmma_attn_fwd / _bwd.
#include "attn_fwd.cuh"

namespace b200wmma
{
    namespace attn
    {
        constexpr uint32_t CHUNK = 128; // keys (or queries) of one step; threads of a block

        __device__ __forceinline__ bool visible(const Params& p, uint32_t b, uint32_t i, uint32_t j, int32_t prefix)
        {
            const int64_t at = int64_t(i) + p.off;
            if(p.causal && int64_t(j) > at && int64_t(j) >= prefix)
                return false;
            if(p.doc_q)
            {
                const int32_t dq = p.doc_q[size_t(b) * p.len_q + i];
                return dq >= 0 && dq == p.doc_kv[size_t(b) * p.len_kv + j];
            }
            return true;
        }
        // score of a dot product, and the derivative of the cap at it
        __device__ __forceinline__ float score_of(const Params& p, float dot, uint32_t i, uint32_t j, float slope, float& slip)
        {
            float s = dot * p.scale;
            slip    = 1.0f;
            if(p.cap > 0.0f)
            {
                const float t = tanh_of(s / p.cap);
                s             = p.cap * t;
                slip          = 1.0f - t * t;
            }
            return s - slope * fabsf(static_cast<float>(int64_t(i) + p.off - int64_t(j)));
        }
        template <typename T>
        __device__ __forceinline__ float dot_row(const T* a, const T* b, uint32_t dim)
        {
            float s = 0.0f;
            for(uint32_t d = 0; d < dim; ++d)
                s = fmaf(to_f32(a[d]), to_f32(b[d]), s);
            return s;
        }
        __device__ __forceinline__ float block_max(float v, float* buf)
        {
            for(int o = 16; o > 0; o >>= 1)
                v = fmaxf(v, __shfl_xor_sync(0xFFFFFFFFu, v, o));
            __syncthreads();
            if((threadIdx.x & 31) == 0)
                buf[threadIdx.x >> 5] = v;
            __syncthreads();
            return fmaxf(fmaxf(buf[0], buf[1]), fmaxf(buf[2], buf[3]));
        }
        __device__ __forceinline__ float block_sum(float v, float* buf)
        {
            for(int o = 16; o > 0; o >>= 1)
                v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
            __syncthreads();
            if((threadIdx.x & 31) == 0)
                buf[threadIdx.x >> 5] = v;
            __syncthreads();
            return (buf[0] + buf[1]) + (buf[2] + buf[3]);
        }

        // delta = rowsum(dout * o), one block to a query
        template <typename T>
        __global__ void __launch_bounds__(CHUNK) delta_kernel(const Params p, const T* o, const T* dout, const float* lse, float* delta)
        {
            __shared__ float buf[4];
            const uint32_t   i = blockIdx.x % p.len_q, h = blockIdx.x / p.len_q % p.heads_q, b = blockIdx.x / p.len_q / p.heads_q;
            const size_t     row = (size_t(b) * p.heads_q + h) * p.len_q + i;
            float            x   = 0.0f;
            if(threadIdx.x < p.dim && lse[row] != -INFINITY)
                x = to_f32(o[b * p.o.batch + i * p.o.token + h * p.o.head + threadIdx.x])
                    * to_f32(dout[b * p.dout.batch + i * p.dout.token + h * p.dout.head + threadIdx.x]);
            x = block_sum(x, buf);
            if(threadIdx.x == 0)
                delta[row] = x;
        }

        // dq: one block to a query, 128 keys at a time
        template <typename T>
        __global__ void __launch_bounds__(CHUNK) dq_kernel(const Params p, const T* q, const T* k, const T* v, const T* dout,
                                                           const float* lse, const float* delta, T* dq)
        {
            __shared__ float w[CHUNK];
            const uint32_t   i = blockIdx.x % p.len_q, h = blockIdx.x / p.len_q % p.heads_q, b = blockIdx.x / p.len_q / p.heads_q;
            const uint32_t   g = h / (p.heads_q / p.heads_kv), t = threadIdx.x;
            const T*         qr     = q + b * p.q.batch + i * p.q.token + h * p.q.head;
            const T*         dr     = dout + b * p.dout.batch + i * p.dout.token + h * p.dout.head;
            const size_t     row    = (size_t(b) * p.heads_q + h) * p.len_q + i;
            const float      slope  = p.slopes ? p.slopes[h] : 0.0f;
            const int32_t    prefix = p.prefix ? p.prefix[b] : 0;
            float            acc    = 0.0f;
            for(uint32_t j0 = 0; j0 < p.len_kv; j0 += CHUNK)
            {
                const uint32_t j = j0 + t;
                float          ds = 0.0f, slip;
                if(j < p.len_kv && visible(p, b, i, j, prefix))
                {
                    const float s = score_of(p, dot_row(qr, k + b * p.k.batch + j * p.k.token + g * p.k.head, p.dim), i, j, slope, slip);
                    const float e = exp2f((s - lse[row]) * LOG2E);
                    ds = e * (dot_row(dr, v + b * p.v.batch + j * p.v.token + g * p.v.head, p.dim) - delta[row]) * slip;
                }
                __syncthreads();
                w[t] = ds;
                __syncthreads();
                for(uint32_t c = 0; c < min(CHUNK, p.len_kv - j0); ++c)
                    if(t < p.dim && w[c] != 0.0f)
                        acc += w[c] * to_f32(k[b * p.k.batch + (j0 + c) * p.k.token + g * p.k.head + t]);
            }
            if(t < p.dim)
                dq[b * p.dq.batch + i * p.dq.token + h * p.dq.head + t] = from_f32<T>(acc * p.scale);
        }

        // dk and dv: one block to a key of one key head, 128 queries at a time over the heads that share it
        template <typename T>
        __global__ void __launch_bounds__(CHUNK) dkv_kernel(const Params p, const T* q, const T* k, const T* v, const T* dout,
                                                            const float* lse, const float* delta, T* dk, T* dv)
        {
            __shared__ float w[CHUNK], e[CHUNK];
            const uint32_t   j = blockIdx.x % p.len_kv, g = blockIdx.x / p.len_kv % p.heads_kv, b = blockIdx.x / p.len_kv / p.heads_kv;
            const uint32_t   t = threadIdx.x, share = p.heads_q / p.heads_kv;
            const T*         kr     = k + b * p.k.batch + j * p.k.token + g * p.k.head;
            const T*         vr     = v + b * p.v.batch + j * p.v.token + g * p.v.head;
            const int32_t    prefix = p.prefix ? p.prefix[b] : 0;
            float            ak = 0.0f, av = 0.0f;
            for(uint32_t h = g * share; h < (g + 1) * share; ++h)
            {
                const float slope = p.slopes ? p.slopes[h] : 0.0f;
                for(uint32_t i0 = 0; i0 < p.len_q; i0 += CHUNK)
                {
                    const uint32_t i = i0 + t;
                    float          ds = 0.0f, pr = 0.0f, slip;
                    if(i < p.len_q && visible(p, b, i, j, prefix))
                    {
                        const size_t row = (size_t(b) * p.heads_q + h) * p.len_q + i;
                        const float s = score_of(p, dot_row(q + b * p.q.batch + i * p.q.token + h * p.q.head, kr, p.dim), i, j, slope, slip);
                        pr = exp2f((s - lse[row]) * LOG2E);
                        ds = pr * (dot_row(dout + b * p.dout.batch + i * p.dout.token + h * p.dout.head, vr, p.dim) - delta[row]) * slip;
                    }
                    __syncthreads();
                    w[t] = ds, e[t] = pr;
                    __syncthreads();
                    for(uint32_t c = 0; c < min(CHUNK, p.len_q - i0); ++c)
                        if(t < p.dim && e[c] != 0.0f)
                        {
                            ak += w[c] * to_f32(q[b * p.q.batch + (i0 + c) * p.q.token + h * p.q.head + t]);
                            av += e[c] * to_f32(dout[b * p.dout.batch + (i0 + c) * p.dout.token + h * p.dout.head + t]);
                        }
                }
            }
            if(t < p.dim)
            {
                dk[b * p.dk.batch + j * p.dk.token + g * p.dk.head + t] = from_f32<T>(ak * p.scale);
                dv[b * p.dv.batch + j * p.dv.token + g * p.dv.head + t] = from_f32<T>(av);
            }
        }

        // Workspace: documents of the query and key tiles, then (backward) delta.
        static size_t tiles_of(uint32_t len)
        {
            return (len + TILE - 1) / TILE;
        }
        static size_t workspace_bytes(uint32_t batch, uint32_t heads_q, uint32_t len_q, uint32_t len_kv, int backward)
        {
            const size_t docs = batch * (tiles_of(len_q) + tiles_of(len_kv)) * sizeof(DocTile);
            return docs + (backward ? size_t(batch) * heads_q * len_q * sizeof(float) : 0);
        }
        static int list_documents(const Params& p, void* workspace, const DocTile** q, const DocTile** kv, cudaStream_t stream)
        {
            *q = *kv = nullptr;
            if(!p.doc_q)
                return B200WMMA_OK;
            DocTile*       dq = static_cast<DocTile*>(workspace);
            const uint32_t nq = uint32_t(tiles_of(p.len_q)), nk = uint32_t(tiles_of(p.len_kv));
            DocTile*       dk = dq + size_t(p.batch) * nq;
            doc_tiles_kernel<<<ceil_div(p.batch * nq, 4), 128, 0, stream>>>(p.doc_q, p.len_q, nq, p.batch * nq, dq);
            doc_tiles_kernel<<<ceil_div(p.batch * nk, 4), 128, 0, stream>>>(p.doc_kv, p.len_kv, nk, p.batch * nk, dk);
            B200_CHECK_CUDA(cudaGetLastError());
            *q = dq, *kv = dk;
            return B200WMMA_OK;
        }

        // Fills Params from checked arguments.
        static int check_args(const char* who, const b200wmma_attn_args* a, const void* q, const void* k, const void* v, const void* o,
                              Params* p)
        {
            if(int e = check_common(who, a))
                return e;
            B200_REQUIRE(a->len_q && a->len_kv, B200WMMA_ERR_INVALID_ARG, "%s: len_q and len_kv must be non-zero", who);
            B200_REQUIRE(a->len_q < (1u << 30) && a->len_kv < (1u << 30), B200WMMA_ERR_UNSUPPORTED, "%s: len_q and len_kv must be below 2^30", who);
            B200_REQUIRE(uint64_t(a->batch) * a->heads_q * a->len_q < (uint64_t(1) << 31)
                             && uint64_t(a->batch) * a->heads_kv * a->len_kv < (uint64_t(1) << 31),
                         B200WMMA_ERR_UNSUPPORTED, "%s: batch x heads x tokens must be below 2^31", who);
            B200_REQUIRE(!a->doc_q == !a->doc_kv, B200WMMA_ERR_INVALID_ARG, "%s: doc_q and doc_kv come together", who);
            if(int e = check_strides(who, "q", q, a->q, a->batch, a->len_q, a->heads_q, &p->q))
                return e;
            if(int e = check_strides(who, "k", k, a->k, a->batch, a->len_kv, a->heads_kv, &p->k))
                return e;
            if(int e = check_strides(who, "v", v, a->v, a->batch, a->len_kv, a->heads_kv, &p->v))
                return e;
            if(int e = check_strides(who, "o", o, a->o, a->batch, a->len_q, a->heads_q, &p->o))
                return e;
            p->batch = a->batch, p->heads_q = a->heads_q, p->heads_kv = a->heads_kv, p->len_q = a->len_q, p->len_kv = a->len_kv;
            p->dim = a->head_dim, p->off = int32_t(a->len_kv) - int32_t(a->len_q), p->causal = a->causal != 0;
            p->scale = a->scale, p->cap = a->cap, p->slopes = a->slopes, p->prefix = a->prefix, p->doc_q = a->doc_q, p->doc_kv = a->doc_kv;
            return B200WMMA_OK;
        }
        static int check_written(const char* who, const char* name, const Strides& s, uint32_t batch, uint32_t tokens, uint32_t heads,
                                 uint32_t dim)
        {
            B200_REQUIRE(disjoint(s, batch, tokens, heads, dim), B200WMMA_ERR_INVALID_ARG, "%s: rows of %s overlap", who, name);
            return B200WMMA_OK;
        }
        static int check_workspace(const char* who, const void* ws, size_t have, size_t need)
        {
            B200_REQUIRE(need == 0 || (ws && have >= need), B200WMMA_ERR_INVALID_ARG, "%s: workspace of %zu bytes needed, %zu given", who,
                         need, ws ? have : size_t(0));
            B200_REQUIRE(need == 0 || aligned16(ws), B200WMMA_ERR_ALIGNMENT, "%s: workspace must be 16-byte aligned", who);
            return B200WMMA_OK;
        }

        template <typename T, uint32_t HD, bool CAP, bool BIAS, bool PLAIN>
        static int launch_fwd(const Params& p, const CUtensorMap (&maps)[3], void* o, float* lse, const DocTile* dq, const DocTile* dk,
                              unsigned* status, cudaStream_t stream)
        {
            auto kern = fwd_tc05_kernel<T, HD, CAP, BIAS, PLAIN>;
            B200_CHECK_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, FwdSmem<HD>::BYTES));
            const uint32_t q_blocks = ceil_div(p.len_q, 2 * TILE);
            kern<<<q_blocks * p.batch * p.heads_q, FWD_THREADS, FwdSmem<HD>::BYTES, stream>>>(maps[0], maps[1], maps[2], p, static_cast<T*>(o), lse,
                                                                                              dq, dk, q_blocks, status);
            B200_CHECK_CUDA(cudaGetLastError());
            return B200WMMA_OK;
        }
        template <typename T, uint32_t HD>
        static int run_fwd(const Params& p, const CUtensorMap (&maps)[3], void* o, float* lse, const DocTile* dq, const DocTile* dk,
                           unsigned* status, cudaStream_t stream)
        {
            const bool cap = p.cap > 0.0f, bias = p.slopes != nullptr;
            if(cap)
                return bias ? launch_fwd<T, HD, true, true, false>(p, maps, o, lse, dq, dk, status, stream)
                            : launch_fwd<T, HD, true, false, false>(p, maps, o, lse, dq, dk, status, stream);
            if(bias)
                return launch_fwd<T, HD, false, true, false>(p, maps, o, lse, dq, dk, status, stream);
            // the softmax scales plain scores in the exponential's argument, which takes a positive scale
            return p.scale > 0.0f ? launch_fwd<T, HD, false, false, true>(p, maps, o, lse, dq, dk, status, stream)
                                  : launch_fwd<T, HD, false, false, false>(p, maps, o, lse, dq, dk, status, stream);
        }
        template <typename T>
        static int run_bwd(const Params& p, const void* q_, const void* k_, const void* v_, const void* o_, const void* dout_, const float* lse,
                           void* dq, void* dk, void* dv, float* delta, cudaStream_t stream)
        {
            const T *q = static_cast<const T*>(q_), *k = static_cast<const T*>(k_), *v = static_cast<const T*>(v_);
            const T *o = static_cast<const T*>(o_), *dout = static_cast<const T*>(dout_);
            const uint32_t rows_q = p.batch * p.heads_q * p.len_q, rows_kv = p.batch * p.heads_kv * p.len_kv;
            delta_kernel<T><<<rows_q, CHUNK, 0, stream>>>(p, o, dout, lse, delta);
            dq_kernel<T><<<rows_q, CHUNK, 0, stream>>>(p, q, k, v, dout, lse, delta, static_cast<T*>(dq));
            dkv_kernel<T><<<rows_kv, CHUNK, 0, stream>>>(p, q, k, v, dout, lse, delta, static_cast<T*>(dk), static_cast<T*>(dv));
            B200_CHECK_CUDA(cudaGetLastError());
            return B200WMMA_OK;
        }
    } // namespace attn
} // namespace b200wmma

using namespace b200wmma;

extern "C" size_t b200wmma_attn_workspace_bytes(uint32_t batch, uint32_t heads_q, uint32_t len_q, uint32_t len_kv, int backward)
{
    return attn::workspace_bytes(batch, heads_q, len_q, len_kv, backward);
}

extern "C" int b200wmma_attn_fwd(const b200wmma_attn_args* args, const void* q, const void* k, const void* v, void* o, float* lse,
                                 void* workspace, size_t workspace_bytes, void* stream)
{
    clear_error();
    static const char* const who = "attn_fwd";
    attn::Params             p{};
    if(int e = attn::check_args(who, args, q, k, v, o, &p))
        return e;
    if(int e = attn::check_written(who, "o", p.o, p.batch, p.len_q, p.heads_q, p.dim))
        return e;
    const size_t need = p.doc_q ? attn::workspace_bytes(p.batch, p.heads_q, p.len_q, p.len_kv, 0) : 0;
    if(int e = attn::check_workspace(who, workspace, workspace_bytes, need))
        return e;
    if(int e = require_sm100())
        return e;
    unsigned* status = nullptr;
    if(int e = status_word_ptr(&status))
        return e;
    CUtensorMap maps[3];
    if(int e = attn::make_map(&maps[0], args->data_type, q, p.dim, p.len_q, p.heads_q, p.batch, p.q))
        return e;
    if(int e = attn::make_map(&maps[1], args->data_type, k, p.dim, p.len_kv, p.heads_kv, p.batch, p.k))
        return e;
    if(int e = attn::make_map(&maps[2], args->data_type, v, p.dim, p.len_kv, p.heads_kv, p.batch, p.v))
        return e;
    const attn::DocTile *dq = nullptr, *dk = nullptr;
    if(int e = attn::list_documents(p, workspace, &dq, &dk, as_stream(stream)))
        return e;
    if(args->data_type == B200WMMA_OUT_F16)
        return p.dim <= 64 ? attn::run_fwd<__half, 64>(p, maps, o, lse, dq, dk, status, as_stream(stream))
                           : attn::run_fwd<__half, 128>(p, maps, o, lse, dq, dk, status, as_stream(stream));
    return p.dim <= 64 ? attn::run_fwd<__nv_bfloat16, 64>(p, maps, o, lse, dq, dk, status, as_stream(stream))
                       : attn::run_fwd<__nv_bfloat16, 128>(p, maps, o, lse, dq, dk, status, as_stream(stream));
}

extern "C" int b200wmma_attn_bwd(const b200wmma_attn_args* args, const void* q, const void* k, const void* v, const void* o,
                                 const void* dout, const float* lse, void* dq, void* dk, void* dv, void* workspace,
                                 size_t workspace_bytes, void* stream)
{
    clear_error();
    static const char* const who = "attn_bwd";
    attn::Params             p{};
    if(int e = attn::check_args(who, args, q, k, v, o, &p))
        return e;
    B200_REQUIRE(lse, B200WMMA_ERR_INVALID_ARG, "%s: lse must be non-null", who);
    if(int e = attn::check_strides(who, "dout", dout, args->dout, p.batch, p.len_q, p.heads_q, &p.dout))
        return e;
    if(int e = attn::check_strides(who, "dq", dq, args->dq, p.batch, p.len_q, p.heads_q, &p.dq))
        return e;
    if(int e = attn::check_strides(who, "dk", dk, args->dk, p.batch, p.len_kv, p.heads_kv, &p.dk))
        return e;
    if(int e = attn::check_strides(who, "dv", dv, args->dv, p.batch, p.len_kv, p.heads_kv, &p.dv))
        return e;
    if(int e = attn::check_written(who, "dq", p.dq, p.batch, p.len_q, p.heads_q, p.dim))
        return e;
    if(int e = attn::check_written(who, "dk", p.dk, p.batch, p.len_kv, p.heads_kv, p.dim))
        return e;
    if(int e = attn::check_written(who, "dv", p.dv, p.batch, p.len_kv, p.heads_kv, p.dim))
        return e;
    if(int e = attn::check_workspace(who, workspace, workspace_bytes,
                                     attn::workspace_bytes(p.batch, p.heads_q, p.len_q, p.len_kv, 1)))
        return e;
    if(int e = require_sm100())
        return e;
    float* delta = reinterpret_cast<float*>(static_cast<attn::DocTile*>(workspace)
                                            + p.batch * (attn::tiles_of(p.len_q) + attn::tiles_of(p.len_kv)));
    return args->data_type == B200WMMA_OUT_F16
               ? attn::run_bwd<__half>(p, q, k, v, o, dout, lse, dq, dk, dv, delta, as_stream(stream))
               : attn::run_bwd<__nv_bfloat16>(p, q, k, v, o, dout, lse, dq, dk, dv, delta, as_stream(stream));
}
