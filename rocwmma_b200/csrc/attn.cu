// Attention, forward and backward: the entry points b200wmma_attn_fwd / _bwd.
#include "attn_bwd.cuh"
#include "attn_fwd.cuh"

namespace b200wmma
{
    namespace attn
    {
        constexpr uint32_t SLOTS = 148; // blocks that run at once, one to an SM
        static size_t tiles_of(uint32_t len)
        {
            return (len + TILE - 1) / TILE;
        }
        // Blocks of the dkv kernel to a key tile: where those tiles do not fill the machine the steps (query heads x query tiles) are
        // split, at least four to a block, and the parts are summed up by a kernel of their own: 8 query heads to one key head, 1700
        // tokens x 128, causal, gradients 66 us (242 unsplit).
        static uint32_t dkv_splits(uint32_t batch, uint32_t heads_q, uint32_t heads_kv, uint32_t len_q, uint32_t len_kv)
        {
            const uint64_t blocks = tiles_of(len_kv) * batch * heads_kv, most = (tiles_of(len_q) * (heads_q / heads_kv) + 3) / 4;
            const uint64_t n = SLOTS / blocks < most ? SLOTS / blocks : most;
            return n > 1 ? uint32_t(n) : 1u;
        }
        // Blocks of a dkv kernel that is split, for whatever number of key heads makes them most.
        static size_t dkv_parts(uint32_t batch, uint32_t heads_q, uint32_t len_q, uint32_t len_kv)
        {
            const size_t tiles = tiles_of(len_kv) * batch; // of one key head
            size_t       most  = 0;
            for(uint32_t heads_kv = 1; tiles && heads_kv <= heads_q && 2 * tiles * heads_kv <= SLOTS; ++heads_kv)
                if(heads_q % heads_kv == 0)
                {
                    const uint32_t splits = dkv_splits(batch, heads_q, heads_kv, len_q, len_kv);
                    if(splits > 1 && splits * tiles * heads_kv > most)
                        most = splits * tiles * heads_kv;
                }
            return most;
        }
        // Workspace: documents of the query and key tiles, then (backward) lse and delta of each row, padded to whole tiles, then the
        // parts of dk and dv, a tile of each for every block of a dkv kernel that is split.
        static size_t workspace_bytes(uint32_t batch, uint32_t heads_q, uint32_t len_q, uint32_t len_kv, int backward)
        {
            const size_t docs = batch * (tiles_of(len_q) + tiles_of(len_kv)) * sizeof(DocTile);
            if(!backward)
                return docs;
            const size_t rows = 2 * size_t(batch) * heads_q * tiles_of(len_q) * TILE * sizeof(float);
            return docs + rows + dkv_parts(batch, heads_q, len_q, len_kv) * 2 * TILE * MAX_DIM * sizeof(float);
        }
        static int list_documents(const Params& p, void* workspace, const DocTile** q, const DocTile** kv, cudaStream_t stream)
        {
            *q = *kv = nullptr;
            if(!p.doc_q)
                return B200WMMA_OK;
            DocTile*       dq = static_cast<DocTile*>(workspace);
            const uint32_t nq = uint32_t(tiles_of(p.len_q)), nk = uint32_t(tiles_of(p.len_kv));
            DocTile*       dk = dq + size_t(p.batch) * nq;
            const bool     one = p.doc_q == p.doc_kv && p.len_q == p.len_kv; // queries and keys are the same tokens
            const uint32_t total_q = one ? 0 : p.batch * nq, total = total_q + p.batch * nk;
            doc_tiles_kernel<<<ceil_div(total, 4), 128, 0, stream>>>(p.doc_q, p.len_q, nq, total_q, dq, p.doc_kv, p.len_kv, nk, total, dk);
            B200_CHECK_CUDA(cudaGetLastError());
            *q = one ? dk : dq, *kv = dk;
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
            const uint64_t most = uint64_t(1) << 31;
            B200_REQUIRE(uint64_t(a->batch) * a->heads_q < most && uint64_t(a->batch) * a->heads_q * tiles_of(a->len_q) * TILE < most
                             && uint64_t(a->batch) * a->heads_kv * tiles_of(a->len_kv) * TILE < most,
                         B200WMMA_ERR_UNSUPPORTED, "%s: batch x heads x tokens, in tiles of 128 tokens, must be below 2^31", who);
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

        template <typename T, uint32_t HD, bool CAP, bool BIAS, bool PLAIN, uint32_t PER>
        static int launch_fwd_as(const Params& p, const CUtensorMap (&maps)[4], float* lse, const DocTile* dq, const DocTile* dk,
                              unsigned* status, cudaStream_t stream)
        {
            auto kern = fwd_tc05_kernel<T, HD, CAP, BIAS, PLAIN, PER>;
            static Allowed allowed;
            if(int e = allow_smem(reinterpret_cast<const void*>(kern), FwdSmem<HD>::BYTES, allowed))
                return e;
            const uint32_t q_blocks = ceil_div(p.len_q, PER * TILE);
            kern<<<q_blocks * p.batch * p.heads_q, FWD_THREADS, FwdSmem<HD>::BYTES, stream>>>(maps[0], maps[1], maps[2], maps[3], p, lse,
                                                                                              dq, dk, q_blocks, status);
            B200_CHECK_CUDA(cudaGetLastError());
            return B200WMMA_OK;
        }
        // One tile of queries to a block where those blocks still run all at once: 2 x 8 heads of 1024 x 128, causal, 16.6 us (21.5 with
        // two tiles), with cap and slopes 28 us (38); more of them lose (2 x 16 heads of 4096 x 128, causal: 213 us, 140 with two).
        template <typename T, uint32_t HD, bool CAP, bool BIAS, bool PLAIN>
        static int launch_fwd(const Params& p, const CUtensorMap (&maps)[4], float* lse, const DocTile* dq, const DocTile* dk,
                              unsigned* status, cudaStream_t stream)
        {
            return tiles_of(p.len_q) * p.batch * p.heads_q <= SLOTS ? launch_fwd_as<T, HD, CAP, BIAS, PLAIN, 1>(p, maps, lse, dq, dk, status, stream)
                                                                  : launch_fwd_as<T, HD, CAP, BIAS, PLAIN, 2>(p, maps, lse, dq, dk, status, stream);
        }
        template <typename T, uint32_t HD>
        static int run_fwd(const Params& p, const CUtensorMap (&maps)[4], float* lse, const DocTile* dq, const DocTile* dk,
                           unsigned* status, cudaStream_t stream)
        {
            const bool cap = p.cap > 0.0f, bias = p.slopes != nullptr;
            if(cap)
                return bias ? launch_fwd<T, HD, true, true, false>(p, maps, lse, dq, dk, status, stream)
                            : launch_fwd<T, HD, true, false, false>(p, maps, lse, dq, dk, status, stream);
            if(bias)
                return launch_fwd<T, HD, false, true, false>(p, maps, lse, dq, dk, status, stream);
            // the softmax scales plain scores in the exponential's argument, which takes a positive scale
            return p.scale > 0.0f ? launch_fwd<T, HD, false, false, true>(p, maps, lse, dq, dk, status, stream)
                                  : launch_fwd<T, HD, false, false, false>(p, maps, lse, dq, dk, status, stream);
        }
        struct BwdCall
        {
            CUtensorMap    maps[7]; // q, k, v, dout, dq, dk, dv
            const void *   o, *dout;
            const float*   lse;
            float *        lse2, *delta, *partial;
            void *         dk, *dv;
            const DocTile *docs_q, *docs_kv;
            unsigned*      status;
            cudaStream_t   stream;
        };
        template <typename T, uint32_t HD, bool CAP, bool BIAS>
        static int launch_bwd(const Params& p, const BwdCall& c)
        {
            auto dkv = bwd_dkv_kernel<T, HD, CAP, BIAS>;
            auto dq  = bwd_dq_kernel<T, HD, CAP, BIAS>;
            static Allowed allowed[2];
            if(int e = allow_smem(reinterpret_cast<const void*>(dkv), BwdSmem<HD>::BYTES, allowed[0]))
                return e;
            if(int e = allow_smem(reinterpret_cast<const void*>(dq), BwdSmem<HD>::BYTES, allowed[1]))
                return e;
            const uint32_t padded = uint32_t(tiles_of(p.len_q)) * TILE, rows = p.batch * p.heads_q * padded;
            bwd_rows_kernel<T><<<rows / 16, 256, 0, c.stream>>>(p, static_cast<const T*>(c.o), static_cast<const T*>(c.dout), c.lse, c.lse2, c.delta,
                                                                padded, rows);
            B200_CHECK_CUDA(cudaGetLastError());
            cudaLaunchAttribute early{};
            early.id                                         = cudaLaunchAttributeProgrammaticStreamSerialization;
            early.val.programmaticStreamSerializationAllowed = 1;
            cudaLaunchConfig_t cfg{};
            cfg.blockDim = dim3(BwdWarps<CAP>::THREADS), cfg.dynamicSmemBytes = BwdSmem<HD>::BYTES, cfg.stream = c.stream, cfg.attrs = &early, cfg.numAttrs = 1;
            cfg.gridDim = dim3(uint32_t(tiles_of(p.len_q)) * p.batch * p.heads_q);
            B200_CHECK_CUDA(cudaLaunchKernelEx(&cfg, dq, c.maps[0], c.maps[1], c.maps[2], c.maps[3], c.maps[4], p, static_cast<const float*>(c.lse2),
                                               c.delta, c.docs_q, c.docs_kv, c.status));
            const uint32_t blocks = uint32_t(tiles_of(p.len_kv)) * p.batch * p.heads_kv;
            const uint32_t splits = dkv_splits(p.batch, p.heads_q, p.heads_kv, p.len_q, p.len_kv);
            cfg.gridDim = dim3(blocks * splits);
            B200_CHECK_CUDA(cudaLaunchKernelEx(&cfg, dkv, c.maps[0], c.maps[1], c.maps[2], c.maps[3], c.maps[5], c.maps[6], p,
                                               static_cast<const float*>(c.lse2), static_cast<const float*>(c.delta), c.docs_q, c.docs_kv, splits, c.partial, c.status));
            if(splits > 1)
            {
                bwd_join_kernel<T, HD><<<blocks * 2 * (TILE * HD / 1024), 256, 0, c.stream>>>(p, c.partial, splits, blocks, static_cast<T*>(c.dk),
                                                                                           static_cast<T*>(c.dv));
                B200_CHECK_CUDA(cudaGetLastError());
            }
            return B200WMMA_OK;
        }
        template <typename T, uint32_t HD>
        static int run_bwd(const Params& p, const BwdCall& c)
        {
            const bool cap = p.cap > 0.0f, bias = p.slopes != nullptr;
            if(cap)
                return bias ? launch_bwd<T, HD, true, true>(p, c) : launch_bwd<T, HD, true, false>(p, c);
            return bias ? launch_bwd<T, HD, false, true>(p, c) : launch_bwd<T, HD, false, false>(p, c);
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
    CUtensorMap maps[4];
    if(int e = attn::make_map(&maps[0], args->data_type, q, p.dim, p.len_q, p.heads_q, p.batch, p.q))
        return e;
    if(int e = attn::make_map(&maps[1], args->data_type, k, p.dim, p.len_kv, p.heads_kv, p.batch, p.k))
        return e;
    if(int e = attn::make_map(&maps[2], args->data_type, v, p.dim, p.len_kv, p.heads_kv, p.batch, p.v))
        return e;
    if(int e = attn::make_map(&maps[3], args->data_type, o, p.dim, p.len_q, p.heads_q, p.batch, p.o))
        return e;
    const attn::DocTile *dq = nullptr, *dk = nullptr;
    if(int e = attn::list_documents(p, workspace, &dq, &dk, as_stream(stream)))
        return e;
    if(args->data_type == B200WMMA_OUT_F16)
        return p.dim <= 64 ? attn::run_fwd<__half, 64>(p, maps, lse, dq, dk, status, as_stream(stream))
                           : attn::run_fwd<__half, 128>(p, maps, lse, dq, dk, status, as_stream(stream));
    return p.dim <= 64 ? attn::run_fwd<__nv_bfloat16, 64>(p, maps, lse, dq, dk, status, as_stream(stream))
                       : attn::run_fwd<__nv_bfloat16, 128>(p, maps, lse, dq, dk, status, as_stream(stream));
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
    attn::BwdCall c{};
    if(int e = status_word_ptr(&c.status))
        return e;
    if(int e = attn::make_map(&c.maps[0], args->data_type, q, p.dim, p.len_q, p.heads_q, p.batch, p.q))
        return e;
    if(int e = attn::make_map(&c.maps[1], args->data_type, k, p.dim, p.len_kv, p.heads_kv, p.batch, p.k))
        return e;
    if(int e = attn::make_map(&c.maps[2], args->data_type, v, p.dim, p.len_kv, p.heads_kv, p.batch, p.v))
        return e;
    if(int e = attn::make_map(&c.maps[3], args->data_type, dout, p.dim, p.len_q, p.heads_q, p.batch, p.dout))
        return e;
    if(int e = attn::make_map(&c.maps[4], args->data_type, dq, p.dim, p.len_q, p.heads_q, p.batch, p.dq))
        return e;
    if(int e = attn::make_map(&c.maps[5], args->data_type, dk, p.dim, p.len_kv, p.heads_kv, p.batch, p.dk))
        return e;
    if(int e = attn::make_map(&c.maps[6], args->data_type, dv, p.dim, p.len_kv, p.heads_kv, p.batch, p.dv))
        return e;
    const size_t doc_tiles = p.batch * (attn::tiles_of(p.len_q) + attn::tiles_of(p.len_kv));
    c.lse2  = reinterpret_cast<float*>(static_cast<attn::DocTile*>(workspace) + doc_tiles);
    c.delta = c.lse2 + size_t(p.batch) * p.heads_q * attn::tiles_of(p.len_q) * attn::TILE;
    c.partial = c.delta + size_t(p.batch) * p.heads_q * attn::tiles_of(p.len_q) * attn::TILE;
    c.o = o, c.dout = dout, c.lse = lse, c.dk = dk, c.dv = dv, c.stream = as_stream(stream);
    if(int e = attn::list_documents(p, workspace, &c.docs_q, &c.docs_kv, c.stream))
        return e;
    if(args->data_type == B200WMMA_OUT_F16)
        return p.dim <= 64 ? attn::run_bwd<__half, 64>(p, c) : attn::run_bwd<__half, 128>(p, c);
    return p.dim <= 64 ? attn::run_bwd<__nv_bfloat16, 64>(p, c) : attn::run_bwd<__nv_bfloat16, 128>(p, c);
}
