// Pieces of the tcgen05 attention kernels: the instruction forms the GEMM does not use, masks by tile, the arithmetic of a
// score in registers, operand tiles and tensor maps.
//
// Tiles are 128 queries x 128 keys.  An operand tile is 128 rows of HD = 64 or 128 elements (a smaller head is padded with
// zeros by TMA), stored as HD / 64 boxes of 128 rows x 128 bytes with the 128-byte swizzle.  The same bytes serve as a
// K-major operand (the head is the contraction) and as an MN-major one (the tokens are the contraction).
// A product whose left operand comes out of a softmax takes it from tensor memory: its 16-bit values overwrite the fp32
// scores that they were computed from, two to a 32-bit column.
#pragma once
#include "attn_common.cuh"
#include "gemm_tc05_common.cuh"

namespace b200wmma
{
    namespace attn
    {
        constexpr uint32_t TILE      = 128;
        constexpr uint32_t BOX_BYTES = TILE * 128; // 128 rows x 64 elements of 16 bits
        constexpr uint32_t SEG       = 512; // key (or query) tiles that are listed at a time
        // A softmax's maximum is moved where a score passes it by this many powers of two: until then weights grow up to 2^14,
        // which both 16-bit types hold; sums are fp32.
        constexpr float RESCALE_STEP = 14.0f;

        template <typename T>
        constexpr int kind_of = std::is_same<T, __half>::value ? tc05::KIND_F16 : tc05::KIND_BF16;

        // ---- instructions ----
        // True in one lane of a converged warp, always the same one.  Products issued behind this instead of behind `lane == 0`:
        // attn_fwd 1 x 16 heads of 16384 x 128 1208 TFLOP/s (1056), its gradients 704 (652), at that step.
        __device__ __forceinline__ bool elect_one()
        {
            uint32_t yes;
            asm volatile("{\n"
                         ".reg .pred p;\n"
                         "elect.sync _|p, 0xFFFFFFFF;\n"
                         "selp.u32 %0, 1, 0, p;\n"
                         "}"
                         : "=r"(yes));
            return yes != 0;
        }
        // D[tmem] (+)= A[tmem] * B[smem]
        __device__ __forceinline__ void mma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, uint32_t accumulate)
        {
            asm volatile("{\n"
                         ".reg .pred p;\n"
                         "setp.ne.b32 p, %4, 0;\n"
                         "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n"
                         "}" ::"r"(d_tmem),
                         "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
                         : "memory");
        }
        __device__ __forceinline__ void tmem_st_32x32b_x32(uint32_t taddr, const uint32_t (&r)[32])
        {
            asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], "
                         "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
                         "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31};" ::"r"(r[0]),
                         "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
                         "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]),
                         "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]),
                         "r"(r[29]), "r"(r[30]), "r"(r[31]), "r"(taddr)
                         : "memory");
        }
        __device__ __forceinline__ void tmem_st_32x32b_x16(uint32_t taddr, const uint32_t (&r)[16])
        {
            asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], "
                         "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};" ::"r"(r[0]),
                         "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
                         "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(taddr)
                         : "memory");
        }
        __device__ __forceinline__ void tmem_st_wait()
        {
            asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
        }
        __device__ __forceinline__ void tma_load_4d(uint32_t dst_smem, const void* tmap, int32_t c0, int32_t c1, int32_t c2, int32_t c3,
                                                    uint32_t bar)
        {
            asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes"
                         " [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst_smem),
                         "l"(reinterpret_cast<uint64_t>(tmap)), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(bar)
                         : "memory");
        }
        __device__ __forceinline__ float ex2(float x)
        {
            float y;
            asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
            return y;
        }
        __device__ __forceinline__ float rcp(float x)
        {
            float y;
            asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
            return y;
        }
        // Two fp32 numbers in a register pair: one instruction for both.
        __device__ __forceinline__ uint64_t pair(float lo, float hi)
        {
            uint64_t r;
            asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
            return r;
        }
        __device__ __forceinline__ void unpair(uint64_t x, float& lo, float& hi)
        {
            asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(x));
        }
        __device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c)
        {
            uint64_t r;
            asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
            return r;
        }
        __device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b)
        {
            uint64_t r;
            asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
            return r;
        }
        __device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b)
        {
            uint64_t r;
            asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
            return r;
        }
        // Largest of N numbers and `t`, in two independent chains of three-input steps.
        template <int N>
        __device__ __forceinline__ float max_of(const uint32_t (&v)[N], float t)
        {
            float u = fmaxf(__uint_as_float(v[0]), __uint_as_float(v[1]));
#pragma unroll
            for(int k = 2; k < N; k += 4)
            {
                t = fmaxf(fmaxf(t, __uint_as_float(v[k])), __uint_as_float(v[k + 1]));
                if(k + 2 < N)
                    u = fmaxf(fmaxf(u, __uint_as_float(v[k + 2])), __uint_as_float(v[k + 3]));
            }
            return fmaxf(t, u);
        }
        template <typename T>
        __device__ __forceinline__ uint32_t pack2(float lo, float hi)
        {
            return tc05::Pack16<T>::narrow(lo, hi);
        }

        // Bounded wait of a whole warp on the critical path: every lane polls (one instruction for all of them) instead of being
        // parked until the barrier's completion wakes it, which takes longer than these waits last.
        __device__ __forceinline__ bool wait_bounded(uint32_t bar, uint32_t parity, volatile uint32_t* cta_abort, unsigned* status, uint32_t who)
        {
            if(ptx::mbar_try_wait(bar, parity))
                return true;
            const uint64_t t0    = ptx::globaltimer_ns();
            uint32_t       spins = 0;
            while(!ptx::mbar_try_wait(bar, parity))
                if((++spins & 63u) == 0u)
                {
                    if(*cta_abort)
                        return false;
                    if(ptx::globaltimer_ns() - t0 > tc05::WAIT_TIMEOUT_NS)
                    {
                        *cta_abort = 1u;
                        if(atomicCAS(status, 0u, ptx::STATUS_TIMEOUT_CODE) == 0u)
                            status[1] = who;
                        return false;
                    }
                }
            return true;
        }
        __device__ __forceinline__ bool wait_bounded_warp(uint32_t bar, uint32_t parity, volatile uint32_t* cta_abort, unsigned* status, uint32_t who)
        {
            return __all_sync(0xFFFFFFFFu, wait_bounded(bar, parity, cta_abort, status, who));
        }

        // ---- operand tiles --------------------------------------------------------------------
        template <uint32_t HD>
        __device__ __forceinline__ void load_tile(uint32_t dst, const CUtensorMap* map, uint32_t token, uint32_t head, uint32_t batch,
                                                  uint32_t bar)
        {
#pragma unroll
            for(uint32_t s = 0; s < HD / 64; ++s)
                tma_load_4d(dst + s * BOX_BYTES, map, s * 64, token, head, batch, bar);
        }
        // D (+)= A B^T over the head: both operands K-major tiles
        template <typename T, uint32_t HD>
        __device__ __forceinline__ void mma_over_head(uint32_t d_tmem, uint32_t a_smem, uint32_t b_smem)
        {
            constexpr uint32_t idesc = tc05::make_idesc<kind_of<T>, TILE, TILE>();
            const uint64_t     a = ptx::make_kmajor_sw128_desc(a_smem), b = ptx::make_kmajor_sw128_desc(b_smem);
#pragma unroll
            for(uint32_t k = 0; k < HD / 16; ++k)
            {
                const uint32_t at = (k / 4) * (BOX_BYTES >> 4) + (k % 4) * 2;
                ptx::mma_f16_ss(d_tmem, a + at, b + at, idesc, k != 0);
            }
        }
        // D (+)= A B over 128 tokens: A 16-bit values in tensor memory, B an MN-major tile
        template <typename T, uint32_t HD>
        __device__ __forceinline__ void mma_over_tokens(uint32_t d_tmem, uint32_t a_tmem, uint32_t b_smem, bool accumulate)
        {
            constexpr uint32_t idesc = tc05::make_idesc<kind_of<T>, TILE, HD, false, true>();
            const uint64_t     b     = ptx::make_mnmajor_sw128_desc(b_smem, BOX_BYTES);
#pragma unroll
            for(uint32_t k = 0; k < TILE / 16; ++k)
                mma_f16_ts(d_tmem, a_tmem + 8 * k, b + k * (2048u >> 4), idesc, (accumulate || k != 0) ? 1u : 0u);
        }
        // Rows of padding may hold anything: zeroed before a product contracts over them.  One warp; `docs` are the tile's.
        template <uint32_t HD>
        __device__ __forceinline__ void clear_padding(uint8_t* tile, const int32_t* docs, uint32_t rows, uint32_t lane)
        {
            for(uint32_t r = lane; r < rows; r += 32)
                if(docs[r] < 0)
                    for(uint32_t s = 0; s < HD / 64; ++s)
                        for(uint32_t c = 0; c < 8; ++c)
                            *reinterpret_cast<uint4*>(tile + s * BOX_BYTES + r * 128 + c * 16) = make_uint4(0, 0, 0, 0);
            ptx::fence_proxy_async_smem();
            __syncwarp();
        }

        // The two passes of a softmax over a row of 128 scores in tensor memory, 32 columns at a time with the next 32 on their
        // way, so that a thread holds 64 of them and not 128, which took longer than reading tensor memory twice.
        // First pass: the largest.  change(at, x) may alter columns at, at + 1, ...; WRITE puts them back for the second pass.
        template <bool WRITE, typename F>
        __device__ __forceinline__ float row_max(uint32_t taddr, F change)
        {
            uint32_t v[2][32];
            float    top = -INFINITY;
            ptx::tmem_ld_32x32b_x32(taddr, v[0]);
#pragma unroll
            for(int i = 0; i < 4; ++i)
            {
                ptx::tmem_ld_wait();
                if(i < 3)
                    ptx::tmem_ld_32x32b_x32(taddr + 32 * (i + 1), v[(i + 1) & 1]);
                change(32 * i, v[i & 1]);
                top = max_of(v[i & 1], top);
                if(WRITE)
                    tmem_st_32x32b_x32(taddr + 32 * i, v[i & 1]);
            }
            if(WRITE)
                tmem_st_wait();
            return top;
        }
        // Second pass: P = 2^(x c + sub) in 16 bits over the scores' own first 64 columns, always behind the scores still to be
        // read; returns the sum of the unrounded P.
        template <typename T>
        __device__ __forceinline__ float weights(uint32_t taddr, float c, float sub)
        {
            const uint64_t cc = pair(c, c), ss = pair(sub, sub);
            uint64_t       sum[2] = {0, 0};
            uint32_t       v[2][32];
            ptx::tmem_ld_32x32b_x32(taddr, v[0]);
#pragma unroll
            for(int i = 0; i < 4; ++i)
            {
                ptx::tmem_ld_wait();
                if(i < 3)
                    ptx::tmem_ld_32x32b_x32(taddr + 32 * (i + 1), v[(i + 1) & 1]);
                uint32_t w[16];
#pragma unroll
                for(int j = 0; j < 16; ++j)
                {
                    float x, y;
                    unpair(fma2(pair(__uint_as_float(v[i & 1][2 * j]), __uint_as_float(v[i & 1][2 * j + 1])), cc, ss), x, y);
                    x = ex2(x), y = ex2(y);
                    sum[j & 1] = add2(sum[j & 1], pair(x, y));
                    w[j]       = pack2<T>(x, y);
                }
                tmem_st_32x32b_x16(taddr + 16 * i, w);
            }
            float a, b;
            unpair(add2(sum[0], sum[1]), a, b);
            return a + b;
        }

        // Both passes in one, for a maximum that is known already: P stays in registers (16 bits, two to one) until it is clear that
        // no score of the warp has outgrown `sub` too far.  `top`: the largest of the changed scores (not times c).
        template <typename T, typename F>
        __device__ __forceinline__ float weights_at(uint32_t taddr, float c, float sub, uint32_t (&w)[4][16], float& top, F change)
        {
            const uint64_t cc = pair(c, c), ss = pair(sub, sub);
            uint64_t       sum[2] = {0, 0};
            uint32_t       v[2][16];
            top = -INFINITY;
            ptx::tmem_ld_32x32b_x16(taddr, v[0]);
#pragma unroll
            for(int i = 0; i < 8; ++i)
            {
                ptx::tmem_ld_wait();
                if(i < 7)
                    ptx::tmem_ld_32x32b_x16(taddr + 16 * (i + 1), v[(i + 1) & 1]);
                change(16 * i, v[i & 1]);
                top = max_of(v[i & 1], top);
#pragma unroll
                for(int j = 0; j < 8; ++j)
                {
                    float x, y;
                    unpair(fma2(pair(__uint_as_float(v[i & 1][2 * j]), __uint_as_float(v[i & 1][2 * j + 1])), cc, ss), x, y);
                    x = ex2(x), y = ex2(y);
                    sum[j & 1]               = add2(sum[j & 1], pair(x, y));
                    w[i / 2][8 * (i & 1) + j] = pack2<T>(x, y);
                }
            }
            float a, b;
            unpair(add2(sum[0], sum[1]), a, b);
            return a + b;
        }

        // ---- results ----
        __device__ __forceinline__ void tma_store_4d(const void* tmap, int32_t c0, int32_t c1, int32_t c2, int32_t c3, uint32_t src_smem)
        {
            asm volatile("cp.async.bulk.tensor.4d.global.shared::cta.bulk_group [%0, {%1, %2, %3, %4}], [%5];" ::"l"(
                             reinterpret_cast<uint64_t>(tmap)),
                         "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(src_smem)
                         : "memory");
        }
        // 1 / l; NaN stays NaN
        __device__ __forceinline__ float inverse(float l)
        {
            return l > 0.0f ? 1.0f / l : l;
        }
        // Columns [from, to) of this thread's row of an fp32 accumulator, times `by`, as 16-bit values into row `row` of a tile in
        // shared memory with the 128-byte swizzle, from where TMA writes whole rows (a thread's own 16-byte stores to its row
        // would each touch a line of their own: 2.5 us for a tile).  `other`: a second accumulator (0: none), which counts `by2`
        // times.  A factor of 0 takes an accumulator out, whatever it holds.
        template <typename T>
        __device__ __forceinline__ void stage_row(uint8_t* tile, uint32_t row, uint32_t taddr, uint32_t from, uint32_t to, float by,
                                                  uint32_t other = 0, float by2 = 0.0f)
        {
#pragma unroll 1
            for(uint32_t c = from; c < to; c += 32)
            {
                uint32_t w[32];
                __syncwarp();
                ptx::tmem_ld_32x32b_x32(taddr + c, w);
                ptx::tmem_ld_wait();
#pragma unroll
                for(int i = 0; i < 32; ++i)
                    w[i] = by != 0.0f ? __float_as_uint(__uint_as_float(w[i]) * by) : 0u;
                if(other != 0)
                {
                    uint32_t x[32];
                    ptx::tmem_ld_32x32b_x32(other + c, x);
                    ptx::tmem_ld_wait();
#pragma unroll
                    for(int i = 0; i < 32; ++i)
                        w[i] = by2 != 0.0f ? __float_as_uint(fmaf(by2, __uint_as_float(x[i]), __uint_as_float(w[i]))) : w[i];
                }
#pragma unroll
                for(int i = 0; i < 4; ++i)
                {
                    uint32_t u[4];
#pragma unroll
                    for(int j = 0; j < 4; ++j)
                        u[j] = pack2<T>(__uint_as_float(w[8 * i + 2 * j]), __uint_as_float(w[8 * i + 2 * j + 1]));
                    const uint32_t at = c / 8 + i; // 16-byte piece of the row
                    *reinterpret_cast<uint4*>(tile + (at / 8) * BOX_BYTES + row * 128 + (((at % 8) ^ (row & 7u)) << 4)) = make_uint4(u[0], u[1], u[2], u[3]);
                }
            }
        }
        // One thread, after a barrier over those that staged (each with a proxy fence): writes the tile and waits until it has
        // been read.  Rows and columns out of bounds are left out.
        template <uint32_t HD>
        __device__ __forceinline__ void store_tile(const CUtensorMap* map, uint32_t tile_smem, uint32_t token, uint32_t head, uint32_t batch)
        {
#pragma unroll
            for(uint32_t s = 0; s < HD / 64; ++s)
                tma_store_4d(map, s * 64, token, head, batch, tile_smem + s * BOX_BYTES);
            ptx::bulk_commit_group();
            ptx::bulk_wait_group_read<0>();
        }

        // ---- masks by tile --------------------------------------------------------------------
        // Documents of a tile: {smallest, largest, any padding}; smallest > largest where there is nothing but padding.
        struct DocTile
        {
            int32_t lo, hi, neg, unused;
        };
        enum : uint32_t
        {
            TILE_NEED = 1, // some pair of the tile is visible
            TILE_MASK = 2, // some pair is not: each one is looked at
            TILE_DIRTY = 16, // the tile that is listed holds rows of padding
        };
        // Tile of queries [r0, r0 + 128) x keys [c0, c0 + 128).
        __device__ __forceinline__ uint32_t tile_flags(const Params& p, uint32_t r0, uint32_t c0, int32_t prefix, const DocTile* dq,
                                                       const DocTile* dk)
        {
            if(r0 >= p.len_q || c0 >= p.len_kv)
                return 0;
            const int32_t r1 = min(r0 + TILE, p.len_q) - 1, c1 = min(c0 + TILE, p.len_kv) - 1;
            bool          mask = c0 + TILE > p.len_kv;
            if(p.causal)
            {
                if(int32_t(c0) > r1 + p.off && int32_t(c0) >= prefix)
                    return 0;
                mask |= c1 > int32_t(r0) + p.off && c1 >= prefix;
            }
            if(dq)
            {
                const DocTile q = *dq, k = *dk;
                if(q.lo > q.hi || k.lo > k.hi || q.hi < k.lo || k.hi < q.lo)
                    return 0;
                mask |= q.neg || k.neg || q.lo != q.hi || k.lo != k.hi || q.lo != k.lo;
            }
            return TILE_NEED | (mask ? TILE_MASK : 0u);
        }

        // Bit i: document i of 32 N is `doc`, where lane l of the warp holds documents l, 32 + l, ... in `of`.  One round of votes
        // for each document that rows of the warp belong to, mostly one or two.
        template <int N>
        __device__ __forceinline__ void same_docs(const int32_t (&of)[N], int32_t doc, uint32_t (&same)[N])
        {
            uint32_t todo = 0xFFFFFFFFu;
            while(todo)
            {
                const int32_t d = __shfl_sync(0xFFFFFFFFu, doc, __ffs(todo) - 1);
                todo &= ~__ballot_sync(0xFFFFFFFFu, doc == d);
#pragma unroll
                for(int i = 0; i < N; ++i)
                {
                    const uint32_t vote = __ballot_sync(0xFFFFFFFFu, of[i] == d);
                    if(doc == d)
                        same[i] = vote;
                }
            }
        }
        // Bit i of word w: 32 w + i < count.
        __device__ __forceinline__ uint32_t below(int32_t count, int32_t w)
        {
            const int32_t n = count - 32 * w;
            return n >= 32 ? 0xFFFFFFFFu : n <= 0 ? 0u : (1u << n) - 1u;
        }

        // Lists tiles seg .. seg + count that flags_of(tile) says something about, as tile | flags << 24, in order.  Every
        // thread of the block calls it; `raw` holds SEG bytes, `list` SEG words, `length` one.  Returns the list's length.
        template <uint32_t THREADS, typename F>
        __device__ __forceinline__ uint32_t list_tiles(uint32_t seg, uint32_t count, uint32_t* list, uint8_t* raw, uint32_t* length, F flags_of)
        {
            for(uint32_t i = threadIdx.x; i < count; i += THREADS)
                raw[i] = static_cast<uint8_t>(flags_of(seg + i));
            __syncthreads();
            if(threadIdx.x < 32)
            {
                uint32_t n = 0;
                for(uint32_t i0 = 0; i0 < count; i0 += 32)
                {
                    const uint32_t f    = i0 + threadIdx.x < count ? raw[i0 + threadIdx.x] : 0u;
                    const uint32_t vote = __ballot_sync(0xFFFFFFFFu, f != 0);
                    if(f)
                        list[n + __popc(vote & ((1u << threadIdx.x) - 1u))] = (seg + i0 + threadIdx.x) | f << 24;
                    n += __popc(vote);
                }
                if(threadIdx.x == 0)
                    *length = n;
            }
            __syncthreads();
            return *length;
        }
        // One warp to a tile of a batch entry: total_q tiles of queries, then tiles of keys up to `total`.
        static __global__ void __launch_bounds__(128)
            doc_tiles_kernel(const int32_t* docs_q, uint32_t len_q, uint32_t tiles_q, uint32_t total_q, DocTile* out_q, const int32_t* docs_kv,
                             uint32_t len_kv, uint32_t tiles_kv, uint32_t total, DocTile* out_kv)
        {
            uint32_t       at = blockIdx.x * 4 + (threadIdx.x >> 5);
            const uint32_t lane = threadIdx.x & 31u;
            if(at >= total)
                return;
            const bool     kv = at >= total_q;
            const uint32_t tiles = kv ? tiles_kv : tiles_q, len = kv ? len_kv : len_q;
            DocTile*       out = kv ? out_kv : out_q;
            if(kv)
                at -= total_q;
            const int32_t* d  = (kv ? docs_kv : docs_q) + size_t(at / tiles) * len;
            const uint32_t i0 = at % tiles * TILE;
            int32_t        lo = INT32_MAX, hi = -1, neg = 0;
            for(uint32_t i = i0 + lane; i < min(i0 + TILE, len); i += 32)
                if(d[i] < 0)
                    neg = 1;
                else
                    lo = min(lo, d[i]), hi = max(hi, d[i]);
            lo  = __reduce_min_sync(0xFFFFFFFFu, lo);
            hi  = __reduce_max_sync(0xFFFFFFFFu, hi);
            neg = __any_sync(0xFFFFFFFFu, neg);
            if(lane == 0)
                out[at] = {lo, hi, neg, 0};
        }

        // ---- scores ---------------------------------------------------------------------------
        // Constants of a score in units of log 2: x = log2(e) * (cap * tanh(scale * dot / cap) - slope * distance).
        struct ScoreConst
        {
            float c;     // log2(e) * scale (no cap)
            float k1;    // 2 log2(e) scale / cap: e^(2 scale dot / cap) = 2^(k1 dot)
            float k2;    // scale / cap: the argument of tanh is k2 dot
            float cap2;  // log2(e) * cap
            float slope; // log2(e) * slope of this head
        };
        __device__ __forceinline__ ScoreConst score_const(const Params& p, uint32_t head)
        {
            ScoreConst s;
            s.c     = p.scale * LOG2E;
            s.k2    = p.cap > 0.0f ? p.scale / p.cap : 0.0f;
            s.k1    = 2.0f * LOG2E * s.k2;
            s.cap2  = p.cap * LOG2E;
            s.slope = p.slopes ? p.slopes[head] * LOG2E : 0.0f;
            return s;
        }
        // Largest magnitude of N numbers and `t`.
        template <int N>
        __device__ __forceinline__ float magnitude(const uint32_t (&v)[N], float t)
        {
            float u = 0.0f;
#pragma unroll
            for(int k = 0; k < N; k += 4)
            {
                t = fmaxf(fmaxf(t, fabsf(__uint_as_float(v[k]))), fabsf(__uint_as_float(v[k + 1])));
                u = fmaxf(fmaxf(u, fabsf(__uint_as_float(v[k + 2]))), fabsf(__uint_as_float(v[k + 3])));
            }
            return fmaxf(t, u);
        }
        // True where the cap bends the scores of a warp only a little: |k2 dot| <= 1/2, as mostly (NaN counts as small).
        constexpr float TAME_LIMIT = 0.5f;
        template <bool CAP>
        __device__ __forceinline__ bool tame(const ScoreConst& s, float largest)
        {
            if constexpr(CAP)
                return __all_sync(0xFFFFFFFFu, largest * fabsf(s.k2) <= TAME_LIMIT);
            else
                return true;
        }
        template <bool CAP, int N>
        __device__ __forceinline__ bool tame(const ScoreConst& s, const uint32_t (&dot)[N])
        {
            return tame<CAP>(s, CAP ? magnitude(dot, 0.0f) : 0.0f);
        }
        // How scores of a warp are bent: all of them a little, or not; the latter under any cap, or under one of at most MODEST_CAP.
        enum Bend : int
        {
            TAME,
            MODEST,
            ANY
        };
        template <Bend B>
        using Bent = std::integral_constant<Bend, B>;
        // tanh x of two x = k2 dot.
        // TAME (|x| <= 1/2): tanh x / x as a polynomial in x^2, fitted to the smallest largest error: 1.5e-8 of its value, 4e-8 as
        // evaluated in fp32.
        // MODEST: 1 - 2 / (1 + 2^(k1 dot)), off by some ulp of 1: a score by up to 1.3e-7 of the cap, 8e-6 at the largest that this is
        // for, which is nothing next to the rounding of its weight to 16 bits (the hardware's tanh approximation is off by 2^-11 of its
        // value: a capped score of 20 would move by 0.01).  An infinite or zero power gives 1 and -1.  Its three numbers of a score and
        // the softmax's exponential share a unit that takes 16 numbers a cycle: 2 x 16 heads of 4096 x 128, causal, 187 us with the
        // polynomial, 254 us with this.
        // ANY: each by its own size, off by a few ulp of itself, as the cap may be much larger than a score (scores around a cap of 2,
        // 2 x 16 heads of 4096 x 128, causal: 346 us, MODEST 301).
        // NaN stays NaN.
        constexpr float MODEST_CAP = 64.0f;
        template <Bend HOW>
        __device__ __forceinline__ uint64_t tanh2(const ScoreConst& s, uint64_t dot)
        {
            uint64_t u = 0, near = 0, far = 0;
            if constexpr(HOW != MODEST)
            {
                u = mul2(dot, pair(s.k2, s.k2));
                const uint64_t y = mul2(u, u);
                uint64_t       q = fma2(y, pair(0.0172414854f, 0.0172414854f), pair(-0.0530454926f, -0.0530454926f));
                q    = fma2(q, y, pair(0.13325879f, 0.13325879f));
                q    = fma2(q, y, pair(-0.333331436f, -0.333331436f));
                q    = fma2(q, y, pair(1.0f, 1.0f));
                near = mul2(u, q);
            }
            if constexpr(HOW != TAME)
            {
                float a, b;
                unpair(mul2(dot, pair(s.k1, s.k1)), a, b);
                unpair(add2(pair(ex2(a), ex2(b)), pair(1.0f, 1.0f)), a, b);
                far = fma2(pair(rcp(a), rcp(b)), pair(-2.0f, -2.0f), pair(1.0f, 1.0f));
            }
            if constexpr(HOW == ANY)
            {
                float x[2], t[2], f[2];
                unpair(u, x[0], x[1]);
                unpair(near, t[0], t[1]);
                unpair(far, f[0], f[1]);
                return pair(fabsf(x[0]) > TAME_LIMIT ? f[0] : t[0], fabsf(x[1]) > TAME_LIMIT ? f[1] : t[1]);
            }
            else
                return HOW == TAME ? near : far;
        }
        // Calls f with the Bend of a warp's scores.
        template <bool CAP, typename F>
        __device__ __forceinline__ void bend(const ScoreConst& s, bool all_tame, F f)
        {
            if(!CAP || all_tame)
                f(Bent<TAME>{});
            else if(__builtin_expect(s.cap2 > MODEST_CAP * LOG2E, false))
                f(Bent<ANY>{});
            else
                f(Bent<MODEST>{});
        }
        // Two scores whose distances are `dist` and `dist` + `step`, without a cap and from their tanh; the cap's derivative there.
        template <bool BIAS>
        __device__ __forceinline__ uint64_t biased(const ScoreConst& s, uint64_t x, float dist, float step)
        {
            if constexpr(BIAS)
            {
                float a, b;
                unpair(x, a, b);
                x = pair(fmaf(-s.slope, fabsf(dist), a), fmaf(-s.slope, fabsf(dist + step), b));
            }
            return x;
        }
        template <bool BIAS>
        __device__ __forceinline__ uint64_t capped(const ScoreConst& s, uint64_t tanh, float dist, float step)
        {
            return biased<BIAS>(s, mul2(tanh, pair(s.cap2, s.cap2)), dist, step);
        }
        __device__ __forceinline__ uint64_t slip_of(uint64_t tanh)
        {
            return fma2(mul2(tanh, pair(-1.0f, -1.0f)), tanh, pair(1.0f, 1.0f));
        }
        // Either of them; slip: the cap's derivative.
        template <bool CAP, bool BIAS, Bend HOW>
        __device__ __forceinline__ uint64_t score2(const ScoreConst& s, uint64_t dot, float dist, float step, uint64_t& slip)
        {
            if constexpr(CAP)
            {
                const uint64_t tanh = tanh2<HOW>(s, dot);
                slip = slip_of(tanh);
                return capped<BIAS>(s, tanh, dist, step);
            }
            else
                return biased<BIAS>(s, mul2(dot, pair(s.c, s.c)), dist, step);
        }

        // ---- host side ------------------------------------------------------------------------
        // [batch][tokens][heads][dim] with free strides, in boxes of 64 elements x box_tokens tokens; zero fill out of bounds.
        static int make_map(CUtensorMap* out, int data_type, const void* ptr, uint32_t dim, uint32_t tokens, uint32_t heads, uint32_t batch,
                            const Strides& s, uint32_t box_tokens = TILE)
        {
            tc05::EncodeTiledFn fn = tc05::get_encode_fn();
            B200_REQUIRE(fn != nullptr, B200WMMA_ERR_CUDA, "cuTensorMapEncodeTiled not available");
            cuuint64_t gdim[4]    = {dim, tokens, heads, batch};
            cuuint64_t gstride[3] = {cuuint64_t(s.token) * 2, cuuint64_t(s.head) * 2, cuuint64_t(s.batch) * 2};
            cuuint32_t box[4]     = {64, box_tokens, 1, 1};
            cuuint32_t estr[4]    = {1, 1, 1, 1};
            CUresult   r          = fn(out, data_type == B200WMMA_OUT_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4,
                            const_cast<void*>(ptr), gdim, gstride, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
            B200_REQUIRE(r == CUDA_SUCCESS, B200WMMA_ERR_CUDA, "cuTensorMapEncodeTiled (attention operand) failed with CUresult %d",
                         static_cast<int>(r));
            return B200WMMA_OK;
        }
    } // namespace attn
} // namespace b200wmma
