// Products of 4-bit weights with several vectors on tcgen05: the form that gemv_w4.cu takes beyond a few vectors.
//
// A block owns 128 outputs, one to a thread of each of two groups that take 128-column chunks in turn.  A thread turns its row's
// 64 bytes into 16-bit numbers and writes them to tensor memory, where they are the left operand of D = W X (M = 128, N = 16 to
// 64 vectors); the right operand, x, comes by TMA and is paired up in place by two warps.  A weight is converted once for
// all vectors, by 9 (fp16) or 11 (bf16) instructions to a word of eight.
// Sums of a group come out of tensor memory and are scaled and added up in fp32 registers: chunks hold 1, 2 or 4 groups (SETS),
// each with an accumulator of its own; other groups (multiples of 32) are taken as blocks of 32 columns.
#pragma once
#include "attn_tc05.cuh"

namespace b200wmma
{
    namespace gemv_w4
    {
        constexpr uint32_t TC_THREADS = 384; // warps 0-3: even chunks, 4-7: odd chunks, 8: products, 9-10: pair up x, 11: copies x
        constexpr uint32_t TC_K = 128, TC_M = 128; // columns of a chunk, outputs of a block

        template <int N, int SETS>
        struct TcSmem
        {
            static constexpr uint32_t W_STAGES = 8; // chunks of a group of threads on their way
            static constexpr uint32_t TC_X     = N == 16 ? 8 : N == 32 ? 6 : 4; // stages of x
            static constexpr uint32_t W_STAGE = TC_M * TC_K / 2, X_STAGE = N * TC_K * 2;
            static constexpr uint32_t X = 0, W = TC_X * X_STAGE, BARS = W + 2 * W_STAGES * W_STAGE;
            static constexpr uint32_t X_RAW = BARS, X_FULL = X_RAW + 8 * TC_X, X_EMPTY = X_FULL + 8 * TC_X, A_FULL = X_EMPTY + 8 * TC_X, D_FULL = A_FULL + 32, MISC = D_FULL + 32; // [group][buffer]
            static constexpr uint32_t BYTES   = MISC + 16 + 1024;
            static_assert(256 + 4 * SETS * N <= 512, "tensor memory: two operands and two sets of accumulators for each group");
            static_assert(2 * W_STAGES * W_STAGE >= TC_M * N * 4, "sums reuse the ring");
        };
        enum TcRole : uint32_t
        {
            W4_MMA     = 0x81,
            W4_X       = 0x82,
            W4_CONVERT = 0x83
        };

        template <typename T, bool SIGNED, int N, int SETS>
        __global__ void __launch_bounds__(TC_THREADS, 1)
            tc_kernel(const __grid_constant__ Args p, uint32_t parts, unsigned* status, const __grid_constant__ CUtensorMap map_x)
        {
            using L                 = TcSmem<N, SETS>;
            constexpr uint32_t TC_X = L::TC_X;
            extern __shared__ uint8_t smem_raw[];
            const uint32_t     base = (ptx::smem_u32(smem_raw) + 1023u) & ~1023u;
            uint8_t*           smem = smem_raw + (base - ptx::smem_u32(smem_raw));
            uint32_t*          misc = reinterpret_cast<uint32_t*>(smem + L::MISC);
            volatile uint32_t* cta_abort = misc + 1;
            const uint32_t     tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u;
            const uint32_t     part_id = parts > 1 ? blockIdx.x % parts : 0, row0 = (parts > 1 ? blockIdx.x / parts : blockIdx.x) * TC_M;
            const uint32_t     vec0 = blockIdx.y * N, all = (p.n + TC_K - 1) / TC_K;
            const uint32_t     from = uint32_t(uint64_t(all) * part_id / parts), chunks = uint32_t(uint64_t(all) * (part_id + 1) / parts) - from;

            if(tid == 0)
            {
                for(uint32_t s = 0; s < TC_X; ++s)
                {
                    ptx::mbar_init(base + L::X_RAW + 8 * s, 1);
                    ptx::mbar_init(base + L::X_FULL + 8 * s, 1);
                    ptx::mbar_init(base + L::X_EMPTY + 8 * s, 1);
                }
                for(uint32_t u = 0; u < 4; ++u)
                {
                    ptx::mbar_init(base + L::A_FULL + 8 * u, 4);
                    ptx::mbar_init(base + L::D_FULL + 8 * u, 1);
                }
                *cta_abort = 0u;
                ptx::fence_barrier_init();
                ptx::fence_proxy_async_smem();
            }
            if(warp == 8)
            {
                ptx::tmem_alloc(base + L::MISC, 512);
                ptx::tmem_relinquish();
            }
            ptx::tc_fence_before_sync();
            __syncthreads();
            ptx::tc_fence_after_sync();
            const uint32_t tmem = misc[0]; // operand of buffer w (group u: 2 u and 2 u + 1): + 64 w; its accumulators: + 256 + w SETS N
            bool           ok = true;
            float          sum[N];
#pragma unroll
            for(int i = 0; i < N; ++i)
                sum[i] = 0.0f;

            if(warp == 8)
            {
                constexpr uint32_t idesc = tc05::make_idesc<attn::kind_of<T>, TC_M, N>();
                for(uint32_t c = 0; ok && c < chunks; ++c)
                {
                    const uint32_t w = 2 * (c & 1u) + (c >> 1 & 1u), st = c % TC_X;
                    ok = attn::wait_bounded_warp(base + L::X_FULL + 8 * st, c / TC_X & 1u, cta_abort, status, W4_MMA << 24 | (blockIdx.x & 0xFFFFFFu))
                         && attn::wait_bounded_warp(base + L::A_FULL + 8 * w, c >> 2 & 1u, cta_abort, status,
                                                    W4_MMA << 24 | 1u << 20 | (blockIdx.x & 0xFFFFFu));
                    if(!ok)
                        break;
                    ptx::tc_fence_after_sync();
                    if(attn::elect_one())
                    {
                        const uint64_t b = ptx::make_kmajor_sw128_desc(base + L::X + st * L::X_STAGE);
#pragma unroll
                        for(uint32_t k = 0; k < TC_K / 16; ++k)
                        {
                            constexpr uint32_t PER = TC_K / 16 / SETS; // steps of a set
                            attn::mma_f16_ts(tmem + 256 + (w * SETS + k / PER) * N, tmem + 64 * w + 8 * k, b + (k / 4) * (N * 128 >> 4) + (k % 4) * 2, idesc,
                                             k % PER != 0);
                        }
                        ptx::tc_commit(base + L::D_FULL + 8 * w);
                        ptx::tc_commit(base + L::X_EMPTY + 8 * st);
                    }
                }
                __syncwarp();
            }
            else if(warp == 11)
            {
                for(uint32_t c = 0; ok && c < chunks; ++c)
                {
                    const uint32_t st = c % TC_X, raw = base + L::X_RAW + 8 * st;
                    ok = attn::wait_bounded_warp(base + L::X_EMPTY + 8 * st, (c / TC_X & 1u) ^ 1u, cta_abort, status,
                                                 W4_X << 24 | (blockIdx.x & 0xFFFFFFu));
                    if(ok && attn::elect_one())
                    {
                        ptx::mbar_arrive_expect_tx(raw, L::X_STAGE);
                        for(uint32_t b = 0; b < 2; ++b) // boxes of 64 columns x N vectors; what lies out of bounds reads as zeros
                            ptx::tma_load_2d(base + L::X + st * L::X_STAGE + b * (N * 128), &map_x, (from + c) * TC_K + b * 64, vec0, raw);
                    }
                }
                __syncwarp();
            }
            else if(warp >= 9)
            {
                for(uint32_t c = warp - 9; ok && c < chunks; c += 2)
                {
                    const uint32_t st = c % TC_X, at = base + L::X + st * L::X_STAGE + lane * 16;
                    ok = attn::wait_bounded_warp(base + L::X_RAW + 8 * st, c / TC_X & 1u, cta_abort, status,
                                                 W4_X << 24 | 1u << 20 | (blockIdx.x & 0xFFFFFu));
                    if(!ok)
                        break;
                    constexpr int PIECES = N * (TC_K / 8) / 32, BATCH = 8; // 16-byte pieces of a lane, wherever the swizzle put them
#pragma unroll
                    for(int i0 = 0; i0 < PIECES; i0 += BATCH)
                    {
                        uint4 w[BATCH];
#pragma unroll
                        for(int i = 0; i < BATCH; ++i)
                            w[i] = lds128(at + (i0 + i) * 512);
#pragma unroll
                        for(int i = 0; i < BATCH; ++i)
                            sts128(at + (i0 + i) * 512, pair_up(w[i]));
                    }
                    ptx::fence_proxy_async_smem();
                    __syncwarp();
                    if(lane == 0)
                        ptx::mbar_arrive(base + L::X_FULL + 8 * st);
                }
                __syncwarp();
            }
            else
            {
                const uint32_t u = warp >> 2, quad = warp & 3u, row = min(row0 + quad * 32 + lane, p.m - 1);
                const uint32_t mine = chunks > u ? (chunks - u + 1) / 2 : 0; // chunks u, u + 2, ...
                const uint32_t lane_tmem = (quad * 32u) << 16, a_tmem = tmem + 128 * u + lane_tmem, d_tmem = tmem + 256 + 2 * u * SETS * N + lane_tmem;
                const uint32_t ring = base + L::W + u * L::W_STAGES * L::W_STAGE;
                const uint16_t* scales = static_cast<const uint16_t*>(p.scales) + size_t(row) * p.ld_scales;
                const uint8_t*  zeros  = SIGNED ? nullptr : p.zeros + size_t(row) * p.ld_zeros;
                // a stage is [piece of 16 bytes][row]; a warp copies its own 32 rows, four lanes to the 64 bytes of a row
                const auto fetch = [&](uint32_t i) {
                    const uint32_t k = (from + u + 2 * i) * TC_K + (lane & 3u) * 32, to = ring + (i % L::W_STAGES) * L::W_STAGE + (lane & 3u) * (TC_M * 16);
                    const bool     there = k < p.n;
#pragma unroll
                    for(uint32_t j = 0; j < 4; ++j)
                    {
                        const uint32_t r = quad * 32 + j * 8 + (lane >> 2);
                        copy16(to + r * 16, p.a + size_t(min(row0 + r, p.m - 1)) * p.lda + (there ? k / 2 : 0), there);
                    }
                };
                uint32_t   scale[2][SETS], next_scale[SETS], next_zero[SETS];
                const auto groups = [&](uint32_t i) {
#pragma unroll
                    for(int s = 0; s < SETS; ++s)
                    {
                        const uint32_t g = min(((from + u + 2 * i) * TC_K + s * (TC_K / SETS)) / p.group, p.groups - 1);
                        next_scale[s]    = __ldg(scales + g);
                        next_zero[s]     = SIGNED ? 8u : __ldg(zeros + g) & 15u;
                    }
                };
                const auto flush = [&](uint32_t i, uint32_t w) { // sums of chunk i of this group of threads, buffer w = i % 2
                    ok = attn::wait_bounded_warp(base + L::D_FULL + 8 * (2 * u + w), i >> 1 & 1u, cta_abort, status,
                                                 W4_CONVERT << 24 | (blockIdx.x & 0xFFFFFFu));
                    if(!ok)
                        return;
                    ptx::tc_fence_after_sync();
#pragma unroll
                    for(int s = 0; s < SETS; ++s)
                    {
                        const float f = tc05::Pack16<T>::widen(scale[w][s]).x;
#pragma unroll
                        for(int c0 = 0; c0 < N; c0 += 16)
                        {
                            uint32_t d[16];
                            ptx::tmem_ld_32x32b_x16(d_tmem + (w * SETS + s) * N + c0, d);
                            ptx::tmem_ld_wait();
#pragma unroll
                            for(int k = 0; k < 16; ++k)
                                sum[c0 + k] = fmaf(f, __uint_as_float(d[k]), sum[c0 + k]);
                        }
                    }
                };
#pragma unroll
                for(uint32_t i = 0; i < L::W_STAGES; ++i)
                {
                    if(i < mine)
                        fetch(i);
                    copy_commit();
                }
                if(mine)
                    groups(0);
                const auto convert = [&](uint32_t i, auto buffer) {
                    constexpr uint32_t w = decltype(buffer)::value;
                    copy_wait<L::W_STAGES - 1>();
                    __syncwarp();
                    const uint32_t at = ring + (i % L::W_STAGES) * L::W_STAGE + (quad * 32 + lane) * 16;
                    const auto     half = [&](uint32_t h, uint32_t(&a)[32]) { // 64 weights
#pragma unroll
                        for(uint32_t c = 0; c < 2; ++c)
                        {
                            const uint4    x = lds128(at + (2 * h + c) * (TC_M * 16));
                            const uint32_t xs[4] = {x.x, x.y, x.z, x.w};
                            Offset<T>      z;
                            z.set(next_zero[(2 * h + c) * SETS / 4]);
#pragma unroll
                            for(uint32_t j = 0; j < 4; ++j)
                            {
                                uint32_t q[4];
                                unpack<T, SIGNED>(xs[j], z, q);
#pragma unroll
                                for(uint32_t k = 0; k < 4; ++k)
                                    a[c * 16 + j * 4 + k] = q[k];
                            }
                        }
                    };
                    uint32_t a[32];
                    half(0, a);
                    if(i >= 2)
                    {
                        flush(i - 2, w); // and with it the products have read the buffer
                        if(!ok)
                            return;
                    }
                    attn::tmem_st_32x32b_x32(a_tmem + 64 * w, a);
                    half(1, a);
                    attn::tmem_st_32x32b_x32(a_tmem + 64 * w + 32, a);
#pragma unroll
                    for(int s = 0; s < SETS; ++s)
                        scale[w][s] = next_scale[s];
                    if(i + 1 < mine)
                        groups(i + 1);
                    attn::tmem_st_wait();
                    ptx::tc_fence_before_sync();
                    __syncwarp(); // and everyone has read the stage
                    if(lane == 0)
                        ptx::mbar_arrive(base + L::A_FULL + 8 * (2 * u + w));
                    if(i + L::W_STAGES < mine)
                        fetch(i + L::W_STAGES);
                    copy_commit();
                };
                for(uint32_t i = 0; ok && i < mine; i += 2)
                {
                    convert(i, std::integral_constant<uint32_t, 0>{});
                    if(ok && i + 1 < mine)
                        convert(i + 1, std::integral_constant<uint32_t, 1>{});
                }
                // the last two, in order
                if(mine >= 2 && ok)
                {
                    if(mine & 1u)
                        flush(mine - 2, 1);
                    else
                        flush(mine - 2, 0);
                }
                if(mine >= 1 && ok)
                {
                    if(mine & 1u)
                        flush(mine - 1, 0);
                    else
                        flush(mine - 1, 1);
                }
                copy_wait<0>();
            }
            __syncthreads(); // every copy has landed and been read: the ring is free
            // the sums of both groups of threads as [vector][output]
            float* red = reinterpret_cast<float*>(smem + L::W);
            if(warp >= 4 && warp < 8)
#pragma unroll
                for(int i = 0; i < N; ++i)
                    red[i * TC_M + (tid & 127u)] = sum[i];
            __syncthreads();
            if(warp < 4)
#pragma unroll
                for(int i = 0; i < N; ++i)
                    red[i * TC_M + tid] += sum[i];
            if(parts > 1)
                ptx::cluster_sync();
            else
                __syncthreads();
            // the blocks of a cluster share the outputs among them
            const uint32_t vecs = min(uint32_t(N), p.rows - vec0);
            for(uint32_t e = part_id * TC_THREADS + tid; e < TC_M * vecs && !*cta_abort; e += parts * TC_THREADS)
            {
                const uint32_t r = vec0 + e / TC_M, i = row0 + e % TC_M;
                if(i >= p.m)
                    continue;
                put<T>(p, r, i, parts > 1 ? cluster_sum(red + e, parts) : red[e]);
            }
            if(parts > 1)
                ptx::cluster_sync(); // no block leaves while another reads its sums
            ptx::tc_fence_before_sync();
            __syncthreads();
            if(*cta_abort)
            {
                // A wait was abandoned: products may still be in flight.  Give them a bounded grace period.
                const uint64_t t0 = ptx::globaltimer_ns();
                while(ptx::globaltimer_ns() - t0 < 2000000ull)
                    __nanosleep(1000);
                __syncthreads();
            }
            if(warp == 8)
            {
                ptx::tc_fence_after_sync();
                ptx::tmem_dealloc(tmem, 512);
            }
        }
    } // namespace gemv_w4
} // namespace b200wmma
