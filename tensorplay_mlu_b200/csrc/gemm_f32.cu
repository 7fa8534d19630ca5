// float32 feed-forward products at fp32 accuracy on the tensor cores, one
// launch each: the forward layers with their epilogue, dz w and dz^T x.
//
// Every operand element is split on its way into shared memory, x = hi + lo
// with hi = tf32(x) and lo = tf32(x - hi) (round to nearest), and a product is
// hi hi + hi lo + lo hi: three TF32 MMAs.  The dropped lo lo and the rounding
// of lo are 2^-22 of |a b|.  The tensor core rounds its running sum towards
// zero, so a TMEM accumulator only takes kChain k-blocks (kChain * 32 terms);
// warps of their own then add it to fp32 sums in registers, rounded to
// nearest, while the MMAs fill the other accumulator.
//
// Why not pre-split copies and library-style tiles: those write and read each
// operand three times and take a launch per chunk of K; for the sizes of a
// layer (512 x 1024 x 4096) the launches alone cost more than the product.
//
// Operands are read with plain loads (any strides, no alignment needed: a
// transposed operand is read along its unit stride and transposed by the
// shared-memory store), two or three k-blocks ahead in registers.  As in
// gemm_few.cu a tile is 128 result columns by kNT rows, and a cluster shares K.
//
// Infinities and NaN: hi = inf makes lo = NaN, and values within half a TF32
// step of the largest float round to inf, so such a sum comes out NaN; every
// NaN sum is recomputed as a plain fp32 dot product, which gives the infinity
// or NaN that fp32 arithmetic gives.

#include "gemm_few.cuh"

namespace tpb {
namespace {

constexpr int kLoadWarps = 8;
constexpr int kChain = 4;

struct F32Operands {
    const float* w;  // element (n, k) at w + n * sw_n + k * sw_k
    int64_t sw_n, sw_k;
    const float* x;  // element (m, k) at x + m * sx_m + k * sx_k
    int64_t sx_m, sx_k;
    int vec_w, vec_x;  // 16-byte loads along k
    int tf32;          // one TF32 product is enough
};

template <int NT>
struct F32Shape {
    static constexpr uint32_t kWBytes = 128 * 128;  // 128 rows of 32 floats
    static constexpr uint32_t kXBytes = NT * 128;
    static constexpr uint32_t kStageBytes = 2 * (kWBytes + kXBytes);
    static constexpr int kStages = int(200 * 1024 / kStageBytes);
    static constexpr int kAccWarps = NT == 128 ? 8 : 4;
    static constexpr int kAccCols = NT * 4 / kAccWarps;  // columns an accumulator warp sums
    static constexpr int kThreads = 32 * (kLoadWarps + 1 + kAccWarps);
    static constexpr int kDepth = NT == 128 ? 2 : 3;  // k-blocks in registers
    static constexpr size_t kSmem = size_t(kStages) * kStageBytes + 1024 + 256;
    static constexpr int kTmemCols = 2 * NT;
    static_assert(NT * 512 <= kStages * int(kStageBytes), "partial sums fit the stages");
};

// Four consecutive k of one row (zero outside).
template <bool MN>
__device__ __forceinline__ float4 load_chunk(const float* base, int64_t s_row, int64_t s_k, int64_t row, bool row_ok,
                                             int k, int K, bool vec) {
    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (!row_ok) return v;
    if constexpr (MN) {
        const float* p = base + row + int64_t(k) * s_k;
        if (k < K) v.x = p[0];
        if (k + 1 < K) v.y = p[s_k];
        if (k + 2 < K) v.z = p[2 * s_k];
        if (k + 3 < K) v.w = p[3 * s_k];
    } else {
        const float* p = base + row * s_row + k;
        if (vec && k + 4 <= K) {
            v = *reinterpret_cast<const float4*>(p);
        } else {
            if (k < K) v.x = p[0];
            if (k + 1 < K) v.y = p[1];
            if (k + 2 < K) v.z = p[2];
            if (k + 3 < K) v.w = p[3];
        }
    }
    return v;
}

__device__ __forceinline__ float tf32_of(float x) {
    uint32_t u;
    asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(u) : "f"(x));
    return __uint_as_float(u & 0xffffe000u);
}

// hi and lo of a chunk to row r, chunk q of their swizzled tiles.
__device__ __forceinline__ void store_split(uint8_t* hi_tile, uint8_t* lo_tile, int r, int q, float4 v) {
    const int at = r * 128 + ((q ^ (r & 7)) << 4);
    const float4 h = make_float4(tf32_of(v.x), tf32_of(v.y), tf32_of(v.z), tf32_of(v.w));
    *reinterpret_cast<float4*>(hi_tile + at) = h;
    *reinterpret_cast<float4*>(lo_tile + at) =
        make_float4(tf32_of(v.x - h.x), tf32_of(v.y - h.y), tf32_of(v.z - h.z), tf32_of(v.w - h.w));
}

template <int PARTS, int NT, bool W_MN, bool X_MN>
__global__ void __launch_bounds__(F32Shape<NT>::kThreads, 1) gemm_f32_kernel(const FewParams p, const F32Operands o) {
    using S = F32Shape<NT>;
    constexpr int kStages = S::kStages;
    constexpr int kColumns = 128 / PARTS;
    constexpr int kWChunks = 128 * 8 / (kLoadWarps * 32);
    constexpr int kXChunks = NT * 8 / (kLoadWarps * 32);
    constexpr int kDepth = S::kDepth;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + kStages * S::kStageBytes);
    uint64_t* empty = full + kStages;
    uint64_t* acc_full = empty + kStages;
    uint64_t* acc_empty = acc_full + 2;
    uint64_t* drain = acc_empty + 2;
    volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(drain + 1);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    pdl_trigger();
    const int ranks = int(cluster_size());
    const int rank = int(cluster_ctarank());
    const int tile = blockIdx.x / ranks;
    const int wt = tile / p.row_tiles, mt = tile - wt * p.row_tiles;
    const int n0 = wt * kColumns, m0 = mt * NT;
    const int kb0 = int(int64_t(p.k_blocks) * rank / ranks), kb1 = int(int64_t(p.k_blocks) * (rank + 1) / ranks);

    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(smem_addr(&full[s]), kLoadWarps);
            mbar_init(smem_addr(&empty[s]), 1);
        }
        for (int a = 0; a < 2; ++a) {
            mbar_init(smem_addr(&acc_full[a]), 1);
            mbar_init(smem_addr(&acc_empty[a]), S::kAccWarps);
        }
        mbar_init(smem_addr(drain), 1);
        *abort_flag = 0;
        mbar_fence_init();
    }
    if (warp == kLoadWarps) {
        tmem_alloc(smem_addr(const_cast<uint32_t*>(tmem_slot)), S::kTmemCols);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    pdl_wait();

    if (warp < kLoadWarps) {
        // ------------------------------------------------- load and split --
        float4 reg[kDepth][kWChunks + kXChunks];
        const auto row_of = [](bool mn, int c, int rows) { return mn ? c % rows : c >> 3; };
        const auto part_of = [](bool mn, int c, int rows) { return mn ? c / rows : c & 7; };
        const auto fetch = [&](int kb, float4 (&r)[kWChunks + kXChunks]) {
            if (kb >= kb1) return;
#pragma unroll
            for (int i = 0; i < kWChunks; ++i) {
                const int c = int(threadIdx.x) + i * kLoadWarps * 32;
                const int row = row_of(W_MN, c, 128), q = part_of(W_MN, c, 128);
                const int col = n0 + row % kColumns;
                r[i] = load_chunk<W_MN>(o.w, o.sw_n, o.sw_k, col + int64_t(row / kColumns) * p.N, col < p.N,
                                        kb * 32 + q * 4, p.K, o.vec_w);
            }
#pragma unroll
            for (int i = 0; i < kXChunks; ++i) {
                const int c = int(threadIdx.x) + i * kLoadWarps * 32;
                const int row = m0 + row_of(X_MN, c, NT), q = part_of(X_MN, c, NT);
                r[kWChunks + i] = load_chunk<X_MN>(o.x, o.sx_m, o.sx_k, row, row < p.M, kb * 32 + q * 4, p.K, o.vec_x);
            }
        };
#pragma unroll
        for (int d = 0; d < kDepth - 1; ++d) fetch(kb0 + d, reg[d]);
        int stage = 0;
        uint32_t phase = 0;
        bool ok = true;
        for (int kb = kb0; kb < kb1 && ok; kb += kDepth) {
#pragma unroll
            for (int d = 0; d < kDepth; ++d) {
                if (kb + d >= kb1 || !ok) break;
                fetch(kb + d + kDepth - 1, reg[(d + kDepth - 1) % kDepth]);
                int granted = 1;
                if (lane == 0) granted = mbar_wait(smem_addr(&empty[stage]), phase ^ 1, abort_flag) ? 1 : 0;
                ok = __shfl_sync(0xffffffffu, granted, 0) != 0;
                if (!ok) break;
                uint8_t* at = smem + stage * S::kStageBytes;
#pragma unroll
                for (int i = 0; i < kWChunks; ++i) {
                    const int c = int(threadIdx.x) + i * kLoadWarps * 32;
                    store_split(at, at + S::kWBytes, row_of(W_MN, c, 128), part_of(W_MN, c, 128), reg[d][i]);
                }
#pragma unroll
                for (int i = 0; i < kXChunks; ++i) {
                    const int c = int(threadIdx.x) + i * kLoadWarps * 32;
                    store_split(at + 2 * S::kWBytes, at + 2 * S::kWBytes + S::kXBytes, row_of(X_MN, c, NT),
                                part_of(X_MN, c, NT), reg[d][kWChunks + i]);
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_addr(&full[stage]));
                if (++stage == kStages) {
                    stage = 0;
                    phase ^= 1;
                }
            }
        }
        if (!ok && lane == 0) atomicExch(p.err, kErrProducer);
    } else if (warp == kLoadWarps) {
        // ------------------------------------------------------ MMA issuer --
        if (lane == 0) {
            int stage = 0;
            uint32_t phase = 0;
            bool ok = true;
            for (int i = 0; i < kb1 - kb0 && ok; ++i) {
                const int chain = i / kChain, acc = chain & 1;
                if (i % kChain == 0 && !mbar_wait(smem_addr(&acc_empty[acc]), ((chain >> 1) & 1) ^ 1, abort_flag)) {
                    ok = false;
                    break;
                }
                if (!mbar_wait(smem_addr(&full[stage]), phase, abort_flag)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                const uint32_t w_hi = smem_addr(smem + stage * S::kStageBytes), w_lo = w_hi + S::kWBytes;
                const uint32_t x_hi = w_lo + S::kWBytes, x_lo = x_hi + S::kXBytes;
                const uint32_t d = tmem + acc * NT;
#pragma unroll
                for (int kk = 0; kk < 4; ++kk) {
                    const uint64_t wh = sw128_desc(w_hi + kk * 32, 16, 1024), xh = sw128_desc(x_hi + kk * 32, 16, 1024);
                    uint32_t more = (i % kChain != 0 || kk > 0) ? 1u : 0u;
                    if (!o.tf32) {  // the small terms first
                        umma<true>(d, sw128_desc(w_lo + kk * 32, 16, 1024), xh, p.idesc, more);
                        umma<true>(d, wh, sw128_desc(x_lo + kk * 32, 16, 1024), p.idesc, 1u);
                        more = 1u;
                    }
                    umma<true>(d, wh, xh, p.idesc, more);
                }
                umma_commit(smem_addr(&empty[stage]));
                if (i % kChain == kChain - 1 || i == kb1 - kb0 - 1) umma_commit(smem_addr(&acc_full[acc]));
                if (++stage == kStages) {
                    stage = 0;
                    phase ^= 1;
                }
            }
            if (!ok) atomicExch(p.err, kErrMma);
            umma_commit(smem_addr(drain));
            if (!mbar_wait_bounded(smem_addr(drain), 0)) atomicExch(p.err, kErrMma);
        }
    } else {
        // --------------------------------------- fp32 sums of the chains --
        const int quad = warp & 3;  // the TMEM lanes this warp may read
        const int col0 = (warp - kLoadWarps - 1) / 4 * S::kAccCols;
        float sum[S::kAccCols];
#pragma unroll
        for (int j = 0; j < S::kAccCols; ++j) sum[j] = 0.0f;
        const int chains = (kb1 - kb0 + kChain - 1) / kChain;
        bool ok = true;
        for (int chain = 0; chain < chains; ++chain) {
            const int acc = chain & 1;
            int granted = 1;
            if (lane == 0) granted = mbar_wait(smem_addr(&acc_full[acc]), (chain >> 1) & 1, abort_flag) ? 1 : 0;
            ok = __shfl_sync(0xffffffffu, granted, 0) != 0;
            if (!ok) break;
            tc_fence_after();
#pragma unroll
            for (int c = 0; c < S::kAccCols; c += 32) {
                uint32_t r[32];
                tmem_ld32(tmem + (uint32_t(quad * 32) << 16) + acc * NT + col0 + c, r);
                tmem_wait_ld();
#pragma unroll
                for (int j = 0; j < 32; ++j) sum[c + j] += __uint_as_float(r[j]);
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_addr(&acc_empty[acc]));
        }
        if (!ok && lane == 0) atomicExch(p.err, kErrEpilogue);
        if (ok) {
            // The last chain is complete, so the stages are free.
            float* partial = reinterpret_cast<float*>(smem);
#pragma unroll
            for (int j = 0; j < S::kAccCols; ++j) partial[(col0 + j) * 128 + quad * 32 + lane] = sum[j];
        }
    }
    __syncwarp();
    tc_fence_before();
    sum_and_finish<float, PARTS, NT>(
        p, reinterpret_cast<const float*>(smem), m0, n0, S::kThreads / 32, [&](int64_t m, int64_t n, int q, float& z) {
            if (z == z || n >= p.N) return;
            const float* w = o.w + (n + int64_t(q) * p.N) * o.sw_n;
            const float* x = o.x + m * o.sx_m;
            z = 0.0f;
            for (int64_t k = 0; k < p.K; ++k) z = fmaf(w[k * o.sw_k], x[k * o.sx_k], z);
        });
    if (warp == kLoadWarps) {
        __syncwarp();
        tc_fence_after();
        tmem_dealloc(tmem, S::kTmemCols);
    }
}

template <int PARTS, int NT, bool W_MN, bool X_MN>
void launch_f32(FewParams& p, const F32Operands& o, int dev, cudaStream_t stream) {
    using S = F32Shape<NT>;
    auto kern = gemm_f32_kernel<PARTS, NT, W_MN, X_MN>;
    static bool configured[64] = {};
    if (!configured[dev]) {
        TPB_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(S::kSmem)));
        configured[dev] = true;
    }
    p.idesc = (1u << 4) | (2u << 7) | (2u << 10) | (uint32_t(NT >> 3) << 17) | (uint32_t(128 >> 4) << 24);
    p.row_tiles = (p.M + NT - 1) / NT;
    const int64_t tiles = int64_t(p.row_tiles) * ((p.N + 128 / PARTS - 1) / (128 / PARTS));
    p.split = choose_split(tiles, p.k_blocks, num_sms(dev), 16);
    launch_cluster(kern, tiles * p.split, p.split, S::kThreads, S::kSmem, stream, p, o);
    check_launch("gemm_f32");
}

template <int PARTS, bool W_MN, bool X_MN>
void launch_rows(FewParams& p, const F32Operands& o, int dev, cudaStream_t stream) {
    // 128 rows a tile where that still gives every SM one, fewer otherwise.
    const int64_t columns = (p.N + 128 / PARTS - 1) / (128 / PARTS);
    if (p.M <= 32) launch_f32<PARTS, 32, W_MN, X_MN>(p, o, dev, stream);
    else if (p.M <= 64 || columns * ((p.M + 127) / 128) < num_sms(dev)) launch_f32<PARTS, 64, W_MN, X_MN>(p, o, dev, stream);
    else launch_f32<PARTS, 128, W_MN, X_MN>(p, o, dev, stream);
}

bool vectors(const float* p, int64_t s_row) { return aligned16(p) && s_row % 4 == 0; }

}  // namespace

void gemm_f32(const FfnProblem& q, int dev, cudaStream_t stream) {
    FewParams p = few_params(q, dev, 32);
    F32Operands o{};
    o.w = static_cast<const float*>(q.w);
    o.sw_n = q.sw_n;
    o.sw_k = q.sw_k;
    o.x = static_cast<const float*>(q.x);
    o.sx_m = q.sx_m;
    o.sx_k = q.sx_k;
    o.vec_w = vectors(o.w, o.sw_n);
    o.vec_x = vectors(o.x, o.sx_m);
    o.tf32 = (q.flags & TPB_GEMM_ALLOW_TF32) != 0;
    // A layer reads w and x along k; dz w reads w along its rows' elements,
    // dz^T x both operands (w's strides are then both 1 when it has one column).
    const bool x_mn = q.sx_k != 1, w_mn = q.sw_k != 1 || x_mn;
    if (q.parts == 2) launch_rows<2, false, false>(p, o, dev, stream);
    else if (!w_mn) launch_rows<1, false, false>(p, o, dev, stream);
    else if (!x_mn) launch_rows<1, true, false>(p, o, dev, stream);
    else launch_rows<1, true, true>(p, o, dev, stream);
}

}  // namespace tpb
