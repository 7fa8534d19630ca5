// Feed-forward products for few rows (one token to a few hundred): the same
// results as gemm_ffn.cu where its 256 x 256 tiles would leave most SMs idle
// or compute mostly padding.
//
// With M rows the product reads the weight once (2 N K bytes in 16 bits) and
// does 2 M N K operations, so up to M of about 250 its bound is HBM: every SM
// has to stream weights all the time.  Hence
//   * the weight is the MMA's 128-row operand and the rows of x its N
//     dimension (kNT = 16 .. 128), so no tensor work goes into padding rows
//     beyond the next 16;
//   * a gated tile is 64 gate rows and 64 up rows of the weight, or 128 and
//     128 for up to 32 rows of x; two CTAs fit an SM, and one's set-up and
//     final sum overlap the other's stream;
//   * K is split over a cluster of C CTAs, because N / 128 tiles alone do not
//     fill 148 SMs; each CTA streams its share of K through a TMA ring into
//     TMEM accumulators;
//   * the partial accumulators go to shared memory and each CTA of the cluster
//     sums its share of the outputs over distributed shared memory, in rank
//     order (the same bits on every run, no workspace, no atomics), then
//     applies bias, activation, gate and residual in fp32.
// The weight is read K-major (x W^T) or, for the input gradient dz W, in
// place as an MN-major operand.  The weight gradient dz^T x of many rows and
// few features has the same shape of problem (a long sum, few tiles); there
// both operands are MN-major.
//
// Every wait is bounded as in gemm_tc.cu; all threads reach the cluster
// barriers.  No TMA multicast is used.

#include <cmath>

#include "gemm_few.cuh"

namespace tpb {
namespace {

constexpr int kFewThreads = 192;  // warp 0 TMA producer, 1 MMA issuer, 2-5 accumulator readers
constexpr int kFewWarps = kFewThreads / 32;

// WT: 128-row accumulators of a tile.
template <int NT, int WT>
struct FewShape {
    static constexpr uint32_t kWBytes = WT * 128 * 128;
    static constexpr uint32_t kXBytes = NT * 128;
    static constexpr uint32_t kStageBytes = kWBytes + kXBytes;
    // Two CTAs an SM, 110 KB of stages each.
    static constexpr int kStages = int(110 * 1024 / kStageBytes);
    static constexpr uint32_t kPartialBytes = WT * NT * 128 * 4;  // reuses the stages
    static_assert(kPartialBytes <= kStages * kStageBytes, "partial sums fit the stages");
    static constexpr size_t kSmem = size_t(kStages) * kStageBytes + 1024 + 256;
    static constexpr int kTmemCols = WT * NT < 32 ? 32 : WT * NT;  // a power of two
};

template <typename T, int PARTS, int NT, int WT, bool W_MN, bool X_MN>
__global__ void __launch_bounds__(kFewThreads)
    gemm_few_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX, const FewParams p) {
    using S = FewShape<NT, WT>;
    constexpr int kStages = S::kStages;
    constexpr int kColumns = WT * 128 / PARTS;  // result columns of a tile
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + kStages * S::kStageBytes);
    uint64_t* empty = full + kStages;
    uint64_t* done = empty + kStages;
    volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(done + 1);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    pdl_trigger();
    const int ranks = int(cluster_size());
    const int rank = int(cluster_ctarank());
    const int tile = blockIdx.x / ranks;
    // Row tiles of one weight tile are neighbours, so its later readers hit L2.
    const int wt = tile / p.row_tiles, mt = tile - wt * p.row_tiles;
    const int n0 = wt * kColumns, m0 = mt * NT;
    const int kb0 = int(int64_t(p.k_blocks) * rank / ranks), kb1 = int(int64_t(p.k_blocks) * (rank + 1) / ranks);

    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(smem_addr(&full[s]), 1);
            mbar_init(smem_addr(&empty[s]), 1);
        }
        mbar_init(smem_addr(done), 1);
        *abort_flag = 0;
        mbar_fence_init();
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&tmW)) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&tmX)) : "memory");
    }
    if (warp == 1) {
        tmem_alloc(smem_addr(const_cast<uint32_t*>(tmem_slot)), S::kTmemCols);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    if (threadIdx.x == 0) {
        // The weight's first block starts for L2 while the previous kernel ends:
        // nothing is read from it yet, so it does not matter if that kernel
        // still writes it (one token, 4096 -> 2 * 11008: 31.2 -> 30.6 us; more
        // blocks ahead slow down the products that K's split makes short).
#pragma unroll
        for (int q = 0; q < PARTS; ++q) {
#pragma unroll
            for (int j = 0; j < kColumns / 64; ++j) {
                if constexpr (W_MN) tma_prefetch_2d(&tmW, n0 + q * p.N + j * 64, kb0 * 64);
                else tma_prefetch_2d(&tmW, kb0 * 64, n0 + q * p.N + j * 64);
            }
        }
    }
    pdl_wait();

    if (warp == 0) {
        if (lane == 0) {
            int stage = 0;
            uint32_t phase = 0;
            bool ok = true;
            for (int kb = kb0; kb < kb1; ++kb) {
                if (!mbar_wait(smem_addr(&empty[stage]), phase ^ 1, abort_flag)) {
                    ok = false;
                    break;
                }
                const uint32_t fb = smem_addr(&full[stage]);
                const uint32_t at = smem_addr(smem + stage * S::kStageBytes);
                mbar_expect_tx(fb, S::kStageBytes);
#pragma unroll
                for (int q = 0; q < PARTS; ++q) {
                    load_operand<2, W_MN, false, false>(at + q * (S::kWBytes / PARTS), &tmW, fb, n0 + q * p.N, kb * 64,
                                                        0, kColumns);
                }
                if constexpr (X_MN) load_operand<2, true, false, false>(at + S::kWBytes, &tmX, fb, m0, kb * 64, 0, NT);
                else tma_load_2d(at + S::kWBytes, &tmX, fb, kb * 64, m0);
                if (++stage == kStages) {
                    stage = 0;
                    phase ^= 1;
                }
            }
            if (!ok) {
                atomicExch(p.err, kErrProducer);
                // Loads already issued land before the CTA leaves.
                for (int s = 0; s < kStages; ++s) {
                    mbar_wait_bounded(smem_addr(&full[s]), (s < stage) ? phase : phase ^ 1);
                }
            }
        }
    } else if (warp == 1) {
        if (lane == 0) {
            constexpr uint32_t a_lbo = W_MN ? 8192 : 16;
            constexpr uint32_t a_kstep = W_MN ? 16 * 128 : 32;
            int stage = 0;
            uint32_t phase = 0;
            bool ok = true;
            for (int kb = kb0; kb < kb1; ++kb) {
                if (!mbar_wait(smem_addr(&full[stage]), phase, abort_flag)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                const uint32_t at = smem_addr(smem + stage * S::kStageBytes);
#pragma unroll
                for (int kk = 0; kk < 4; ++kk) {
                    const uint64_t bd = sw128_desc(at + S::kWBytes + kk * (X_MN ? 16 * 128 : 32), X_MN ? 8192 : 16, 1024);
#pragma unroll
                    for (int t = 0; t < WT; ++t) {
                        const uint64_t ad = sw128_desc(at + t * 16384 + kk * a_kstep, a_lbo, 1024);
                        umma<false>(tmem + t * NT, ad, bd, p.idesc, (kb > kb0 || kk > 0) ? 1u : 0u);
                    }
                }
                umma_commit(smem_addr(&empty[stage]));
                if (++stage == kStages) {
                    stage = 0;
                    phase ^= 1;
                }
            }
            if (!ok) atomicExch(p.err, kErrMma);
            // The accumulators are complete (or, after a failure, every MMA
            // issued is, so that TMEM can be released).
            umma_commit(smem_addr(done));
            if (!mbar_wait_bounded(smem_addr(done), 0)) atomicExch(p.err, kErrMma);
        }
    } else {
        const int quad = warp & 3;  // the TMEM lanes this warp may read
        if (!mbar_wait_bounded(smem_addr(done), 0)) {
            if (lane == 0) atomicExch(p.err, kErrEpilogue);
        } else {
            tc_fence_after();
            float* partial = reinterpret_cast<float*>(smem);
#pragma unroll
            for (int c = 0; c < WT * NT; c += 16) {
                if (c % NT >= p.M - m0) continue;  // rows of x past M
                uint32_t r[16];
                tmem_ld16(tmem + (uint32_t(quad * 32) << 16) + c, r);
                tmem_wait_ld();
#pragma unroll
                for (int j = 0; j < 16; ++j) partial[(c + j) * 128 + quad * 32 + lane] = __uint_as_float(r[j]);
            }
        }
    }
    __syncwarp();
    tc_fence_before();
    cluster_sync();  // every CTA's partial sums are in its shared memory
    finish_rows<T, PARTS, NT, (WT > 1)>(p, reinterpret_cast<const float*>(smem), m0, n0, warp, kFewWarps, rank, ranks,
                              [](int64_t, int64_t, int, float&) {});
    cluster_sync();  // no CTA leaves while another reads its shared memory
    if (warp == 1) {
        __syncwarp();
        tc_fence_after();
        tmem_dealloc(tmem, S::kTmemCols);
    }
}

// Microseconds of a product of few rows, which streams its weight: n CTAs of
// `mb` megabytes each, at most `slots` at a time.  What n CTAs draw together
// saturates: 3.5 TB/s was measured for 64 of them, 5.7 for 172, 6.2 for 256,
// close to 6.5 (1 - exp(-n / 92)); a wave's ramp takes 2.5 us, the cluster's
// sum 0.1 us a rank.  (4096 -> 2 * 11008, one token: 64 + 64 columns 35.5 /
// measured 34 - 38 us, 128 + 128 with K split by three 32.5 / 30.7 us; 2 *
// 16384: 46.5 / 45.0, 46.6 / 47.0.)
double stream_us(int64_t n, int64_t slots, double mb, int split) {
    const auto wave = [&](int64_t ctas) { return ctas * mb / (6.5 * (1.0 - std::exp(-double(ctas) / 92.0))) + 2.5; };
    const int64_t full = n / slots, rest = n - full * slots;
    return (full > 0 ? full * wave(slots) : 0.0) + (rest > 0 ? wave(rest) : 0.0) + 0.1 * split;
}

// Launches the product, or with `us` only estimates its time.
template <typename T, int PARTS, int NT, int WT, bool W_MN, bool X_MN>
void launch_few(const FfnProblem& q, CUtensorMapDataType type, int dev, cudaStream_t stream, double* us) {
    using S = FewShape<NT, WT>;
    auto kern = gemm_few_kernel<T, PARTS, NT, WT, W_MN, X_MN>;
    const Slots& slots = cluster_slots<gemm_few_kernel<T, PARTS, NT, WT, W_MN, X_MN>>(kFewThreads, S::kSmem, dev);
    const int row_tiles = static_cast<int>((q.M + NT - 1) / NT), k_blocks = static_cast<int>((q.K + 63) / 64);
    const int64_t tiles = int64_t(row_tiles) * ((q.N + WT * 128 / PARTS - 1) / (WT * 128 / PARTS));
    int64_t waves = 1;
    int split = 1;
    double stream_best = 1e30;
    if constexpr (NT <= 64) {
        // A block's weight rows, and its rows of x from L2 at a fraction of
        // their cost.
        const double block_mb = (S::kWBytes + 0.4 * S::kXBytes) * 1e-6;
        for (int c = 1; c <= 8 && c <= k_blocks; ++c) {
            const double t = stream_us(tiles * c, slots.ctas[c], block_mb * ((k_blocks + c - 1) / c), c);
            if (t < stream_best) {
                stream_best = t;
                split = c;
            }
        }
        if (us != nullptr) {
            *us = stream_best;
            return;
        }
    } else {
        split = choose_split(tiles, k_blocks, slots, 8, &waves);
    }
    if (us != nullptr) {
        *us = 6.0 + waves * ((k_blocks + split - 1) / split * (tiles * split > num_sms(dev) ? 0.5 : 0.27) + 2.0);
        return;
    }
    FewParams p = few_params(q, dev, 64);
    const uint32_t fmt = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
    p.idesc = (1u << 4) | (fmt << 7) | (fmt << 10) | (uint32_t(W_MN) << 15) | (uint32_t(X_MN) << 16) |
              (uint32_t(NT >> 3) << 17) |
              (uint32_t(128 >> 4) << 24);
    p.row_tiles = row_tiles;
    static_assert(!X_MN || NT >= 64, "an MN-major operand is staged 64 rows at a time");
    const CUtensorMap mx = X_MN ? make_map(q.x, type, 2, q.M, q.K, q.sx_k, 1, 0, 64)
                                : make_map(q.x, type, 2, q.K, q.M, q.sx_m, 1, 0, NT);
    const CUtensorMap mw = W_MN ? make_map(q.w, type, 2, q.N, q.K, q.sw_k, 1, 0, 64)
                                : make_map(q.w, type, 2, q.K, PARTS * q.N, q.sw_n, 1, 0, kBoxRows);
    launch_cluster(kern, tiles * split, split, kFewThreads, S::kSmem, stream, mw, mx, p);
    check_launch("gemm_few");
}

// Gated tiles of 64 + 64 or 128 + 128 columns, whichever fills the device
// better.
template <typename T, int PARTS, int NT, bool W_MN>
void launch_narrow(const FfnProblem& q, CUtensorMapDataType type, int dev, cudaStream_t stream, double* us) {
    if constexpr (PARTS == 2) {
        double one = 0.0, two = 0.0;
        launch_few<T, PARTS, NT, 1, W_MN, false>(q, type, dev, stream, &one);
        launch_few<T, PARTS, NT, 2, W_MN, false>(q, type, dev, stream, &two);
        if (us != nullptr) *us = std::min(one, two);
        else if (two < one) launch_few<T, PARTS, NT, 2, W_MN, false>(q, type, dev, stream, nullptr);
        else launch_few<T, PARTS, NT, 1, W_MN, false>(q, type, dev, stream, nullptr);
    } else {
        launch_few<T, PARTS, NT, 1, W_MN, false>(q, type, dev, stream, us);
    }
}

template <typename T, int PARTS, bool W_MN>
void launch_rows(const FfnProblem& q, CUtensorMapDataType type, int dev, cudaStream_t stream, double* us) {
    if (q.M <= 16) launch_narrow<T, PARTS, 16, W_MN>(q, type, dev, stream, us);
    else if (q.M <= 32) launch_narrow<T, PARTS, 32, W_MN>(q, type, dev, stream, us);
    else if (q.M <= 64) launch_few<T, PARTS, 64, 1, W_MN, false>(q, type, dev, stream, us);
    else launch_few<T, PARTS, 128, 1, W_MN, false>(q, type, dev, stream, us);
}

template <typename T>
void launch_typed(const FfnProblem& q, CUtensorMapDataType type, int dev, cudaStream_t stream, double* us) {
    if (q.sx_k != 1) {
        if (q.M <= 64) launch_few<T, 1, 64, 1, true, true>(q, type, dev, stream, us);
        else launch_few<T, 1, 128, 1, true, true>(q, type, dev, stream, us);
    } else if (q.sw_k != 1) launch_rows<T, 1, true>(q, type, dev, stream, us);
    else if (q.parts == 2) launch_rows<T, 2, false>(q, type, dev, stream, us);
    else launch_rows<T, 1, false>(q, type, dev, stream, us);
}

void dispatch(const FfnProblem& q, int dev, cudaStream_t stream, double* us) {
    if (q.dtype == TPB_BF16) launch_typed<__nv_bfloat16>(q, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, dev, stream, us);
    else launch_typed<__half>(q, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, dev, stream, us);
}

}  // namespace

void gemm_few(const FfnProblem& q, int dev, cudaStream_t stream) { dispatch(q, dev, stream, nullptr); }

double gemm_few_us(const FfnProblem& q, int dev) {
    double us = 0.0;
    dispatch(q, dev, nullptr, &us);
    return us;
}

}  // namespace tpb
