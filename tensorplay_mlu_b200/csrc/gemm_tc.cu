// Tensor-core matrix product for sm_100a: tcgen05.mma with TMEM accumulators,
// operands staged by TMA into 128-byte-swizzled shared memory, and a
// persistent, warp-specialised CTA per SM (tensorplay-mlu runs these
// products on cnnlMatMul_v2 / cnnlStrideBatchMatMul_v3, BlasKernels.cpp:202-242).
//
// CTA layout (320 threads, one CTA per SM):
//   warp 0      TMA producer: one elected thread fills a ring of kStages
//               shared-memory stages (A: 128 x 64 bf16, B: BN x 64 bf16) and
//               arms each stage's "full" mbarrier with the byte count;
//   warp 1      MMA issuer: allocates TMEM (2 accumulators of 128 x BN fp32),
//               one elected thread issues 4 x tcgen05.mma (K = 16 each) per
//               stage and releases the stage with tcgen05.commit on its
//               "empty" mbarrier; after a tile's last stage it commits to the
//               accumulator's "full" barrier;
//   warps 2..9  epilogue: two warps per TMEM lane quadrant (the lanes a
//               warp may access), each taking half of the columns:
//               tcgen05.ld 32 columns at a time (the next chunk's load
//               issued before the current one is stored), apply
//               alpha/beta/addend, convert and store; then release the
//               accumulator.
// Two accumulators let the epilogue of tile i overlap the mainloop of
// tile i+1.  Tiles are visited in groups of kGroupM row-tiles so the CTAs in
// flight share A and B panels in L2.
//
// Transposed operands are read in place: an operand whose unit stride is on
// the M (or N) side is loaded as 64-element MN-major chunks and described to
// the MMA as MN-major (the instruction descriptor's transpose bits), the way
// as_operand (BlasKernels.cpp:40-54) passes a transpose flag.
//
// Every wait is bounded (kWaitNs): a role that gives up records an error
// code in the library's device error word, tells the other roles through
// shared memory, drains what it has in flight and leaves; the host reports
// it through tp_b200_take_device_error.  No TMA multicast is used.

#include "gemm_tc.cuh"

namespace tpb {

void copy_impl(const tpb_tensor& dst, const tpb_tensor& src, cudaStream_t stream, int dev);

namespace {

template <typename T, int BN, bool A_MN, bool B_MN, bool BATCHED>
__global__ void __launch_bounds__(kTcThreads, 1)
    gemm_tc_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                   const __grid_constant__ CUtensorMap tmC,
                   const TcParams p) {
    using E = TcElem<T>;
    constexpr int kStages = TcShape<BN>::kStages;
    constexpr int kTmemCols = TcShape<BN>::kTmemCols;
    constexpr int kEPR = 128 / E::kES;             // elements per 128-byte row (K per stage)
    constexpr int kUmmaK = 32 / E::kES;            // K per instruction
    constexpr int kKSteps = kEPR / kUmmaK;         // instructions per stage (4)
    constexpr uint32_t kABytes = kBM * 128;        // A stage bytes
    constexpr uint32_t kBBytes = BN * 128;         // B stage bytes
    constexpr uint32_t kChunk = kEPR * 128;        // one MN-major chunk: kEPR rows of K x 128 B

    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* smem_a = smem;
    uint8_t* smem_b = smem + kStages * kABytes;
    uint8_t* staging = smem_b + kStages * kBBytes;  // kEpilogueWarps tiles for TMA stores
    uint64_t* bars = reinterpret_cast<uint64_t*>(staging + kEpilogueWarps * staging_bytes<T>());
    uint64_t* full = bars;
    uint64_t* empty = bars + kStages;
    uint64_t* acc_full = bars + 2 * kStages;
    uint64_t* acc_empty = acc_full + 2;
    uint64_t* drain = acc_empty + 2;
    volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(drain + 1);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    pdl_trigger();

    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(smem_addr(&full[s]), 1);
            mbar_init(smem_addr(&empty[s]), 1);
        }
        for (int a = 0; a < 2; ++a) {
            mbar_init(smem_addr(&acc_full[a]), 1);
            mbar_init(smem_addr(&acc_empty[a]), kEpilogueWarps);
        }
        mbar_init(smem_addr(drain), 1);
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&tmA)) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&tmB)) : "memory");
    }
    if (warp == 1) {
        tmem_alloc(smem_addr(const_cast<uint32_t*>(tmem_slot)), kTmemCols);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    pdl_wait();  // set-up above overlaps the previous kernel; memory access starts here

    if (warp == 0) {
        // ---------------------------------------------------- producer --
        if (lane == 0) {
            int stage = 0;
            uint32_t phase = 0;
            bool ok = true;
            for (int tile = blockIdx.x; tile < p.num_tiles && ok; tile += gridDim.x) {
                int b, mt, nt;
                tile_coords(p, tile, b, mt, nt);
                const int m0 = mt * kBM, n0 = nt * BN;
                for (int kb = 0; kb < p.k_blocks; ++kb) {
                    if (!mbar_wait(smem_addr(&empty[stage]), phase ^ 1, abort_flag)) {
                        ok = false;
                        break;
                    }
                    const uint32_t fb = smem_addr(&full[stage]);
                    mbar_expect_tx(fb, kABytes + kBBytes);
                    const uint32_t da = smem_addr(smem_a + stage * kABytes);
                    const uint32_t db = smem_addr(smem_b + stage * kBBytes);
                    const int k0 = kb * kEPR;
                    load_operand<E::kES, A_MN, BATCHED, false>(da, &tmA, fb, m0, k0, b, kBM);
                    load_operand<E::kES, B_MN, BATCHED, false>(db, &tmB, fb, n0, k0, b, BN);
                    if (++stage == kStages) {
                        stage = 0;
                        phase ^= 1;
                    }
                }
            }
            if (!ok) {
                atomicExch(p.err, kErrProducer);
                // Let the loads already issued land before the CTA leaves:
                // every stage's most recent phase completes once its bytes do.
                for (int s = 0; s < kStages; ++s) {
                    const uint64_t start = global_ns();
                    while (!mbar_try_wait(smem_addr(&full[s]), (s < stage) ? phase : phase ^ 1)) {
                        if (global_ns() - start > kWaitNs) break;
                    }
                }
            }
        }
    } else if (warp == 1) {
        // ------------------------------------------------- MMA issuer --
        if (lane == 0) {
            int stage = 0;
            uint32_t phase = 0;
            int local = 0;
            bool ok = true;
            constexpr uint32_t a_lbo = A_MN ? kChunk : 16;
            constexpr uint32_t b_lbo = B_MN ? kChunk : 16;
            constexpr uint32_t a_kstep = A_MN ? kUmmaK * 128 : 32;
            constexpr uint32_t b_kstep = B_MN ? kUmmaK * 128 : 32;
            for (int tile = blockIdx.x; tile < p.num_tiles && ok; tile += gridDim.x, ++local) {
                const int acc = local & 1;
                const uint32_t acc_phase = (local >> 1) & 1;
                if (!mbar_wait(smem_addr(&acc_empty[acc]), acc_phase ^ 1, abort_flag)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                const uint32_t d_tmem = tmem_base + acc * BN;
                for (int kb = 0; kb < p.k_blocks; ++kb) {
                    if (!mbar_wait(smem_addr(&full[stage]), phase, abort_flag)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint32_t sa = smem_addr(smem_a + stage * kABytes);
                    const uint32_t sb = smem_addr(smem_b + stage * kBBytes);
#pragma unroll
                    for (int kk = 0; kk < kKSteps; ++kk) {
                        const uint64_t ad = sw128_desc(sa + kk * a_kstep, a_lbo, 1024);
                        const uint64_t bd = sw128_desc(sb + kk * b_kstep, b_lbo, 1024);
                        umma<E::kTF32>(d_tmem, ad, bd, p.idesc, (kb | kk) != 0 ? 1u : 0u);
                    }
                    umma_commit(smem_addr(&empty[stage]));
                    if (++stage == kStages) {
                        stage = 0;
                        phase ^= 1;
                    }
                }
                if (!ok) break;
                umma_commit(smem_addr(&acc_full[acc]));
            }
            if (!ok) atomicExch(p.err, kErrMma);
            // Drain: every MMA issued by this thread completes before TMEM
            // is released.
            umma_commit(smem_addr(drain));
            const uint64_t start = global_ns();
            while (!mbar_try_wait(smem_addr(drain), 0)) {
                if (global_ns() - start > kWaitNs) break;
            }
        }
    } else {
        // --------------------------------------------------- epilogue --
        // Warps 2-9: lane quadrant warp & 3 (the TMEM lanes a warp may read),
        // column half (warp - 2) / 4.
        const int quad = warp & 3;
        const int half = (warp - 2) / 4;
        const int row_in_tile = quad * 32 + lane;
        int local = 0;
        for (int tile = blockIdx.x; tile < p.num_tiles; tile += gridDim.x, ++local) {
            const int acc = local & 1;
            const uint32_t acc_phase = (local >> 1) & 1;
            if (!mbar_wait(smem_addr(&acc_full[acc]), acc_phase, abort_flag)) {
                if (lane == 0) atomicExch(p.err, kErrEpilogue);
                break;
            }
            tc_fence_after();
            int b, mt, nt;
            tile_coords(p, tile, b, mt, nt);
            const int64_t gm = int64_t(mt) * kBM + row_in_tile;
            const uint32_t t_rows = tmem_base + (uint32_t(quad * 32) << 16) + acc * BN;
            if (p.tma_store) {
                store_accumulator_tma<T, BN / 2, BATCHED>(p, &tmC, staging + (warp - 2) * staging_bytes<T>(), t_rows,
                                                          half * (BN / 2), b, gm, gm - lane, int64_t(nt) * BN,
                                                          gm < p.M);
            } else {
                store_accumulator_plain<T, BN / 2>(p, staging + (warp - 2) * staging_bytes<T>(), t_rows, half * (BN / 2),
                                                   b, gm, int64_t(nt) * BN, gm < p.M);
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_relaxed(smem_addr(&acc_empty[acc]));
        }
        // The TMA stores this warp issued are complete before the CTA leaves.
        if (lane == 0) bulk_wait_group0();
    }

    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        __syncwarp();
        tc_fence_after();
        tmem_dealloc(tmem_base, kTmemCols);
    }
}

// ------------------------------------------------------------ host side --

// Counter words of the run-time tile scheduler: one per (device, stream)
// slot; a launch's epoch (per slot, counted on the host) tells its claims
// from those of the launches before it.
constexpr int kSchedSlots = 64;
__device__ unsigned long long g_gemm_sched[kSchedSlots];

// Whether the CTA-pair products on a device claim tiles at run time
// (tp_b200_set_gemm_tile_order; TPB200_GEMM_SCHED=dynamic turns it on for
// every device).  The fixed order is the default: it keeps each wave's
// tiles on neighbouring panels, and claiming costs a round trip per tile.
std::atomic<bool> g_gemm_dynamic[64] = {};

}  // namespace

// The counter word and a fresh epoch for a launch on `stream`, or a null
// word (fixed tile order) unless run-time claims are on for the device;
// also while the stream is being captured into a graph (every replay would
// reuse the recorded epoch), for the per-thread default stream (one handle,
// many streams) and when the slots are used up.
SchedSlot gemm_sched_slot(int dev, cudaStream_t stream) {
    static const bool env_dynamic = [] {
        const char* e = std::getenv("TPB200_GEMM_SCHED");
        return e != nullptr && std::strcmp(e, "dynamic") == 0;
    }();
    const bool dynamic = dev >= 0 && dev < 64 && (env_dynamic || g_gemm_dynamic[dev].load(std::memory_order_relaxed));
    if (!dynamic || stream == cudaStreamPerThread) return {nullptr, 0};
    cudaStreamCaptureStatus cap = cudaStreamCaptureStatusNone;
    TPB_CUDA(cudaStreamIsCapturing(stream, &cap));
    if (cap != cudaStreamCaptureStatusNone) return {nullptr, 0};
    static std::mutex lock;
    static unsigned long long* base[64] = {};
    static std::map<std::pair<int, cudaStream_t>, std::pair<int, uint32_t>> slots;
    static int used[64] = {};
    std::lock_guard<std::mutex> g(lock);
    if (base[dev] == nullptr) {
        void* ptr = nullptr;
        TPB_CUDA(cudaGetSymbolAddress(&ptr, g_gemm_sched));
        base[dev] = static_cast<unsigned long long*>(ptr);
    }
    auto it = slots.find({dev, stream});
    if (it == slots.end()) {
        if (used[dev] >= kSchedSlots) return {nullptr, 0};
        it = slots.emplace(std::make_pair(dev, stream), std::make_pair(used[dev]++, 0u)).first;
    }
    uint32_t& epoch = it->second.second;
    if (++epoch == 0) epoch = 1;  // 0 is the words' initial value
    return {base[dev] + it->second.first, epoch};
}

namespace {

// Per-shape tile choice, computed once and cached (BlasKernels.cpp:70-104
// caches a CNNL plan per problem the same way).
int choose_bn(int64_t M, int64_t N, int64_t batch, int sms) {
    using Key = std::tuple<int64_t, int64_t, int64_t, int>;
    static std::mutex lock;
    static std::map<Key, int> cache;
    const Key key{M, N, batch, sms};
    {
        std::lock_guard<std::mutex> g(lock);
        auto it = cache.find(key);
        if (it != cache.end()) return it->second;
    }
    // Cost in units of one 128 x 128 tile; a 128 x 256 tile costs a little
    // under two (better operand reuse per MMA).
    auto cost = [&](int bn) {
        const int64_t tiles = batch * ((M + kBM - 1) / kBM) * ((N + bn - 1) / bn);
        const int64_t waves = (tiles + sms - 1) / sms;
        return static_cast<double>(waves) * (bn == 256 ? 1.9 : 1.0);
    };
    const int bn = N <= 128 ? 128 : (cost(256) <= cost(128) ? 256 : 128);
    std::lock_guard<std::mutex> g(lock);
    cache[key] = bn;
    return bn;
}

template <typename T, int BN, bool A_MN, bool B_MN, bool BATCHED>
void launch_tc(const GemmProblem& p, const CUtensorMap& ma, const CUtensorMap& mb, const CUtensorMap& mc,
               TcParams& tp, int dev, cudaStream_t stream) {
    constexpr size_t smem = tc_smem_bytes<T, BN>();
    auto kern = gemm_tc_kernel<T, BN, A_MN, B_MN, BATCHED>;
    static bool configured[64] = {};
    if (!configured[dev]) {
        TPB_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)));
        configured[dev] = true;
    }
    tp.m_tiles = static_cast<int>((p.M + kBM - 1) / kBM);
    tp.n_tiles = static_cast<int>((p.N + BN - 1) / BN);
    tp.num_tiles = static_cast<int>(p.batch) * tp.m_tiles * tp.n_tiles;
    // Instruction descriptor: fp32 accumulate (bit 4), A/B format (bits 7-9,
    // 10-12: f16 0, bf16 1, tf32 2), A/B MN-major (bits 15, 16), N >> 3
    // (bits 17-22), M >> 4 (bits 24-28).
    const uint32_t fmt = std::is_same<T, __nv_bfloat16>::value ? 1u : std::is_same<T, float>::value ? 2u : 0u;
    tp.idesc = (1u << 4) | (fmt << 7) | (fmt << 10) | (uint32_t(tp.a_mn) << 15) |
               (uint32_t(tp.b_mn) << 16) | (uint32_t(BN >> 3) << 17) | (uint32_t(kBM >> 4) << 24);
    const int grid = std::min(tp.num_tiles, gemm_sm_budget(dev));
    launch_pdl(kern, grid, kTcThreads, smem, stream, ma, mb, mc, tp);
    check_launch("gemm_tc");
}

// The kernel instance for the operands' layouts and batching.  fp32 (TF32)
// operands always arrive K-major, so only that instance is built for them.
template <typename T, bool A_MN, bool B_MN, bool BATCHED>
void launch_layout(bool pair, int bn, const GemmProblem& p, const CUtensorMap& ma, const CUtensorMap& mb,
                   const CUtensorMap& mc, TcParams& tp, int dev, cudaStream_t stream) {
    if (pair) launch_tc2<T, A_MN, B_MN, BATCHED>(ma, mb, mc, tp, dev, stream);
    else if (bn == 256) launch_tc<T, 256, A_MN, B_MN, BATCHED>(p, ma, mb, mc, tp, dev, stream);
    else launch_tc<T, 128, A_MN, B_MN, BATCHED>(p, ma, mb, mc, tp, dev, stream);
}

template <typename T>
void launch_any(bool pair, int bn, const GemmProblem& p, const CUtensorMap& ma, const CUtensorMap& mb,
                const CUtensorMap& mc, TcParams& tp, int dev, cudaStream_t stream) {
    const bool bt = tp.batched != 0;
    if constexpr (std::is_same<T, float>::value) {
        TPB_CHECK(!tp.a_mn && !tp.b_mn, "gemm: TF32 operands must be K-major");
        if (bt) launch_layout<T, false, false, true>(pair, bn, p, ma, mb, mc, tp, dev, stream);
        else launch_layout<T, false, false, false>(pair, bn, p, ma, mb, mc, tp, dev, stream);
    } else {
        const int code = (tp.a_mn ? 4 : 0) | (tp.b_mn ? 2 : 0) | (bt ? 1 : 0);
        switch (code) {
            case 0: launch_layout<T, false, false, false>(pair, bn, p, ma, mb, mc, tp, dev, stream); break;
            case 1: launch_layout<T, false, false, true>(pair, bn, p, ma, mb, mc, tp, dev, stream); break;
            case 2: launch_layout<T, false, true, false>(pair, bn, p, ma, mb, mc, tp, dev, stream); break;
            case 3: launch_layout<T, false, true, true>(pair, bn, p, ma, mb, mc, tp, dev, stream); break;
            case 4: launch_layout<T, true, false, false>(pair, bn, p, ma, mb, mc, tp, dev, stream); break;
            case 5: launch_layout<T, true, false, true>(pair, bn, p, ma, mb, mc, tp, dev, stream); break;
            case 6: launch_layout<T, true, true, false>(pair, bn, p, ma, mb, mc, tp, dev, stream); break;
            default: launch_layout<T, true, true, true>(pair, bn, p, ma, mb, mc, tp, dev, stream); break;
        }
    }
}

// Which kernel: the CTA-pair kernel for problems with at least one full
// 256 x 256 tile, the single-SM kernel otherwise; TPB200_GEMM_KERNEL=1sm|2sm
// overrides the choice (for A/B measurements).
bool use_pair_kernel(const GemmProblem& p) {
    static const char* force = std::getenv("TPB200_GEMM_KERNEL");
    if (force != nullptr && std::strcmp(force, "1sm") == 0) return false;
    if (force != nullptr && std::strcmp(force, "2sm") == 0) return true;
    return p.M >= kPairBM && p.N >= kPairBN;
}

// The fused-epilogue instances: bf16, unbatched, CTA-pair kernel.
template <typename T, int EPI>
void launch_epi(const CUtensorMap& ma, const CUtensorMap& mb, const CUtensorMap& mc, const CUtensorMap& maux,
                TcParams& tp, int dev, cudaStream_t stream) {
    const int code = (tp.a_mn ? 2 : 0) | (tp.b_mn ? 1 : 0);
    switch (code) {
        case 0: launch_tc2<T, false, false, false, EPI>(ma, mb, mc, tp, dev, stream, &maux); break;
        case 1: launch_tc2<T, false, true, false, EPI>(ma, mb, mc, tp, dev, stream, &maux); break;
        case 2: launch_tc2<T, true, false, false, EPI>(ma, mb, mc, tp, dev, stream, &maux); break;
        default: launch_tc2<T, true, true, false, EPI>(ma, mb, mc, tp, dev, stream, &maux); break;
    }
}

template <typename T>
bool gemm_tc_typed(const GemmProblem& p_in, int dev, cudaStream_t stream, CUtensorMapDataType type) {
    constexpr int es = sizeof(T);
    GemmProblem p = p_in;
    if (p.epi != kEpiPlain) {
        // Fused epilogues: bf16 products with a full CTA-pair tile, no batch,
        // the result (and gelu's pre-activation) written by TMA stores.
        if constexpr (!std::is_same<T, __nv_bfloat16>::value) {
            return false;
        } else {
            if (p.batch != 1 || !use_pair_kernel(p) || p.aux == nullptr) return false;
            if (p.epi == kEpiGeluBackward && p.cin != nullptr) return false;
            if (p.epi == kEpiGelu && !(aligned16(p.aux) && p.saux_m > 0 && (p.saux_m * es) % 16 == 0)) return false;
            if (std::getenv("TPB200_NO_TMA_STORE") != nullptr) return false;
            if (!(aligned16(p.c) && p.sc_m > 0 && (p.sc_m * es) % 16 == 0)) return false;
        }
    }
    // TF32 operands must be K-major here: the 128-byte-swizzled MN-major
    // layout this kernel stages is defined for 16-bit elements only (32-bit
    // MN-major operands need the 32-byte-atom swizzle variant).  An MN-major
    // fp32 operand is first copied K-major (one transposing pass).
    std::unique_ptr<Scratch> a_copy, b_copy;
    if constexpr (std::is_same<T, float>::value) {
        if (!(p.sa_k == 1 || p.K == 1)) {
            a_copy.reset(new Scratch(sizeof(float) * p.batch * p.M * p.K, dev, stream));
            Scratch& tmp = *a_copy;
            tpb_tensor src{}, dst{};
            src.data = const_cast<void*>(p.a);
            src.dtype = dst.dtype = TPB_F32;
            src.ndim = dst.ndim = 3;
            const int64_t sizes[3] = {p.batch, p.M, p.K};
            const int64_t sstr[3] = {p.sa_b, p.sa_m, p.sa_k};
            const int64_t dstr[3] = {p.M * p.K, p.K, 1};
            for (int i = 0; i < 3; ++i) {
                src.sizes[i] = dst.sizes[i] = sizes[i];
                src.strides[i] = sstr[i];
                dst.strides[i] = dstr[i];
            }
            dst.data = tmp.get();
            copy_impl(dst, src, stream, dev);
            p.a = tmp.get();
            p.sa_b = p.batch > 1 ? p.M * p.K : 0;
            p.sa_m = p.K;
            p.sa_k = 1;
        }
        if (!(p.sb_k == 1 || p.K == 1)) {
            b_copy.reset(new Scratch(sizeof(float) * p.batch * p.N * p.K, dev, stream));
            Scratch& tmp = *b_copy;
            tpb_tensor src{}, dst{};
            src.data = const_cast<void*>(p.b);
            src.dtype = dst.dtype = TPB_F32;
            src.ndim = dst.ndim = 3;
            const int64_t sizes[3] = {p.batch, p.N, p.K};
            const int64_t sstr[3] = {p.sb_b, p.sb_n, p.sb_k};
            const int64_t dstr[3] = {p.N * p.K, p.K, 1};
            for (int i = 0; i < 3; ++i) {
                src.sizes[i] = dst.sizes[i] = sizes[i];
                src.strides[i] = sstr[i];
                dst.strides[i] = dstr[i];
            }
            dst.data = tmp.get();
            copy_impl(dst, src, stream, dev);
            p.b = tmp.get();
            p.sb_b = p.batch > 1 ? p.N * p.K : 0;
            p.sb_n = p.K;
            p.sb_k = 1;
        }
    }
    // A: K-major (unit stride along K) or M-major; same for B along K / N.
    const bool a_k = p.sa_k == 1 || p.K == 1;
    const bool a_m = !a_k && (p.sa_m == 1 || p.M == 1);
    const bool b_k = p.sb_k == 1 || p.K == 1;
    const bool b_n = !b_k && (p.sb_n == 1 || p.N == 1);
    if (!(a_k || a_m) || !(b_k || b_n)) return false;
    if (!tma_ok(p.a, es, a_k ? p.sa_m : p.sa_k, p.batch, p.sa_b)) return false;
    if (!tma_ok(p.b, es, b_k ? p.sb_n : p.sb_k, p.batch, p.sb_b)) return false;
    if (p.M >= (int64_t(1) << 31) || p.N >= (int64_t(1) << 31) || p.K >= (int64_t(1) << 31)) return false;
    const int sms = gemm_sm_budget(dev);
    const bool pair = use_pair_kernel(p);
    const int bn = pair ? 128 : choose_bn(p.M, p.N, p.batch, sms);  // B rows staged per CTA
    constexpr int kEPR = 128 / es;
    // Boxes: K-major operands kEPR (K) x kBoxRows rows (a stage takes 128 /
    // kBoxRows, or bn / kBoxRows, of them); MN-major operands kEPR (MN) x kEPR
    // (K) chunks.
    const CUtensorMap ma = a_k ? make_map(p.a, type, es, p.K, p.M, p.sa_m, p.batch, p.sa_b, kBoxRows)
                               : make_map(p.a, type, es, p.M, p.K, p.sa_k, p.batch, p.sa_b, kEPR);
    const CUtensorMap mb = b_k ? make_map(p.b, type, es, p.K, p.N, p.sb_n, p.batch, p.sb_b, kBoxRows)
                               : make_map(p.b, type, es, p.N, p.K, p.sb_k, p.batch, p.sb_b, kEPR);
    TcParams tp{};
    tp.M = static_cast<int>(p.M);
    tp.N = static_cast<int>(p.N);
    tp.K = static_cast<int>(p.K);
    tp.batch = static_cast<int>(p.batch);
    tp.k_blocks = static_cast<int>((p.K + kEPR - 1) / kEPR);
    tp.a_mn = a_k ? 0 : 1;
    tp.b_mn = b_k ? 0 : 1;
    tp.batched = p.batch > 1 ? 1 : 0;
    tp.c = p.c;
    tp.sc_b = p.sc_b;
    tp.sc_m = p.sc_m;
    tp.cin = p.cin;
    tp.sci_b = p.sci_b;
    tp.sci_m = p.sci_m;
    tp.sci_n = p.sci_n;
    tp.alpha = static_cast<float>(p.alpha);
    tp.beta = static_cast<float>(p.beta);
    tp.vec_store = aligned16(p.c) && (p.sc_m * es) % 16 == 0 && (p.batch == 1 || (p.sc_b * es) % 16 == 0);
    tp.aux = p.aux;
    tp.saux_m = p.saux_m;
    tp.err = device_error_word(dev);
    // The result through a C tensor map (TMA stores) when its layout allows.
    // TPB200_NO_TMA_STORE=1 keeps the direct-store epilogue (A/B measurements).
    static const bool no_tma_store = std::getenv("TPB200_NO_TMA_STORE") != nullptr;
    const bool c_tma = !no_tma_store && aligned16(p.c) && p.sc_m > 0 && (p.sc_m * es) % 16 == 0 &&
                       (p.batch == 1 || (p.sc_b > 0 && (p.sc_b * es) % 16 == 0));
    tp.tma_store = c_tma ? 1 : 0;
    const CUtensorMap mc = c_tma ? make_c_map(p.c, type, es, p.N, p.M, p.sc_m, p.batch, p.sc_b) : ma;
    if (p.epi != kEpiPlain) {
        if constexpr (std::is_same<T, __nv_bfloat16>::value) {
            TPB_CHECK(pair && c_tma, "gemm: fused epilogue without the CTA-pair TMA-store kernel");
            if (p.epi == kEpiGelu) {
                const CUtensorMap maux = make_c_map(p.aux, type, es, p.N, p.M, p.saux_m, 1, 0);
                launch_epi<T, kEpiGelu>(ma, mb, mc, maux, tp, dev, stream);
            } else {
                launch_epi<T, kEpiGeluBackward>(ma, mb, mc, mc, tp, dev, stream);
            }
        }
        return true;
    }
    launch_any<T>(pair, bn, p, ma, mb, mc, tp, dev, stream);
    return true;
}

// ---------------------------------------------- fp32 through 3 x TF32 --
//
// Without TF32 permission an fp32 product keeps fp32 accuracy by the
// split-precision ("3xTF32") method: every operand element x is split into
// hi = tf32(x) and lo = tf32(x - hi), both exact TF32 values (low 13
// mantissa bits zero, so the tensor core's reading of an fp32 word as TF32
// changes nothing), and A.B ~= Alo.Bhi + Ahi.Blo + Ahi.Bhi.  The dropped
// Alo.Blo term and the rounding of lo are both ~2^-22 relative to |a b|.
// The three products run as TF32 tensor-core GEMMs over K-concatenated
// operands, K in chunks of kSplitChunk:
//   A' chunk j = [Alo_j | Ahi_j | Ahi_j],   B' chunk j = [Bhi_j ; Blo_j ; Bhi_j]
// (both K-major; the small correction terms come first, while the
// accumulator is still small).  The tensor core adds into its accumulator
// with truncation after alignment, an error that grows with the number of
// additions; so each chunk is one GEMM launch whose epilogue adds its
// result into the output in fp32 with round-to-nearest (beta = 1 after the
// first chunk), keeping every accumulator chain short.
// A non-finite element (inf, NaN) has lo = 0, and inf * 0 in a cross term
// would turn an fp32 inf into NaN; the split marks such rows of A / columns
// of B and a fix-up pass recomputes the outputs in them with plain fp32 dot
// products.
constexpr int64_t kSplitChunk = 1024;

// Round to the nearest TF32 value (ties away from zero); a rounding that
// would overflow truncates instead; inf and NaN are returned unchanged.
__device__ __forceinline__ float tf32_round(float x) {
    const uint32_t u = __float_as_uint(x);
    if ((u & 0x7f800000u) == 0x7f800000u) return x;
    uint32_t r = (u + 0x1000u) & 0xffffe000u;
    if ((r & 0x7f800000u) == 0x7f800000u) r = u & 0xffffe000u;
    return __uint_as_float(r);
}

// Rows of a K-major operand (row `row` of batch `row / R` at
// src + (row / R) * s_b + (row % R) * s_r) into rows of `ld` floats, chunk j
// of K at j * 3 * kSplitChunk holding its three parts back to back (each
// K_j = min(kSplitChunk, K - j * kSplitChunk) wide): [lo | hi | hi] for A
// (b_side 0), [hi | lo | hi] for B (b_side 1).  flags[row] is set when the
// row holds a non-finite element.
__global__ void __launch_bounds__(256) split_tf32_kernel(const float* __restrict__ src, float* __restrict__ dst,
                                                         int64_t rows, int64_t R, int64_t K, int64_t s_b,
                                                         int64_t s_r, int64_t ld, int b_side,
                                                         unsigned* __restrict__ flags) {
    for (int64_t row = blockIdx.y; row < rows; row += gridDim.y) {
        const float* s = src + (row / R) * s_b + (row % R) * s_r;
        float* d = dst + row * ld;
        int bad = 0;
        for (int64_t k = int64_t(blockIdx.x) * blockDim.x + threadIdx.x; k < K;
             k += int64_t(gridDim.x) * blockDim.x) {
            const float x = s[k];
            const float hi = tf32_round(x);
            const bool finite = isfinite(x);
            const float lo = finite ? tf32_round(x - hi) : 0.0f;
            bad |= !finite;
            const int64_t j = k / kSplitChunk, kk = k % kSplitChunk;
            const int64_t kj = K - j * kSplitChunk < kSplitChunk ? K - j * kSplitChunk : kSplitChunk;
            float* c = d + j * 3 * kSplitChunk + kk;
            c[0] = b_side ? hi : lo;
            c[kj] = b_side ? lo : hi;
            c[2 * kj] = hi;
        }
        if (__syncthreads_or(bad) && threadIdx.x == 0) flags[row] = 1u;
    }
}

struct FixupParams {
    const float* a;
    int64_t sa_b, sa_m, sa_k;
    const float* b;
    int64_t sb_b, sb_k, sb_n;
    float* c;
    int64_t sc_b, sc_m;
    const float* cin;
    int64_t sci_b, sci_m, sci_n;
    float alpha, beta;
    int64_t M, N, K, batch;
    int64_t a_rows_per_batch, b_rows_per_batch;  // 0 when that operand is broadcast over the batch
};

__device__ __forceinline__ void fixup_one(const FixupParams& p, int64_t bt, int64_t i, int64_t j) {
    const float* a = p.a + bt * p.sa_b + i * p.sa_m;
    const float* b = p.b + bt * p.sb_b + j * p.sb_n;
    float acc = 0.0f;
    for (int64_t k = 0; k < p.K; ++k) acc = fmaf(a[k * p.sa_k], b[k * p.sb_k], acc);
    float v = p.alpha * acc;
    if (p.cin != nullptr) v += p.beta * p.cin[bt * p.sci_b + i * p.sci_m + j * p.sci_n];
    p.c[bt * p.sc_b + i * p.sc_m + j] = v;
}

// Block per (batch, row of A) / (batch, column of B): recompute the flagged
// ones.  Unflagged blocks leave at once.
__global__ void __launch_bounds__(256) fixup_rows_kernel(FixupParams p, const unsigned* __restrict__ a_flags) {
    const int64_t bt = blockIdx.y, i = blockIdx.x;
    if (!a_flags[(p.a_rows_per_batch ? bt : 0) * p.M + i]) return;
    for (int64_t j = threadIdx.x; j < p.N; j += blockDim.x) fixup_one(p, bt, i, j);
}

__global__ void __launch_bounds__(256) fixup_cols_kernel(FixupParams p, const unsigned* __restrict__ b_flags) {
    const int64_t bt = blockIdx.y, j = blockIdx.x;
    if (!b_flags[(p.b_rows_per_batch ? bt : 0) * p.N + j]) return;
    for (int64_t i = threadIdx.x; i < p.M; i += blockDim.x) fixup_one(p, bt, i, j);
}

// A K-major view of an operand: `rows` rows of K floats at base + b*s_b + r*s_r.
struct KMajor {
    const float* base;
    int64_t s_b, s_r;
};

// Split one operand ([batches, R, K] with strides sb_, sr, sk) into a
// [batches * R, ld] scratch of split rows; MN-major operands are first
// copied K-major.
void split_operand(const float* src, int64_t batches, int64_t R, int64_t K, int64_t s_b, int64_t s_r,
                   int64_t s_k, int b_side, float* dst, int64_t ld, unsigned* flags,
                   std::unique_ptr<Scratch>& kmajor, int dev, cudaStream_t stream) {
    KMajor v{src, s_b, s_r};
    if (!(s_k == 1 || K == 1)) {
        kmajor.reset(new Scratch(sizeof(float) * batches * R * K, dev, stream));
        tpb_tensor s{}, d{};
        s.data = const_cast<float*>(src);
        s.dtype = d.dtype = TPB_F32;
        s.ndim = d.ndim = 3;
        const int64_t sizes[3] = {batches, R, K};
        const int64_t sstr[3] = {s_b, s_r, s_k};
        const int64_t dstr[3] = {R * K, K, 1};
        for (int i = 0; i < 3; ++i) {
            s.sizes[i] = d.sizes[i] = sizes[i];
            s.strides[i] = sstr[i];
            d.strides[i] = dstr[i];
        }
        d.data = kmajor->get();
        copy_impl(d, s, stream, dev);
        v = KMajor{static_cast<const float*>(kmajor->get()), R * K, K};
    }
    const int64_t rows = batches * R;
    dim3 grid(static_cast<unsigned>(std::min<int64_t>((K + 255) / 256, 64)),
              static_cast<unsigned>(std::min<int64_t>(rows, 65535)));
    split_tf32_kernel<<<grid, 256, 0, stream>>>(v.base, dst, rows, R, K, v.s_b, v.s_r, ld, b_side, flags);
    check_launch("split_tf32");
}

// Problems this large take the split path; smaller ones stay on the CUDA
// cores, where the three-fold operand traffic and launches would not pay.
bool use_split_tf32(const GemmProblem& p) {
    static const char* force = std::getenv("TPB200_GEMM_F32");
    if (force != nullptr && std::strcmp(force, "simt") == 0) return false;
    if (3 * p.K >= (int64_t(1) << 31) || p.M >= (int64_t(1) << 31) || p.N >= (int64_t(1) << 31)) return false;
    if (p.batch > 65535) return false;  // the fix-up grids' y extent
    // An operand broadcast over the batch (batch stride 0) has no batched
    // tensor map; such products take the CUDA-core kernel, as TF32 ones do.
    if (p.batch > 1 && (p.sa_b == 0 || p.sb_b == 0)) return false;
    return p.M >= 128 && p.N >= 128 && p.K >= 16 && p.M * p.N * p.K * p.batch >= (int64_t(1) << 27);
}

bool gemm_f32_split(const GemmProblem& p, int dev, cudaStream_t stream) {
    if (!use_split_tf32(p)) return false;
    const int64_t chunks = (p.K + kSplitChunk - 1) / kSplitChunk;
    const int64_t ld = chunks * 3 * kSplitChunk;  // a multiple of 4: 16-byte row pitch
    const int64_t a_batches = p.sa_b == 0 ? 1 : p.batch;
    const int64_t b_batches = p.sb_b == 0 ? 1 : p.batch;
    Scratch a3(sizeof(float) * a_batches * p.M * ld, dev, stream);
    Scratch b3(sizeof(float) * b_batches * p.N * ld, dev, stream);
    const int64_t nflags = a_batches * p.M + b_batches * p.N;
    Scratch flags(sizeof(unsigned) * nflags, dev, stream);
    TPB_CUDA(cudaMemsetAsync(flags.get(), 0, sizeof(unsigned) * nflags, stream));
    unsigned* a_flags = static_cast<unsigned*>(flags.get());
    unsigned* b_flags = a_flags + a_batches * p.M;
    std::unique_ptr<Scratch> a_k, b_k;
    split_operand(static_cast<const float*>(p.a), a_batches, p.M, p.K, p.sa_b, p.sa_m, p.sa_k, 0,
                  static_cast<float*>(a3.get()), ld, a_flags, a_k, dev, stream);
    split_operand(static_cast<const float*>(p.b), b_batches, p.N, p.K, p.sb_b, p.sb_n, p.sb_k, 1,
                  static_cast<float*>(b3.get()), ld, b_flags, b_k, dev, stream);
    a_k.reset();
    b_k.reset();
    for (int64_t j = 0; j < chunks; ++j) {
        const int64_t kj = std::min(kSplitChunk, p.K - j * kSplitChunk);
        GemmProblem q = p;
        q.K = 3 * kj;
        q.a = static_cast<const float*>(a3.get()) + j * 3 * kSplitChunk;
        q.sa_k = 1;
        q.sa_m = ld;
        q.sa_b = a_batches > 1 ? p.M * ld : 0;
        q.b = static_cast<const float*>(b3.get()) + j * 3 * kSplitChunk;
        q.sb_k = 1;
        q.sb_n = ld;
        q.sb_b = b_batches > 1 ? p.N * ld : 0;
        q.flags = p.flags | TPB_GEMM_ALLOW_TF32;
        if (j > 0) {  // out = alpha * A_j.B_j + out
            q.cin = p.c;
            q.sci_b = p.sc_b;
            q.sci_m = p.sc_m;
            q.sci_n = 1;
            q.beta = 1.0;
        }
        TPB_CHECK(gemm_tc_typed<float>(q, dev, stream, CU_TENSOR_MAP_DATA_TYPE_FLOAT32),
                  "gemm: the split-TF32 operands were not accepted by the tensor-core kernel");
    }
    FixupParams f{};
    f.a = static_cast<const float*>(p.a);
    f.sa_b = p.sa_b;
    f.sa_m = p.sa_m;
    f.sa_k = p.sa_k;
    f.b = static_cast<const float*>(p.b);
    f.sb_b = p.sb_b;
    f.sb_k = p.sb_k;
    f.sb_n = p.sb_n;
    f.c = static_cast<float*>(p.c);
    f.sc_b = p.sc_b;
    f.sc_m = p.sc_m;
    f.cin = static_cast<const float*>(p.cin);
    f.sci_b = p.sci_b;
    f.sci_m = p.sci_m;
    f.sci_n = p.sci_n;
    f.alpha = static_cast<float>(p.alpha);
    f.beta = static_cast<float>(p.beta);
    f.M = p.M;
    f.N = p.N;
    f.K = p.K;
    f.batch = p.batch;
    f.a_rows_per_batch = a_batches > 1 ? p.M : 0;
    f.b_rows_per_batch = b_batches > 1 ? p.N : 0;
    fixup_rows_kernel<<<dim3(static_cast<unsigned>(p.M), static_cast<unsigned>(p.batch)), 256, 0, stream>>>(
        f, a_flags);
    check_launch("gemm_f32_fixup_rows");
    fixup_cols_kernel<<<dim3(static_cast<unsigned>(p.N), static_cast<unsigned>(p.batch)), 256, 0, stream>>>(
        f, b_flags);
    check_launch("gemm_f32_fixup_cols");
    return true;
}

}  // namespace

bool gemm_tc(const GemmProblem& p, int dev, cudaStream_t stream) {
    if (p.M == 0 || p.N == 0 || p.K == 0) return false;
    if (p.epi != kEpiPlain && p.dtype != TPB_BF16) return false;
    switch (p.dtype) {
        case TPB_BF16: return gemm_tc_typed<__nv_bfloat16>(p, dev, stream, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16);
        case TPB_F16: return gemm_tc_typed<__half>(p, dev, stream, CU_TENSOR_MAP_DATA_TYPE_FLOAT16);
        case TPB_F32:
            if (!(p.flags & TPB_GEMM_ALLOW_TF32)) return gemm_f32_split(p, dev, stream);
            return gemm_tc_typed<float>(p, dev, stream, CU_TENSOR_MAP_DATA_TYPE_FLOAT32);
        default: return false;
    }
}

}  // namespace tpb

extern "C" int tp_b200_set_gemm_tile_order(int dev, int dynamic) {
    return tpb::guarded([&] {
        TPB_CHECK(dev >= 0 && dev < 64, "invalid device index %d", dev);
        tpb::g_gemm_dynamic[dev].store(dynamic != 0, std::memory_order_relaxed);
    });
}
