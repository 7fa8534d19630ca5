// What the split-K feed-forward products share (gemm_few.cu for 16-bit floats,
// gemm_f32.cu for float32): the sum of a cluster's partial accumulators over
// distributed shared memory and the epilogue behind it.
//
// A tile is 128 rows of the weight -- the result's contiguous columns, so that
// a warp stores whole segments of a row -- by kNT rows of x.  A gated tile is
// 64 gate and 64 up rows of the weight.
#pragma once

#include "act.cuh"
#include "gemm_tc.cuh"

namespace tpb {
namespace {

// 32 lanes x 16 consecutive 32-bit columns of TMEM into 16 registers.
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
}

struct FewParams {
    int M, N, K;       // rows of x; result columns of one part; contraction
    int k_blocks;
    int row_tiles;     // ceil(M / kNT)
    uint32_t idesc;
    void* y;
    int64_t sy_m;
    FfnParams ffn;
    int* err;
};

template <int V>
__device__ __forceinline__ void ld_cluster(uint32_t cluster_addr, float (&v)[V]) {
    static_assert(V == 2 || V == 4, "8 or 16 bytes");
    if constexpr (V == 4) {
        asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                     : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3])
                     : "r"(cluster_addr)
                     : "memory");
    } else {
        asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v[0]), "=f"(v[1]) : "r"(cluster_addr) : "memory");
    }
}

// V consecutive elements of a row, vectorised where all of them exist on a
// boundary of their size.
template <typename T, int V>
__device__ __forceinline__ void load_few(const T* src, int64_t left, float (&v)[V]) {
    if (left >= V && reinterpret_cast<uintptr_t>(src) % (V * sizeof(T)) == 0) {
        unpack_vec(*reinterpret_cast<const Vec<T, V>*>(src), v);
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = j < left ? load_as<float>(src[j]) : 0.0f;
    }
}
template <typename T, int V>
__device__ __forceinline__ void store_few(T* dst, int64_t left, const float (&v)[V]) {
    if (left >= V && reinterpret_cast<uintptr_t>(dst) % (V * sizeof(T)) == 0) {
        Vec<T, V> o;
        pack_vec(v, o);
        *reinterpret_cast<Vec<T, V>*>(dst) = o;
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j) {
            if (j < left) dst[j] = store_as<T>(v[j]);
        }
    }
}

__device__ __forceinline__ uint32_t cluster_size() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(r));
    return r;
}

// V elements of the residual of row m from column n on (zero without one).
template <typename T, int V>
__device__ __forceinline__ void load_residual(const FewParams& p, int64_t m, int64_t n, float (&r)[V]) {
    const FfnParams& f = p.ffn;
    if (f.residual != nullptr && n < p.N) {
        load_few<T, V>(static_cast<const T*>(f.residual) + m * f.sres_m + n, p.N - n, r);
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j) r[j] = 0.0f;
    }
}

// V results of row m from column n on (a warp holds 32 V consecutive ones):
// z[part] are their summed pre-activations, r the residual.
template <typename T, int PARTS, int V>
__device__ __forceinline__ void finish_few(const FewParams& p, int64_t m, int64_t n, float (&z)[PARTS][V],
                                           const float (&r)[V]) {
    const FfnParams& f = p.ffn;
    const int64_t left = p.N - n;  // may be negative
    const T* bias = static_cast<const T*>(f.bias);
#pragma unroll
    for (int q = 0; q < PARTS; ++q) {
        if (bias != nullptr && left > 0) {
            float b[V];
            load_few<T, V>(bias + int64_t(q) * p.N + n, left, b);
#pragma unroll
            for (int j = 0; j < V; ++j) z[q][j] += b[j];
        }
#pragma unroll
        for (int j = 0; j < V; ++j) {  // rows of the weight past this part
            if (j >= left) z[q][j] = 0.0f;
        }
        if (f.saved != nullptr && left > 0) {
            store_few<T, V>(static_cast<T*>(f.saved) + m * f.ssaved_m + q * f.ssaved_p + n, left, z[q]);
        }
        if (f.values != nullptr) {
            float amax = 0.0f;
#pragma unroll
            for (int j = 0; j < V; ++j) amax = max_nan(amax, fabsf(z[q][j]));
#pragma unroll
            for (int o = 1; o < kCkptBlock / V; o <<= 1) amax = max_nan(amax, __shfl_xor_sync(0xffffffffu, amax, o));
            float qmax;
            const int stored = ckpt_exponent<T>(amax, qmax);
            const Vec<int8_t, V> packed = ckpt_quantise<V>(z[q], stored, qmax);
            const int64_t row = m * PARTS + q;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                if (j < left) f.values[row * p.N + n + j] = packed.v[j];
            }
            if (n % kCkptBlock == 0 && left > 0) f.exponents[row * f.nb + n / kCkptBlock] = static_cast<uint8_t>(stored);
        }
    }
    if (left <= 0) return;
    act_values<Narrow<T>::value, V>(f.act, z[0]);
    if constexpr (PARTS == 2) {
#pragma unroll
        for (int j = 0; j < V; ++j) z[0][j] *= z[1][j];
    }
    if (f.residual != nullptr) add_to<V>(z[0], r);
    store_few<T, V>(static_cast<T*>(p.y) + m * p.sy_m + n, left, z[0]);
}

// Sums a tile over the cluster's ranks and finishes it.  partial: a CTA's sums,
// [row of x][row of the weight tile] floats at the same address in every
// rank; with kWide, a gated tile of 128 columns, [part][row of x][column].  Warp `warp` of `warps` takes every warps-th row of x of this rank's
// share, each lane V columns of it, four ranks' loads in flight at a time,
// added in rank order.  fix(row of x, result column, part, z): a chance to
// replace a sum.
template <typename T, int PARTS, int NT, bool kWide = false, typename Fix>
__device__ __forceinline__ void finish_rows(const FewParams& p, const float* partial, int m0, int n0, int warp,
                                            int warps, int rank, int ranks, Fix fix) {
    constexpr int kColumns = kWide ? 128 : 128 / PARTS;  // result columns of a tile
    constexpr int kV = kColumns / 32;
    const auto offset = [](int m, int q, int lane) {
        return (kWide ? (q * NT + m) * 128 : m * 128 + q * kColumns) + lane * kV;
    };
    const int lane = threadIdx.x & 31;
    const int rows = min(NT, p.M - m0);
    const int64_t n = int64_t(n0) + lane * kV;
    if (ranks == 1) {
        // Four rows at a time, so that their reads are in flight together.
        constexpr int kRows = 4;
        for (int first = warp; first < rows; first += kRows * warps) {
            float z[kRows][PARTS][kV], r[kRows][kV];
#pragma unroll
            for (int i = 0; i < kRows; ++i) {
                const int m = first + i * warps;
                if (m >= rows) break;
                load_residual<T, kV>(p, int64_t(m0) + m, n, r[i]);
#pragma unroll
                for (int q = 0; q < PARTS; ++q) {
                    const Vec<float, kV> v = *reinterpret_cast<const Vec<float, kV>*>(partial + offset(m, q, lane));
#pragma unroll
                    for (int j = 0; j < kV; ++j) z[i][q][j] = v.v[j];
                }
            }
#pragma unroll
            for (int i = 0; i < kRows; ++i) {
                const int m = first + i * warps;
                if (m >= rows) break;
#pragma unroll
                for (int q = 0; q < PARTS; ++q) {
#pragma unroll
                    for (int j = 0; j < kV; ++j) fix(int64_t(m0) + m, n + j, q, z[i][q][j]);
                }
                finish_few<T, PARTS, kV>(p, int64_t(m0) + m, n, z[i], r[i]);
            }
        }
        return;
    }
    for (int m = rank + ranks * warp; m < rows; m += ranks * warps) {
        float z[PARTS][kV], r[kV];
        load_residual<T, kV>(p, int64_t(m0) + m, n, r);
#pragma unroll
        for (int q = 0; q < PARTS; ++q) {
            const uint32_t at = smem_addr(partial + offset(m, q, lane));
#pragma unroll
            for (int j = 0; j < kV; ++j) z[q][j] = 0.0f;
            for (int c0 = 0; c0 < ranks; c0 += 4) {
                float v[4][kV];
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    if (c0 + c < ranks) ld_cluster<kV>(map_to_cta(at, uint32_t(c0 + c)), v[c]);
                }
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    if (c0 + c < ranks) {
#pragma unroll
                        for (int j = 0; j < kV; ++j) z[q][j] += v[c][j];
                    }
                }
            }
#pragma unroll
            for (int j = 0; j < kV; ++j) fix(int64_t(m0) + m, n + j, q, z[q][j]);
        }
        finish_few<T, PARTS, kV>(p, int64_t(m0) + m, n, z, r);
    }
}

// CTAs of a kernel that run at a time in clusters of 1 .. 8 (index 1 .. 8) on a
// device, asked once: GPCs hold different numbers of SMs, so clusters of some
// sizes leave slots empty (clusters of three: 96 tiles x 3 took a second wave
// on 296 slots, 16.2 us against 12.9 us for clusters of two).
struct Slots {
    int ctas[9];
};
template <auto kKernel>
const Slots& cluster_slots(int threads, size_t smem, int dev) {
    const auto kern = kKernel;
    static Slots slots[64];
    static std::mutex lock;
    static std::atomic<bool> ready[64];
    if (!ready[dev].load(std::memory_order_acquire)) {
        std::lock_guard<std::mutex> g(lock);
        if (!ready[dev].load(std::memory_order_relaxed)) {
            TPB_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)));
            for (int c = 1; c <= 8; ++c) {
                cudaLaunchConfig_t cfg = {};
                cfg.gridDim = static_cast<unsigned>(c);
                cfg.blockDim = threads;
                cfg.dynamicSmemBytes = smem;
                cudaLaunchAttribute attr[1];
                attr[0].id = cudaLaunchAttributeClusterDimension;
                attr[0].val.clusterDim.x = static_cast<unsigned>(c);
                attr[0].val.clusterDim.y = 1;
                attr[0].val.clusterDim.z = 1;
                cfg.attrs = attr;
                cfg.numAttrs = 1;
                int clusters = 0;
                TPB_CUDA(cudaOccupancyMaxActiveClusters(&clusters, kern, &cfg));
                slots[dev].ctas[c] = std::max(clusters, 1) * c;
            }
            ready[dev].store(true, std::memory_order_release);
        }
    }
    return slots[dev];
}

// K's split: the cluster size with the fewest k-blocks in a row, a CTA's
// set-up and its share of the sum counted as `fixed` of them.
inline int choose_split(int64_t tiles, int k_blocks, const Slots& slots, int fixed, int64_t* waves_out = nullptr) {
    int split = 1;
    int64_t best = INT64_MAX;
    for (int c = 1; c <= 8 && c <= k_blocks; ++c) {
        const int64_t waves = (tiles * c + slots.ctas[c] - 1) / slots.ctas[c];
        const int64_t cost = waves * ((k_blocks + c - 1) / c + fixed);
        if (cost < best) {
            best = cost;
            split = c;
            if (waves_out != nullptr) *waves_out = waves;
        }
    }
    return split;
}

template <typename K, typename... Args>
void launch_cluster(K* kern, int64_t ctas, int cluster, int threads, size_t smem, cudaStream_t stream,
                    const Args&... args) {
    TPB_CHECK(ctas < (int64_t(1) << 31), "feed-forward product: too many tiles");
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = static_cast<unsigned>(ctas);
    cfg.blockDim = threads;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = static_cast<unsigned>(cluster);
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl_enabled() ? 2 : 1;
    TPB_CUDA(cudaLaunchKernelEx(&cfg, kern, args...));
}

// The operands of a problem's epilogue.
inline FewParams few_params(const FfnProblem& q, int dev, int k_block) {
    FewParams p{};
    p.M = static_cast<int>(q.M);
    p.N = static_cast<int>(q.N);
    p.K = static_cast<int>(q.K);
    p.k_blocks = static_cast<int>((q.K + k_block - 1) / k_block);
    p.y = q.y;
    p.sy_m = q.sy_m;
    p.err = device_error_word(dev);
    FfnParams& f = p.ffn;
    f.bias = q.bias;
    f.residual = q.residual;
    f.sres_m = q.sres_m;
    f.saved = q.saved;
    f.ssaved_m = q.parts * q.N;
    f.ssaved_p = q.N;
    f.values = q.values;
    f.exponents = q.exponents;
    f.nb = (q.N + kCkptBlock - 1) / kCkptBlock;
    f.act = q.act;
    return p;
}

}  // namespace
}  // namespace tpb
