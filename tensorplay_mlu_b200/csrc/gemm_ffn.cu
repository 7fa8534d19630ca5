// The feed-forward products on tcgen05 tensor cores: a linear layer with its
// bias, activation and residual, and the gated block's two projections with
// the activation and their product (no single counterpart in the reference;
// see include/tpb200.h).
//
// Both are the CTA-pair kernel of gemm_tc.cuh with another epilogue, so the
// pre-activations stay in TMEM: written out, they would cost the gated block
// 8 M F bytes of traffic (written, read back) beside the 2 M F of its result.
//   * linear_act: a 256 x 256 tile of x W^T, as in a plain product.
//   * gated_linear: the pair's tile is 256 rows by 128 gate and 128 up
//     columns; the leader CTA stages the gate rows of W and its peer the up
//     rows, so each CTA's accumulator holds both pre-activations of its 128
//     rows (columns 0-127 and 128-255) and the epilogue multiplies them
//     without an exchange.  The mainloop is the plain product's.
// Sums, bias, activation, gate and residual are fp32; the result is rounded
// once.  Pre-activations saved for the backward pass are rounded to T, or to
// 8 bits (act.cuh): a TMEM lane is a row and a 32-column chunk is exactly one
// checkpoint block, so its scale is found in one thread's registers.

#include "act.cuh"
#include "gemm_tc.cuh"

namespace tpb {
namespace {

// bias[n .. n + 32) added to a chunk (every lane reads the same addresses).
template <typename T>
__device__ __forceinline__ void add_bias_chunk(const T* bias, int64_t n, int64_t N, float (&z)[32]) {
    if (n + 32 <= N && (reinterpret_cast<uintptr_t>(bias + n) & 15u) == 0) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            float f[8];
            unpack_vec(reinterpret_cast<const Vec<T, 8>*>(bias + n)[q], f);
#pragma unroll
            for (int j = 0; j < 8; ++j) z[q * 8 + j] += f[j];
        }
    } else {
#pragma unroll
        for (int j = 0; j < 32; ++j) {
            if (n + j < N) z[j] += load_as<float>(bias[n + j]);
        }
    }
}

// One row's 32-element block as int8 into a staging tile; returns the
// exponent.
template <typename T>
__device__ __forceinline__ uint8_t stage_checkpoint(uint8_t* stage, int lane, const float (&z)[32]) {
    float amax = 0.0f;
#pragma unroll
    for (int j = 0; j < 32; ++j) amax = max_nan(amax, fabsf(z[j]));
    float qmax;
    const int stored = ckpt_exponent<T>(amax, qmax);
    const Vec<int8_t, 32> q = ckpt_quantise<32>(z, stored, qmax);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        *reinterpret_cast<Vec<int8_t, 16>*>(stage + stage_offset(1, lane, h * 16)) =
            reinterpret_cast<const Vec<int8_t, 16>*>(&q)[h];
    }
    return static_cast<uint8_t>(stored);
}

// Rows [row0, row0 + 32) (this warp's TMEM lanes) of one accumulator.  half:
// which half of the tile's result columns this warp stores, in chunks of 32.
template <typename T, int EPI>
__device__ void store_ffn(const TcParams& p, const CUtensorMap* tmC, const CUtensorMap* tmSaved, uint8_t* stage,
                          uint32_t t_rows, int half, int64_t row0, int64_t n_tile0) {
    constexpr int kParts = EPI == kEpiGated ? 2 : 1;
    constexpr int kCols = pair_tile_columns<EPI>() / 2;
    const FfnParams& f = p.ffn;
    const int lane = threadIdx.x & 31;
    const int64_t rows = p.M - row0;
    const T* bias = static_cast<const T*>(f.bias);
    uint8_t* stage2 = stage + staging_bytes<T>();
    for (int c0 = half * kCols; c0 < (half + 1) * kCols; c0 += 32) {
        const int64_t n = n_tile0 + c0;
        if (rows <= 0 || n >= p.N) break;
        const int64_t cols = p.N - n;
        uint32_t raw[kParts][32];
        __syncwarp();
#pragma unroll
        for (int q = 0; q < kParts; ++q) tmem_ld32(t_rows + c0 + q * 128, raw[q]);
        // The residual's loads are in flight while the accumulator arrives.
        // Rows on 16-byte boundaries: a lane's own row.  Others: a lane's own
        // column, transposed through the staging tile below.
        Vec<T, 32> res;
        const bool res_vec = f.residual_vec && cols >= 32;
        if (EPI == kEpiAct && f.residual != nullptr) {
            const T* r = static_cast<const T*>(f.residual) + row0 * f.sres_m + n;
            if (res_vec) {
                if (lane < rows) {
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        reinterpret_cast<Vec<T, 8>*>(&res)[q] =
                            reinterpret_cast<const Vec<T, 8>*>(r + lane * f.sres_m)[q];
                    }
                }
            } else {
#pragma unroll
                for (int i = 0; i < 32; ++i) res.v[i] = i < rows && lane < cols ? r[i * f.sres_m + lane] : T(0.0f);
            }
        }
        tmem_wait_ld();
        float z[kParts][32];
#pragma unroll
        for (int q = 0; q < kParts; ++q) {
#pragma unroll
            for (int j = 0; j < 32; ++j) z[q][j] = __uint_as_float(raw[q][j]);
            if (bias != nullptr) add_bias_chunk<T>(bias + q * p.N, n, p.N, z[q]);
            if (cols < 32) {  // columns past N hold other rows of W, or nothing
#pragma unroll
                for (int j = 0; j < 32; ++j) {
                    if (j >= cols) z[q][j] = 0.0f;
                }
            }
        }
        // The previous stores from the staging tiles have finished reading.
        if (lane == 0) bulk_wait_group_read0();
        __syncwarp();
        if (f.saved != nullptr) {
            // Two tiles: z into the second (gate into the first, which the
            // result takes over once it has been read).
            uint8_t* tile[2] = {kParts == 2 ? stage : stage2, stage2};
#pragma unroll
            for (int q = 0; q < kParts; ++q) {
                Vec<T, 32> packed;
                pack_vec(z[q], packed);
                stage_chunk<T>(tile[q], lane, packed);
            }
            if (f.saved_tma) fence_proxy_async_smem();
            __syncwarp();
            if (f.saved_tma) {
                if (lane == 0) {
#pragma unroll
                    for (int q = 0; q < kParts; ++q) tma_store_3d(tmSaved, smem_addr(tile[q]), int(n), q, int(row0));
                    bulk_commit_group();
                    if (kParts == 2) bulk_wait_group_read0();
                }
            } else {
                T* dst = static_cast<T*>(f.saved) + row0 * f.ssaved_m + n;
#pragma unroll
                for (int q = 0; q < kParts; ++q) {
                    store_staged_rows<T>(tile[q], lane, dst + q * f.ssaved_p, f.ssaved_m, cols, rows);
                }
            }
            if (kParts == 2) __syncwarp();
        }
        if (f.values != nullptr) {
            if (f.saved != nullptr) {
                // Both forms are kept: the second tile once more, when z has
                // left it.
                if (lane == 0) bulk_wait_group_read0();
                __syncwarp();
            }
#pragma unroll
            for (int q = 0; q < kParts; ++q) {
                const uint8_t stored = stage_checkpoint<T>(stage2 + q * 1024, lane, z[q]);
                if (lane < rows) f.exponents[((row0 + lane) * kParts + q) * f.nb + (n >> 5)] = stored;
            }
            if (!f.values_tma) {
                __syncwarp();
#pragma unroll
                for (int q = 0; q < kParts; ++q) {
                    store_staged_rows<int8_t>(stage2 + q * 1024, lane, f.values + (row0 * kParts + q) * p.N + n,
                                              int64_t(kParts) * p.N, cols, rows);
                }
            }
        }
        act_values<true, 32>(f.act, z[0]);
        if constexpr (kParts == 2) {
#pragma unroll
            for (int j = 0; j < 32; ++j) z[0][j] *= z[1][j];
        }
        if (EPI == kEpiAct && f.residual != nullptr) {
            if (!res_vec) {
#pragma unroll
                for (int i = 0; i < 32; ++i) *reinterpret_cast<T*>(stage + stage_offset(2, i, lane)) = res.v[i];
                __syncwarp();
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    reinterpret_cast<Vec<T, 8>*>(&res)[q] =
                        *reinterpret_cast<const Vec<T, 8>*>(stage + stage_offset(2, lane, q * 8));
                }
                __syncwarp();
            }
            if (lane < rows) {
                float r[32];
                unpack_vec(res, r);
#pragma unroll
                for (int j = 0; j < 32; ++j) z[0][j] += r[j];
            }
        }
        Vec<T, 32> packed;
        pack_vec(z[0], packed);
        stage_chunk<T>(stage, lane, packed);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
            if (p.tma_store) tma_store_2d(tmC, smem_addr(stage), int(n), int(row0));
            if (f.values_tma) {
#pragma unroll
                for (int q = 0; q < kParts; ++q) {
                    tma_store_3d(tmSaved, smem_addr(stage2 + q * 1024), int(n), q, int(row0));
                }
            }
            bulk_commit_group();
        }
        if (!p.tma_store) {
            store_staged_rows<T>(stage, lane, static_cast<T*>(p.c) + row0 * p.sc_m + n, p.sc_m, cols, rows);
            __syncwarp();
        }
    }
}

// Map of [M, parts, N] for the saved tensors' TMA stores: boxes of 32 columns
// of one part by 32 rows.
CUtensorMap make_saved_map(void* base, CUtensorMapDataType type, int es, int64_t N, int64_t parts, int64_t M,
                           int64_t part_stride, int64_t row_stride) {
    CUtensorMap map;
    cuuint64_t dims[3] = {static_cast<cuuint64_t>(N), static_cast<cuuint64_t>(parts), static_cast<cuuint64_t>(M)};
    cuuint64_t strides[2] = {static_cast<cuuint64_t>(part_stride * es), static_cast<cuuint64_t>(row_stride * es)};
    cuuint32_t box[3] = {32, 1, 32};
    cuuint32_t estr[3] = {1, 1, 1};
    const CUresult r = encode_fn()(&map, type, 3, base, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                   es == 2 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_32B,
                                   CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    TPB_CHECK(r == CUDA_SUCCESS, "cuTensorMapEncodeTiled (saved) failed (%d)", static_cast<int>(r));
    return map;
}

template <typename T>
void launch_ffn_pair(const FfnProblem& q, int dev, cudaStream_t stream, CUtensorMapDataType type) {
    constexpr int es = sizeof(T);
    constexpr int kEPR = 128 / es;
    const CUtensorMap ma = make_map(q.x, type, es, q.K, q.M, q.sx_m, 1, 0, kBoxRows);
    const CUtensorMap mb = make_map(q.w, type, es, q.K, q.parts * q.N, q.sw_n, 1, 0, kBoxRows);
    TcParams tp{};
    tp.M = static_cast<int>(q.M);
    tp.N = static_cast<int>(q.N);
    tp.K = static_cast<int>(q.K);
    tp.batch = 1;
    tp.k_blocks = static_cast<int>((q.K + kEPR - 1) / kEPR);
    tp.c = q.y;
    tp.sc_m = q.sy_m;
    tp.alpha = 1.0f;
    tp.err = device_error_word(dev);
    tp.tma_store = aligned16(q.y) && q.sy_m > 0 && (q.sy_m * es) % 16 == 0;
    const CUtensorMap mc = tp.tma_store ? make_c_map(q.y, type, es, q.N, q.M, q.sy_m, 1, 0) : ma;
    FfnParams& f = tp.ffn;
    f.bias = q.bias;
    f.residual = q.residual;
    f.sres_m = q.sres_m;
    f.residual_vec = aligned16(q.residual) && (q.sres_m * es) % 16 == 0;
    f.act = q.act;
    f.nb = (q.N + kCkptBlock - 1) / kCkptBlock;
    CUtensorMap ms = ma;
    if (q.saved != nullptr) {
        f.saved = q.saved;
        f.ssaved_m = q.parts * q.N;
        f.ssaved_p = q.N;
        f.saved_tma = aligned16(q.saved) && (q.N * es) % 16 == 0;
        if (f.saved_tma) ms = make_saved_map(q.saved, type, es, q.N, q.parts, q.M, f.ssaved_p, f.ssaved_m);
    }
    if (q.values != nullptr) {
        f.values = q.values;
        f.exponents = q.exponents;
        // One tensor map serves both forms; asked for together, the bytes go
        // out by ordinary stores.
        f.values_tma = q.saved == nullptr && aligned16(q.values) && q.N % 16 == 0;
        if (f.values_tma) {
            ms = make_saved_map(q.values, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, q.N, q.parts, q.M, q.N, q.parts * q.N);
        }
    }
    if (q.parts == 2) launch_tc2<T, false, false, false, kEpiGated>(ma, mb, mc, tp, dev, stream, &ms);
    else launch_tc2<T, false, false, false, kEpiAct>(ma, mb, mc, tp, dev, stream, &ms);
}

}  // namespace

// Whether the split-K kernel (gemm_few.cu) takes a product: up to 64 rows
// always (its bound is the weight's one reading), beyond where its estimated
// time is below this kernel's.  Measured, bf16, us, pair / split: 100 rows x
// 4096 -> 512: 27 / 9; 384 x 4096 -> 2048: 28 / 23; 576 x 1024 -> 2048: 12.6 /
// 11.3; 1024 x 1024 -> 2048: 12.7 / 13.6; 2048 x 4096 -> 6000: 79 / 108; dz^T x
// of 13898 rows, 304 x 120: 77 / 16.  The estimates were fitted to forward
// products that keep nothing, and are worst where the split kernel's epilogue
// stores 8 bits (gated, 300 x 2048 -> 2 * 2048: 19 / 32, the slower one taken)
// and in dz w (512 x 4096 -> 4096: 27 / 32, the same).  The estimate here: 0.31
// us for each 64-deep step of a wave of 256 x 256 tiles, 2.2 us for a wave's
// ramp and epilogue, 5 us once.  Under an SM limit (tp_b200_set_gemm_sm_limit)
// only this kernel, which is persistent, leaves the other SMs alone.
bool few_rows(const FfnProblem& q, int dev) {
    if (q.M <= 64 && q.sx_k == 1) return true;
    if (gemm_sm_budget(dev) < num_sms(dev)) return false;
    const int64_t columns = q.parts == 2 ? 128 : kPairBN;
    const int64_t tiles = ((q.M + kPairBM - 1) / kPairBM) * ((q.N + columns - 1) / columns);
    const int64_t clusters = std::max(1, num_sms(dev) / 2);
    const double waves = static_cast<double>((tiles + clusters - 1) / clusters);
    return gemm_few_us(q, dev) < 5.0 + waves * (0.3125 * static_cast<double>((q.K + 63) / 64) + 2.2);
}

bool gemm_ffn(const FfnProblem& q, int dev, cudaStream_t stream) {
    const int64_t limit = int64_t(1) << 30;
    if (q.K == 0 || q.M >= limit || q.N >= limit || q.K >= limit) return false;
    const bool transposed = q.sw_k != 1 || q.sx_k != 1;
    if (!tma_ok(q.x, 2, q.sx_k != 1 ? q.sx_k : q.sx_m, 1, 0) || !tma_ok(q.w, 2, transposed ? q.sw_k : q.sw_n, 1, 0)) return false;
    TPB_CHECK(q.dtype == TPB_BF16 || q.dtype == TPB_F16, "feed-forward product: 16-bit floats only");
    if (few_rows(q, dev)) {
        gemm_few(q, dev, stream);
    } else if (transposed) {
        // Without an epilogue this is the plain product.
        TPB_CHECK(q.bias == nullptr && q.residual == nullptr && q.saved == nullptr && q.values == nullptr &&
                      q.act == TPB_ACT_NONE,
                  "feed-forward product: a weight read transposed takes no epilogue at %lld rows", (long long)q.M);
        GemmProblem p{};
        p.dtype = q.dtype;
        p.M = q.M;
        p.N = q.N;
        p.K = q.K;
        p.batch = 1;
        p.a = q.x;
        p.sa_m = q.sx_m;
        p.sa_k = q.sx_k;
        p.b = q.w;
        p.sb_k = q.sw_k;
        p.sb_n = q.sw_n;
        p.c = q.y;
        p.sc_m = q.sy_m;
        p.alpha = 1.0;
        return gemm_tc(p, dev, stream);
    } else if (q.dtype == TPB_BF16) {
        launch_ffn_pair<__nv_bfloat16>(q, dev, stream, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16);
    } else {
        launch_ffn_pair<__half>(q, dev, stream, CU_TENSOR_MAP_DATA_TYPE_FLOAT16);
    }
    return true;
}

}  // namespace tpb
