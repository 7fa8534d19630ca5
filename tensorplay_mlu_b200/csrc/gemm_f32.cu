// float32 feed-forward products at fp32 accuracy on the tensor cores, one
// launch each: the forward layers with their epilogue, dz w and dz^T x.
//
// Every operand element is split on its way into shared memory, x = hi + lo
// with hi = x rounded to TF32 and lo = x - hi, read by the MMA as TF32 too, and
// a product is hi hi + hi lo + lo hi: three TF32 MMAs, the last two into an
// accumulator of their own.  The dropped lo lo and lo's lost bits are at most
// 2^-21 of |a b|.  The tensor core rounds its running sum towards zero, so a
// TMEM accumulator only takes kChain k-blocks (kChain * 32 terms); warps of
// their own then add it to fp32 sums in registers, rounded to nearest, while
// the MMAs fill the other accumulator.
//
// What bounds it: the loader warps' instructions (2048 x 4096 -> 4096: 745 us,
// 92 TFLOP/s, tensor pipe 26 %), among them spills of the 128-row tiles: 17
// warps leave 96 registers a thread, and a K-major tile stores 132 and loads
// 188 bytes of them.  Sixteen loader warps on narrower tiles, and persistent
// CTAs, measured slower.
//
// Why not the plain product's pre-split copies: those write and read each
// operand three times and take a launch per 1024 of K, and have no epilogue.
// They win where the product is large, 4096^3: 1.03 ms against 1.44 here.
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
//
// Where the caller allows one TF32 product (ONCE, kernels of their own) only
// hi hi is computed, and lo is neither made nor stored.  There a rounding past
// the range shows as an infinity, so sums that are infinite are recomputed too.

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
    int vec_w, vec_x;  // 16-byte loads along the unit stride
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
    static constexpr size_t kSmem = size_t(kStages) * kStageBytes + 1024 + 256;
    static constexpr int kTmemCols = 4 * NT;  // two accumulators: hi hi, and the cross terms
    static_assert(NT * 512 <= kStages * int(kStageBytes), "partial sums fit the stages");
};

__device__ __forceinline__ float4 ldg128(const float* p) {
    float4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                 : "l"(p));
    return v;
}

// x for a single TF32 product: rounded to nearest, ties away.  An infinity stays
// one, and a NaN one, whatever its payload (the addition below would carry
// 0x7fffffff into a zero); a finite x past the largest TF32 becomes an infinity.
__device__ __forceinline__ float tf32_once(float x) {
    uint32_t r;
    asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(r) : "f"(x));
    return __uint_as_float(r);
}

// hi and lo of four consecutive k (chunk q) of row r into their swizzled
// tiles.  hi is rounded to nearest, ties away; lo's low bits are the MMA's to
// drop (2^-10 of lo).  An infinity keeps hi = inf and makes lo NaN; a NaN makes
// lo NaN, whatever the addition leaves of it in hi (0x7fffffff: a zero).
// ONCE: hi alone, which then has to keep them itself.
template <bool ONCE>
__device__ __forceinline__ void store_split(uint8_t* hi_tile, uint32_t lo_offset, int r, int q, float4 v) {
    uint8_t* at = hi_tile + r * 128 + ((q ^ (r & 7)) << 4);
    if constexpr (ONCE) {
        *reinterpret_cast<float4*>(at) = make_float4(tf32_once(v.x), tf32_once(v.y), tf32_once(v.z), tf32_once(v.w));
        return;
    }
    const auto hi = [](float x) { return __uint_as_float((__float_as_uint(x) + 0x1000u) & 0xffffe000u); };
    const float4 h = make_float4(hi(v.x), hi(v.y), hi(v.z), hi(v.w));
    *reinterpret_cast<float4*>(at) = h;
    *reinterpret_cast<float4*>(at + lo_offset) = make_float4(v.x - h.x, v.y - h.y, v.z - h.z, v.w - h.w);
}

// One operand's share of a loader thread: kRows rows by 32 k of a block.
// Along k (MN false): chunk q of rows r0 + 32 i, eight lanes a row.  Along the
// rows (MN true): rows r0 .. r0 + 3 at four k, transposed by the store; the
// lanes are numbered so that eight neighbours store to distinct banks.
template <bool MN, int kRows, bool ONCE>
struct Loader {
    static constexpr int kRegs = MN ? 4 : kRows / 32;
    const float* ptr[MN ? 1 : kRegs];
    int64_t s_k;
    int r0, q, K;
    int rows;  // valid rows from r0 on (MN), a bit for each i (else)
    bool vec, active;

    // row_ptr(r): element (r, 0) of the tile's row r, null outside.
    template <typename RowPtr>
    __device__ __forceinline__ void init(int K_, int64_t s_k_, bool vec_, RowPtr row_ptr) {
        K = K_;
        s_k = s_k_;
        vec = vec_;
        rows = 0;
        if constexpr (MN) {
            const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
            constexpr int kGroups = kRows / 32;
            active = warp < 2 * kGroups;
            r0 = (warp % kGroups) * 32 + (((lane >> 3) << 1) | ((lane >> 2) & 1)) * 4;
            q = (warp / kGroups) * 4 + (lane & 3);
            ptr[0] = active ? row_ptr(r0) : nullptr;
            if (ptr[0] != nullptr) {
                rows = 1;
#pragma unroll
                for (int j = 1; j < 4; ++j) rows += row_ptr(r0 + j) == ptr[0] + j ? 1 : 0;
            }
        } else {
            active = true;
            q = threadIdx.x & 7;
            r0 = threadIdx.x >> 3;
#pragma unroll
            for (int i = 0; i < kRegs; ++i) {
                ptr[i] = row_ptr(r0 + 32 * i);
                if (ptr[i] != nullptr) rows |= 1 << i;
            }
        }
    }

    __device__ __forceinline__ void fetch(int kb, float4 (&reg)[kRegs]) const {
        const int k = kb * 32 + q * 4;
#pragma unroll
        for (int i = 0; i < kRegs; ++i) reg[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if constexpr (MN) {
            if (rows == 0) return;
            const float* p = ptr[0] + int64_t(k) * s_k;
            if (vec && rows == 4 && k + 4 <= K) {
#pragma unroll
                for (int e = 0; e < 4; ++e) reg[e] = ldg128(p + e * s_k);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if (k + e >= K) break;
                    const float* pe = p + e * s_k;
                    reg[e].x = pe[0];
                    if (rows > 1) reg[e].y = pe[1];
                    if (rows > 2) reg[e].z = pe[2];
                    if (rows > 3) reg[e].w = pe[3];
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < kRegs; ++i) {
                if (!((rows >> i) & 1)) continue;
                const float* p = ptr[i] + k;
                if (vec && k + 4 <= K) {
                    reg[i] = ldg128(p);
                } else {
                    if (k < K) reg[i].x = p[0];
                    if (k + 1 < K) reg[i].y = p[1];
                    if (k + 2 < K) reg[i].z = p[2];
                    if (k + 3 < K) reg[i].w = p[3];
                }
            }
        }
    }

    __device__ __forceinline__ void store(uint8_t* tile, uint32_t lo_offset, const float4 (&reg)[kRegs]) const {
        if constexpr (MN) {
            if (!active) return;
            store_split<ONCE>(tile, lo_offset, r0, q, make_float4(reg[0].x, reg[1].x, reg[2].x, reg[3].x));
            store_split<ONCE>(tile, lo_offset, r0 + 1, q, make_float4(reg[0].y, reg[1].y, reg[2].y, reg[3].y));
            store_split<ONCE>(tile, lo_offset, r0 + 2, q, make_float4(reg[0].z, reg[1].z, reg[2].z, reg[3].z));
            store_split<ONCE>(tile, lo_offset, r0 + 3, q, make_float4(reg[0].w, reg[1].w, reg[2].w, reg[3].w));
        } else {
#pragma unroll
            for (int i = 0; i < kRegs; ++i) store_split<ONCE>(tile, lo_offset, r0 + 32 * i, q, reg[i]);
        }
    }
};

template <int PARTS, int NT, bool W_MN, bool X_MN, bool ONCE>
__global__ void __launch_bounds__(F32Shape<NT>::kThreads, 1) gemm_f32_kernel(const FewParams p, const F32Operands o) {
    using S = F32Shape<NT>;
    constexpr int kStages = S::kStages;
    constexpr int kColumns = 128 / PARTS;
    using LoadW = Loader<W_MN, 128, ONCE>;
    using LoadX = Loader<X_MN, NT, ONCE>;
    constexpr int kDepth = LoadW::kRegs + LoadX::kRegs > 6 ? 2 : 3;  // k-blocks in registers
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
        LoadW load_w;
        LoadX load_x;
        load_w.init(p.K, o.sw_k, o.vec_w != 0, [&](int r) -> const float* {
            const int col = n0 + r % kColumns;
            return col < p.N ? o.w + (col + int64_t(r / kColumns) * p.N) * o.sw_n : nullptr;
        });
        load_x.init(p.K, o.sx_k, o.vec_x != 0, [&](int r) -> const float* {
            return m0 + r < p.M ? o.x + int64_t(m0 + r) * o.sx_m : nullptr;
        });
        float4 reg_w[kDepth][LoadW::kRegs], reg_x[kDepth][LoadX::kRegs];
#pragma unroll
        for (int d = 0; d < kDepth - 1; ++d) {
            if (kb0 + d < kb1) {
                load_w.fetch(kb0 + d, reg_w[d]);
                load_x.fetch(kb0 + d, reg_x[d]);
            }
        }
        int stage = 0;
        uint32_t phase = 0;
        bool ok = true;
        for (int kb = kb0; kb < kb1 && ok; kb += kDepth) {
#pragma unroll
            for (int d = 0; d < kDepth; ++d) {
                if (kb + d >= kb1 || !ok) break;
                if (kb + d + kDepth - 1 < kb1) {
                    load_w.fetch(kb + d + kDepth - 1, reg_w[(d + kDepth - 1) % kDepth]);
                    load_x.fetch(kb + d + kDepth - 1, reg_x[(d + kDepth - 1) % kDepth]);
                }
                int granted = 1;
                if (lane == 0) granted = mbar_wait(smem_addr(&empty[stage]), phase ^ 1, abort_flag) ? 1 : 0;
                ok = __shfl_sync(0xffffffffu, granted, 0) != 0;
                if (!ok) break;
                uint8_t* at = smem + stage * S::kStageBytes;
                load_w.store(at, S::kWBytes, reg_w[d]);
                load_x.store(at + 2 * S::kWBytes, S::kXBytes, reg_x[d]);
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
            const uint64_t desc0 = sw128_desc(smem_addr(smem), 16, 1024);
            const uint32_t wide = p.idesc + (uint32_t(NT >> 3) << 17);  // N = 2 NT
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
                // Descriptors advance in 16-byte units of the address field.
                const uint64_t w_hi = desc0 + uint32_t(stage) * (S::kStageBytes / 16), w_lo = w_hi + S::kWBytes / 16;
                const uint64_t x_hi = w_lo + S::kWBytes / 16;  // x_lo behind it
                const uint32_t d = tmem + acc * 2 * NT;
                uint32_t more = i % kChain != 0 ? 1u : 0u;
                if constexpr (ONCE) {
#pragma unroll
                    for (int kk = 0; kk < 4; ++kk) {
                        umma<true>(d, w_hi + kk * 2, x_hi + kk * 2, p.idesc, more);
                        more = 1u;
                    }
                } else {
                    // One pass over w_hi gives hi hi (columns 0 .. NT - 1) and
                    // hi lo (the next NT), which lo hi joins.
#pragma unroll
                    for (int kk = 0; kk < 4; ++kk) {
                        umma<true>(d, w_hi + kk * 2, x_hi + kk * 2, wide, more);
                        more = 1u;
                        umma<true>(d + NT, w_lo + kk * 2, x_hi + kk * 2, p.idesc, 1u);
                    }
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
            const uint32_t at = tmem + (uint32_t(quad * 32) << 16) + acc * 2 * NT + col0;
#pragma unroll
            for (int c = 0; c < S::kAccCols; c += 16) {
                uint32_t r[16];
                if constexpr (!ONCE) {
                    tmem_ld16(at + NT + c, r);
                    tmem_wait_ld();
#pragma unroll
                    for (int j = 0; j < 16; ++j) sum[c + j] += __uint_as_float(r[j]);
                }
                tmem_ld16(at + c, r);
                tmem_wait_ld();
#pragma unroll
                for (int j = 0; j < 16; ++j) sum[c + j] += __uint_as_float(r[j]);
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
    cluster_sync();  // every CTA's partial sums are in its shared memory
    // A NaN sum (ONCE: or an infinite one) is computed again as fp32 arithmetic
    // would.
    finish_rows<float, PARTS, NT>(
        p, reinterpret_cast<const float*>(smem), m0, n0, warp, S::kThreads / 32, rank, ranks,
        [&](int64_t m, int64_t n, int q, float& z) {
            if ((ONCE ? fabsf(z) < INFINITY : z == z) || n >= p.N) return;
            const float* w = o.w + (n + int64_t(q) * p.N) * o.sw_n;
            const float* x = o.x + m * o.sx_m;
            z = 0.0f;
            for (int64_t k = 0; k < p.K && z == z; ++k) z = fmaf(w[k * o.sw_k], x[k * o.sx_k], z);
        });
    cluster_sync();  // no CTA leaves while another reads its shared memory
    if (warp == kLoadWarps) {
        __syncwarp();
        tc_fence_after();
        tmem_dealloc(tmem, S::kTmemCols);
    }
}

template <int PARTS, int NT, bool W_MN, bool X_MN, bool ONCE>
void launch_f32(FewParams& p, const F32Operands& o, int dev, cudaStream_t stream) {
    using S = F32Shape<NT>;
    auto kern = gemm_f32_kernel<PARTS, NT, W_MN, X_MN, ONCE>;
    const Slots& slots = cluster_slots<gemm_f32_kernel<PARTS, NT, W_MN, X_MN, ONCE>>(S::kThreads, S::kSmem, dev);
    p.idesc = (1u << 4) | (2u << 7) | (2u << 10) | (uint32_t(NT >> 3) << 17) | (uint32_t(128 >> 4) << 24);
    p.row_tiles = (p.M + NT - 1) / NT;
    const int64_t tiles = int64_t(p.row_tiles) * ((p.N + 128 / PARTS - 1) / (128 / PARTS));
    const int split = choose_split(tiles, p.k_blocks, slots, 16);
    launch_cluster(kern, tiles * split, split, S::kThreads, S::kSmem, stream, p, o);
    check_launch("gemm_f32");
}

template <int PARTS, bool W_MN, bool X_MN, bool ONCE>
void launch_rows(FewParams& p, const F32Operands& o, int dev, cudaStream_t stream) {
    // 128 rows a tile where that still gives every SM one, fewer otherwise.
    const int64_t columns = (p.N + 128 / PARTS - 1) / (128 / PARTS);
    if (p.M <= 32) launch_f32<PARTS, 32, W_MN, X_MN, ONCE>(p, o, dev, stream);
    else if (p.M <= 64 || columns * ((p.M + 127) / 128) < num_sms(dev))
        launch_f32<PARTS, 64, W_MN, X_MN, ONCE>(p, o, dev, stream);
    else launch_f32<PARTS, 128, W_MN, X_MN, ONCE>(p, o, dev, stream);
}

template <int PARTS, bool W_MN, bool X_MN>
void launch_products(bool once, FewParams& p, const F32Operands& o, int dev, cudaStream_t stream) {
    if (once) launch_rows<PARTS, W_MN, X_MN, true>(p, o, dev, stream);
    else launch_rows<PARTS, W_MN, X_MN, false>(p, o, dev, stream);
}

// 16-byte loads: along k rows have to start on such boundaries, along the rows
// every k.
bool vectors(const float* p, int64_t stride) { return aligned16(p) && stride % 4 == 0; }

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
    const bool once = (q.flags & TPB_GEMM_ALLOW_TF32) != 0;  // one TF32 product is enough
    // A layer reads w and x along k; dz w reads w along its rows' elements,
    // dz^T x both operands (w's strides are then both 1 when it has one column).
    const bool x_mn = q.sx_k != 1, w_mn = q.sw_k != 1 || x_mn;
    o.vec_w = vectors(o.w, w_mn ? o.sw_k : o.sw_n);
    o.vec_x = vectors(o.x, x_mn ? o.sx_k : o.sx_m);
    if (q.parts == 2) launch_products<2, false, false>(once, p, o, dev, stream);
    else if (!w_mn) launch_products<1, false, false>(once, p, o, dev, stream);
    else if (!x_mn) launch_products<1, true, false>(once, p, o, dev, stream);
    else launch_products<1, true, true>(once, p, o, dev, stream);
}

}  // namespace tpb
