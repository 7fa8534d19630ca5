// Elementwise kernels of the feed-forward operators: the gradients of
// activation and gate with the bias gradient, 8-bit checkpoints, and the
// activation, gate and residual of a layer without input features (others
// have them in their product's epilogue).
//
// tensorplay-mlu runs these as separate activation, mul and add kernels
// (UnaryKernels.cpp:52-104, BinaryKernels.cpp:148-248) and has no
// checkpoints.  All are bound by memory: each reads its inputs and writes its
// results once.

#include "act.cuh"
#include "gemm.h"

namespace tpb {
namespace {

// How a kernel's rows lie: kAligned, every chunk of V elements on a 16-byte
// boundary (8 bytes for checkpoint values) and whole; kWords, on a 4-byte
// boundary, checkpoint values on a 2-byte one, a row's last chunk perhaps
// short; kAnywhere, some rows half a word off.  (One kernel for the last two
// took 1.3 to 1.7 times as long on rows of words.)
constexpr int kAligned = 0;
constexpr int kWords = 1;
constexpr int kAnywhere = 2;

// N bytes at p in words of W bytes (p a multiple of W).
template <typename W, int N>
__device__ __forceinline__ void copy_in(void* to, const void* p) {
#pragma unroll
    for (int i = 0; i < N / int(sizeof(W)); ++i) reinterpret_cast<W*>(to)[i] = reinterpret_cast<const W*>(p)[i];
}

// V consecutive elements of E at p (`count` of them exist).
template <typename E, int V, int MODE>
struct Chunk {
    static constexpr int kBytes = V * int(sizeof(E));
    static constexpr int kPer = (16 < kBytes ? 16 : kBytes) / int(sizeof(E));
    // Rows half a word off: pairs from the second element on lie on boundaries.
    static constexpr bool kShifted = MODE == kAnywhere && sizeof(E) <= 2;
    using Pair = typename std::conditional<sizeof(E) == 1, uint16_t, uint32_t>::type;
    Vec<E, kPer> part[V / kPer];

    __device__ __forceinline__ void load(const E* p, int count) {
        if constexpr (MODE == kAligned) {
#pragma unroll
            for (int i = 0; i < V / kPer; ++i) part[i] = reinterpret_cast<const Vec<E, kPer>*>(p)[i];
        } else {
            const uintptr_t at = reinterpret_cast<uintptr_t>(p);
            if (count == V && (at % 4 == 0 || (MODE == kWords && sizeof(E) > 1))) {
                copy_in<uint32_t, kBytes>(part, p);
            } else if (count == V && sizeof(E) == 1 && (at % 2 == 0 || MODE == kWords)) {
                copy_in<uint16_t, kBytes>(part, p);
            } else if (count == V && kShifted) {
                // One element, pairs of elements, one element.
                E* e = reinterpret_cast<E*>(part);
                e[0] = p[0];
#pragma unroll
                for (int j = 1; j + 2 < V; j += 2) {
                    const Pair two = *reinterpret_cast<const Pair*>(p + j);
                    memcpy(&e[j], &two, sizeof(Pair));
                }
                e[V - 1] = p[V - 1];
            } else {
                E* e = reinterpret_cast<E*>(part);
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    if (j < count) e[j] = p[j];
                    else memset(&e[j], 0, sizeof(E));
                }
            }
        }
    }
    __device__ __forceinline__ void store(E* p, int count) const {
        if constexpr (MODE == kAligned) {
#pragma unroll
            for (int i = 0; i < V / kPer; ++i) reinterpret_cast<Vec<E, kPer>*>(p)[i] = part[i];
        } else {
            const uintptr_t at = reinterpret_cast<uintptr_t>(p);
            if (count == V && (at % 4 == 0 || (MODE == kWords && sizeof(E) > 1))) {
                copy_in<uint32_t, kBytes>(p, part);
            } else if (count == V && sizeof(E) == 1 && (at % 2 == 0 || MODE == kWords)) {
                copy_in<uint16_t, kBytes>(p, part);
            } else if (count == V && kShifted) {
                const E* e = reinterpret_cast<const E*>(part);
                p[0] = e[0];
#pragma unroll
                for (int j = 1; j + 2 < V; j += 2) {
                    Pair two;
                    memcpy(&two, &e[j], sizeof(Pair));
                    *reinterpret_cast<Pair*>(p + j) = two;
                }
                p[V - 1] = e[V - 1];
            } else {
                const E* e = reinterpret_cast<const E*>(part);
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    if (j < count) p[j] = e[j];
                }
            }
        }
    }
    __device__ __forceinline__ void get(float (&f)[V]) const {
#pragma unroll
        for (int i = 0; i < V / kPer; ++i) {
            float t[kPer];
            unpack_vec(part[i], t);
#pragma unroll
            for (int j = 0; j < kPer; ++j) f[i * kPer + j] = t[j];
        }
    }
    __device__ __forceinline__ void set(const float (&f)[V]) {
#pragma unroll
        for (int i = 0; i < V / kPer; ++i) {
            float t[kPer];
#pragma unroll
            for (int j = 0; j < kPer; ++j) t[j] = f[i * kPer + j];
            pack_vec(t, part[i]);
        }
    }
};

// A checkpoint's int8 values, V of them.
template <int V, int MODE>
struct ByteChunk : Chunk<int8_t, V, MODE> {
    __device__ __forceinline__ const Vec<int8_t, V>& all() const {
        static_assert(V <= 16, "one part");
        return this->part[0];
    }
};

// Rows of 32-element blocks: unit u is block u % nb of row u / nb, and 32 / V
// neighbouring lanes share it.
struct Units {
    int64_t count;
    int64_t nb;
    FastDiv div;
    __device__ __forceinline__ void split(int64_t u, int64_t& row, int64_t& blk) const {
        row = count <= 0xffffffffll ? int64_t(div.div(uint32_t(u))) : u / nb;
        blk = u - row * nb;
    }
};

Units make_units(int64_t rows, int64_t n) {
    Units u;
    u.nb = (n + kCkptBlock - 1) / kCkptBlock;
    u.count = rows * u.nb;
    u.div = FastDiv(static_cast<uint32_t>(std::min<int64_t>(u.nb, 0xffffffffll)));
    return u;
}

// The largest magnitude of a chunk's elements (NaN if one is); 16-bit floats
// are compared two at a time as they lie.
template <typename T, int V, int MODE>
__device__ __forceinline__ float largest(const Chunk<T, V, MODE>& c) {
    using C = Chunk<T, V, MODE>;
    if constexpr (sizeof(T) == 2) {
        using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
        const T2* p = reinterpret_cast<const T2*>(&c.part);
        T2 m = __habs2(p[0]);
#pragma unroll
        for (int j = 1; j < V / 2; ++j) m = __hmax2_nan(m, __habs2(p[j]));
        return max_nan(load_as<float>(m.x), load_as<float>(m.y));
    } else {
        float m = 0.0f;
#pragma unroll
        for (int i = 0; i < V / C::kPer; ++i) {
#pragma unroll
            for (int j = 0; j < C::kPer; ++j) m = max_nan(m, fabsf(c.part[i].v[j]));
        }
        return m;
    }
}

// One block's values and exponent, from V elements in each of its lanes and
// their largest magnitude (zero past the row's end; `count` of them exist).
template <typename T, int V, int MODE>
__device__ __forceinline__ void pack_block(const float (&x)[V], float amax, int count, int lane_in_block,
                                           int8_t* values, uint8_t* exponent) {
#pragma unroll
    for (int o = 1; o < kCkptBlock / V; o <<= 1) amax = max_nan(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    float qmax;
    const int stored = ckpt_exponent<T>(amax, qmax);
    if (count > 0) {
        Chunk<int8_t, V, MODE> q;
        q.part[0] = ckpt_quantise<V>(x, stored, qmax);
        q.store(values, count);
    }
    if (lane_in_block == 0 && exponent != nullptr) *exponent = static_cast<uint8_t>(stored);
}

template <typename T>
struct ForwardParams {
    const T* z;
    int64_t sz_m, sz_p;
    const T* residual;
    int64_t sr_m;
    T* y;
    int64_t sy_m;
    int8_t* values;     // [rows, parts, n], contiguous
    uint8_t* exponents; // [rows, parts, nb], contiguous
    int64_t n;
    int act;
    Units units;
};

// y = act(z0) [* z1] [+ residual] and the checkpoint of z0 [and z1]; a thread
// holds V elements of a unit, kU units at a time so that their loads are in
// flight together.  PACK: the checkpoint alone.
template <typename T, int V, bool GATED, int MODE, bool PACK>
__global__ void __launch_bounds__(kThreads, 4) ffn_forward_kernel(const ForwardParams<T> p) {
    pdl_entry();
    constexpr int kLanes = kCkptBlock / V;
    constexpr int kU = (sizeof(T) == 4 || GATED ? 16 : 32) / V;
    constexpr int kParts = GATED ? 2 : 1;
    constexpr bool kFast = Narrow<T>::value;
    const int lane = threadIdx.x % kLanes;
    const int64_t per_pass = int64_t(blockDim.x / kLanes);
    const int64_t u0 = int64_t(blockIdx.x) * per_pass * kU + threadIdx.x / kLanes;
    Chunk<T, V, MODE> in[kU][kParts], res[kU];
    int64_t row[kU], blk[kU];
    int count[kU];  // elements of the row in this lane's chunk
#pragma unroll
    for (int i = 0; i < kU; ++i) {
        const int64_t u = u0 + i * per_pass;
        count[i] = 0;
        if (u >= p.units.count) continue;
        p.units.split(u, row[i], blk[i]);
        const int64_t col = blk[i] * kCkptBlock + lane * V;
        count[i] = static_cast<int>(max(int64_t(0), min(int64_t(V), p.n - col)));
        if (count[i] == 0) continue;
#pragma unroll
        for (int q = 0; q < kParts; ++q) in[i][q].load(p.z + row[i] * p.sz_m + q * p.sz_p + col, count[i]);
        if (!PACK && p.residual != nullptr) res[i].load(p.residual + row[i] * p.sr_m + col, count[i]);
    }
#pragma unroll
    for (int i = 0; i < kU; ++i) {
        const bool in_range = u0 + i * per_pass < p.units.count;
        const int64_t r = in_range ? row[i] : 0, b = in_range ? blk[i] : 0;
        const int64_t col = b * kCkptBlock + lane * V;
        float z[kParts][V];
#pragma unroll
        for (int q = 0; q < kParts; ++q) {
            if (count[i] > 0) in[i][q].get(z[q]);
            else {
#pragma unroll
                for (int j = 0; j < V; ++j) z[q][j] = 0.0f;
            }
        }
        if (PACK || p.values != nullptr) {
#pragma unroll
            for (int q = 0; q < kParts; ++q) {
                const int64_t at = r * kParts + q;
                pack_block<T, V, MODE>(z[q], count[i] > 0 ? largest(in[i][q]) : 0.0f, count[i], lane, p.values + at * p.n + (count[i] > 0 ? col : 0),
                                          in_range ? p.exponents + at * p.units.nb + b : nullptr);
            }
        }
        if (!PACK && p.y != nullptr && count[i] > 0) {
            act_values<kFast, V>(p.act, z[0]);
            if constexpr (GATED) {
#pragma unroll
                for (int j = 0; j < V; ++j) z[0][j] *= z[1][j];
            }
            if (p.residual != nullptr) {
                float t[V];
                res[i].get(t);
#pragma unroll
                for (int j = 0; j < V; ++j) z[0][j] += t[j];
            }
            Chunk<T, V, MODE> out;
            out.set(z[0]);
            out.store(p.y + r * p.sy_m + col, count[i]);
        }
    }
}

template <typename T>
struct UnpackParams {
    T* y;
    int64_t sy_m;
    const int8_t* values;
    const uint8_t* exponents;
    int64_t n;
    Units units;
};

template <typename T, int V, int MODE>
__global__ void __launch_bounds__(kThreads) checkpoint_unpack_kernel(const UnpackParams<T> p) {
    pdl_entry();
    constexpr int kLanes = kCkptBlock / V;
    constexpr int kU = 32 / V;
    const int lane = threadIdx.x % kLanes;
    const int64_t per_pass = int64_t(blockDim.x / kLanes);
    const int64_t u0 = int64_t(blockIdx.x) * per_pass * kU + threadIdx.x / kLanes;
    ByteChunk<V, MODE> q[kU];
    int stored[kU], count[kU];
    int64_t row[kU], col[kU];
#pragma unroll
    for (int i = 0; i < kU; ++i) {
        const int64_t u = u0 + i * per_pass;
        count[i] = 0;
        if (u >= p.units.count) continue;
        int64_t blk;
        p.units.split(u, row[i], blk);
        col[i] = blk * kCkptBlock + lane * V;
        count[i] = static_cast<int>(max(int64_t(0), min(int64_t(V), p.n - col[i])));
        if (count[i] == 0) continue;
        q[i].load(p.values + row[i] * p.n + col[i], count[i]);
        stored[i] = p.exponents[u];
    }
#pragma unroll
    for (int i = 0; i < kU; ++i) {
        if (count[i] == 0) continue;
        float f[V];
        ckpt_values<V>(q[i].all(), stored[i], f);
        Chunk<T, V, MODE> out;
        out.set(f);
        out.store(p.y + row[i] * p.sy_m + col[i], count[i]);
    }
}

template <typename T>
struct BackwardParams {
    const T* dy;
    int64_t sdy_m;
    const T* z;
    int64_t sz_m, sz_p;
    const int8_t* values;
    const uint8_t* exponents;
    int64_t nb;
    T* dz;
    int64_t sdz_m, sdz_p;
    float* partial;  // [gridDim.y, parts, n] column sums of dz, or null
    int64_t m, n;
    int64_t rows_per_block;
    int act;
    int tx;  // threads along the columns (a power of two)
};

// Rows a thread loads before it computes, and blocks an SM: one or two rows
// with four blocks (64 registers) keep 48 to 64 KB in flight.  fp32 gated rows
// do better with two rows and two blocks (8192 x 2 x 11008: 305 against 351 us).
template <typename T, bool GATED>
__host__ __device__ constexpr int rows_at_once() {
    return GATED ? (sizeof(T) == 4 ? 2 : 1) : (sizeof(T) == 4 ? 1 : 2);
}
template <typename T, bool GATED>
__host__ __device__ constexpr int backward_blocks() {
    return GATED && sizeof(T) == 4 ? 2 : 4;
}

// dz0 = dy [* z1] act'(z0) [, dz1 = dy act(z0)] and, for the bias gradient,
// the fp32 sums of dz (before its rounding) over the block's rows.  A thread
// keeps its V columns and walks the rows, so the sums stay in registers; they
// are joined over the block in a fixed order and written as one partial row.
// dz is computed in fp32 and rounded once, to T: the two products want operands
// of T (a 16-bit MMA has nominally six times the rate of three TF32 ones, and
// dz is written once and read twice).  That rounding is half a step of each
// element, as large as the results' own, so dx and dw are off by about sqrt(2)
// times the final rounding alone.  In float16 an element of dz beyond 65504 is
// infinite and one below 6e-5 loses bits, as with separate float16 layers:
// gradients are scaled as for those.
template <typename T, int V, bool GATED, bool SAVED8, int MODE, bool SUMS>
__global__ void __launch_bounds__(kThreads, (backward_blocks<T, GATED>())) ffn_backward_kernel(const BackwardParams<T> p) {
    pdl_entry();
    constexpr int kParts = GATED ? 2 : 1;
    constexpr int kU = rows_at_once<T, GATED>();
    constexpr bool kFast = Narrow<T>::value;
    const int tx = threadIdx.x & (p.tx - 1);
    const int ty = threadIdx.x / p.tx;
    const int ny = kThreads / p.tx;
    const int64_t col = (int64_t(blockIdx.x) * p.tx + tx) * V;
    const int64_t r1 = min(p.m, (int64_t(blockIdx.y) + 1) * p.rows_per_block);
    const int count = static_cast<int>(max(int64_t(0), min(int64_t(V), p.n - col)));
    float acc[kParts][V];
#pragma unroll
    for (int q = 0; q < kParts; ++q) {
#pragma unroll
        for (int j = 0; j < V; ++j) acc[q][j] = 0.0f;
    }
    if (count > 0) {
        for (int64_t r = int64_t(blockIdx.y) * p.rows_per_block + ty; r < r1; r += int64_t(ny) * kU) {
            Chunk<T, V, MODE> dyv[kU], zv[kU][kParts];
            ByteChunk<V, MODE> qv[kU][kParts];
            int ev[kU][kParts];
#pragma unroll
            for (int i = 0; i < kU; ++i) {
                const int64_t row = r + int64_t(i) * ny;
                if (row >= r1) continue;
                dyv[i].load(p.dy + row * p.sdy_m + col, count);
#pragma unroll
                for (int q = 0; q < kParts; ++q) {
                    if constexpr (SAVED8) {
                        const int64_t at = row * kParts + q;
                        qv[i][q].load(p.values + at * p.n + col, count);
                        ev[i][q] = p.exponents[at * p.nb + col / kCkptBlock];
                    } else {
                        zv[i][q].load(p.z + row * p.sz_m + q * p.sz_p + col, count);
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < kU; ++i) {
                const int64_t row = r + int64_t(i) * ny;
                if (row >= r1) continue;
                float dy[V], z[kParts][V], a[V], d[V];
                dyv[i].get(dy);
#pragma unroll
                for (int q = 0; q < kParts; ++q) {
                    if constexpr (SAVED8) {
                        ckpt_values<V>(qv[i][q].all(), ev[i][q], z[q]);
                    } else {
                        zv[i][q].get(z[q]);
                    }
                }
                act_slopes<kFast, V>(p.act, z[0], a, d);
                Chunk<T, V, MODE> out;
                if constexpr (GATED) {
                    mul_to<V>(a, dy);
                    if constexpr (SUMS) add_to<V>(acc[1], a);
                    mul_to<V>(dy, z[1]);
                    out.set(a);
                    out.store(p.dz + row * p.sdz_m + p.sdz_p + col, count);
                }
                mul_to<V>(d, dy);
                if constexpr (SUMS) add_to<V>(acc[0], d);
                out.set(d);
                out.store(p.dz + row * p.sdz_m + col, count);
            }
        }
    }
    if constexpr (!SUMS) return;
    __shared__ float sums[kThreads * V];
#pragma unroll
    for (int q = 0; q < kParts; ++q) {
        __syncthreads();
#pragma unroll
        for (int j = 0; j < V; ++j) sums[j * kThreads + threadIdx.x] = acc[q][j];
        __syncthreads();
        for (int c = threadIdx.x; c < p.tx * V; c += kThreads) {
            const int x = c / V, j = c % V;
            const int64_t at = (int64_t(blockIdx.x) * p.tx + x) * V + j;
            if (at >= p.n) continue;
            float s = 0.0f;
            for (int y = 0; y < ny; ++y) s += sums[j * kThreads + y * p.tx + x];
            p.partial[(int64_t(blockIdx.y) * kParts + q) * p.n + at] = s;
        }
    }
}

// Rows off 16-byte boundaries copied to rows on them, for operands that
// tensor maps or 16-byte loads read: a thread writes 16 bytes, from aligned
// words shifted into place where all of them lie inside the row, element by
// element at the row's ends.  E: 2- or 4-byte elements.
template <typename E>
__global__ void __launch_bounds__(kThreads) align_rows_kernel(E* __restrict__ dst, int64_t dst_pitch,
                                                              const E* __restrict__ src, int64_t src_pitch, int64_t n,
                                                              int64_t chunks, int64_t row_chunks, FastDiv div) {
    pdl_entry();
    constexpr int kPer = 16 / int(sizeof(E));
    constexpr int kU = 4;
    const int64_t first = int64_t(blockIdx.x) * kThreads * kU + threadIdx.x;
#pragma unroll
    for (int u = 0; u < kU; ++u) {
        const int64_t i = first + int64_t(u) * kThreads;
        if (i >= chunks) break;
        const int64_t row = chunks <= 0xffffffffll ? int64_t(div.div(uint32_t(i))) : i / row_chunks;
        const int64_t col = (i - row * row_chunks) * kPer;
        const E* s = src + row * src_pitch + col;
        Vec<E, kPer> out;
        const bool odd = sizeof(E) == 2 && (reinterpret_cast<uintptr_t>(s) & 2) != 0;
        if (col + kPer + 1 <= n && (!odd || col > 0)) {
            const uint32_t* w = reinterpret_cast<const uint32_t*>(odd ? s - 1 : s);
            uint32_t v[5];
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = w[j];
            v[4] = odd ? w[4] : 0;
            uint32_t* o = reinterpret_cast<uint32_t*>(&out);
#pragma unroll
            for (int j = 0; j < 4; ++j) o[j] = odd ? __funnelshift_r(v[j], v[j + 1], 16) : v[j];
        } else {
#pragma unroll
            for (int j = 0; j < kPer; ++j) out.v[j] = col + j < n ? s[j] : E(0);
        }
        *reinterpret_cast<Vec<E, kPer>*>(dst + row * dst_pitch + col) = out;
    }
}

// out[c] = sum of partial[g][c] over the groups, in order: 32 columns a block,
// its warps over the groups.
template <typename T>
__global__ void __launch_bounds__(kThreads) column_sum_kernel(const float* __restrict__ partial, T* __restrict__ out,
                                                              int groups, int64_t n) {
    pdl_entry();
    constexpr int kRows = kThreads / 32;
    __shared__ float sums[kRows][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t c = int64_t(blockIdx.x) * 32 + lane;
    float s = 0.0f;
    if (c < n) {
#pragma unroll 4
        for (int g = warp; g < groups; g += kRows) s += partial[int64_t(g) * n + c];
    }
    sums[warp][lane] = s;
    __syncthreads();
    if (warp == 0 && c < n) {
        float total = 0.0f;
#pragma unroll
        for (int r = 0; r < kRows; ++r) total += sums[r][lane];
        out[c] = store_as<T>(total);
    }
}

void require_act(int act, const char* what) {
    TPB_CHECK(act >= TPB_ACT_NONE && act <= TPB_ACT_SILU, "%s: unknown activation %d", what, act);
}

// Rows on 4-byte boundaries (checkpoint values of even rows: 2-byte ones).
bool rows4(const void* p, int64_t pitch, size_t es) {
    return p == nullptr || (reinterpret_cast<uintptr_t>(p) % 4 == 0 && (pitch * int64_t(es)) % 4 == 0);
}
// 16-byte vectors along n are possible for an operand of `es`-byte elements.
bool rows16(const void* p, int64_t pitch, size_t es) {
    return p == nullptr || (aligned16(p) && (pitch * int64_t(es)) % 16 == 0);
}

unsigned unit_blocks(const Units& u, int lanes, int unroll) {
    const int64_t blocks = (u.count + int64_t(kThreads / lanes) * unroll - 1) / (int64_t(kThreads / lanes) * unroll);
    TPB_CHECK(blocks < (int64_t(1) << 31), "checkpoint: too many elements for one call");
    return static_cast<unsigned>(blocks);
}

template <typename T, bool GATED>
void launch_forward(ForwardParams<T>& p, cudaStream_t s) {
    constexpr int per = sizeof(T) == 4 || GATED ? 16 : 32;  // elements a thread holds
    constexpr size_t es = sizeof(T);
    const bool aligned = p.n % 8 == 0 && rows16(p.z, p.sz_m, es) && rows16(p.z, p.sz_p, es) &&
                         rows16(p.residual, p.sr_m, es) && rows16(p.y, p.sy_m, es) &&
                         reinterpret_cast<uintptr_t>(p.values) % 8 == 0;
    const bool words = p.n % 2 == 0 && rows4(p.z, p.sz_m, es) && rows4(p.z, p.sz_p, es) &&
                       rows4(p.residual, p.sr_m, es) && rows4(p.y, p.sy_m, es) &&
                       reinterpret_cast<uintptr_t>(p.values) % 2 == 0;
    const auto go = [&](auto kernel, int v) {
        launch_pdl(kernel, unit_blocks(p.units, kCkptBlock / v, per / v), kThreads, 0, s, p);
    };
    if (!GATED && p.y == nullptr) {
        if (aligned && p.n % 16 == 0 && aligned16(p.values)) go(ffn_forward_kernel<T, 16, false, kAligned, true>, 16);
        else if (aligned) go(ffn_forward_kernel<T, 8, false, kAligned, true>, 8);
        else if (words) go(ffn_forward_kernel<T, 8, false, kWords, true>, 8);
        else go(ffn_forward_kernel<T, 8, false, kAnywhere, true>, 8);
    } else if (aligned) {
        go(ffn_forward_kernel<T, 8, GATED, kAligned, false>, 8);
    } else {
        go(ffn_forward_kernel<T, 8, GATED, kAnywhere, false>, 8);
    }
    check_launch("ffn_forward");
}

template <typename T, bool GATED, bool SAVED8, int MODE>
void launch_backward(BackwardParams<T>& p, int64_t partial_rows, int dev, cudaStream_t s) {
    constexpr int V = 8;
    // Threads along the columns: enough for one row, at most the block, or two
    // warps where the rows' split is free (a warp covers 512 bytes of a row).
    const int widest = p.partial != nullptr ? kThreads : 64;
    int tx = 1;
    while (tx < widest && int64_t(tx) * V < p.n) tx <<= 1;
    // Where the partial sums fix the rows' split, narrower blocks until there
    // are sixteen for every SM.
    while (p.partial != nullptr && tx > 32 &&
           (p.n + int64_t(tx) * V - 1) / (int64_t(tx) * V) * partial_rows < int64_t(num_sms(dev)) * 16) {
        tx >>= 1;
    }
    p.tx = tx;
    const int64_t gx = (p.n + int64_t(tx) * V - 1) / (int64_t(tx) * V);
    int64_t gy;
    if (p.partial != nullptr) {
        gy = partial_rows;
    } else {
        // About 32 blocks an SM, and no more than one pass of rows needs.
        const int64_t pass = int64_t(kThreads / tx) * rows_at_once<T, GATED>();
        gy = std::max<int64_t>(1, std::min<int64_t>((p.m + pass - 1) / pass, (int64_t(num_sms(dev)) * 32 + gx - 1) / gx));
        gy = std::min<int64_t>(gy, 65535);
    }
    p.rows_per_block = (p.m + gy - 1) / gy;
    TPB_CHECK(gx < (int64_t(1) << 31), "feed-forward gradients: too many columns");
    const dim3 grid{unsigned(gx), unsigned(gy), 1};
    if (p.partial != nullptr) launch_pdl(ffn_backward_kernel<T, V, GATED, SAVED8, MODE, true>, grid, kThreads, 0, s, p);
    else launch_pdl(ffn_backward_kernel<T, V, GATED, SAVED8, MODE, false>, grid, kThreads, 0, s, p);
    check_launch("ffn_backward");
}

template <typename T, bool GATED>
void dispatch_backward(BackwardParams<T>& p, int64_t partial_rows, int dev, cudaStream_t s) {
    constexpr size_t es = sizeof(T);
    const bool aligned = p.n % 8 == 0 && rows16(p.dy, p.sdy_m, es) && rows16(p.z, p.sz_m, es) &&
                         rows16(p.z, p.sz_p, es) && rows16(p.dz, p.sdz_m, es) && rows16(p.dz, p.sdz_p, es) &&
                         reinterpret_cast<uintptr_t>(p.values) % 8 == 0;
    const bool words = p.n % 2 == 0 && rows4(p.dy, p.sdy_m, es) && rows4(p.z, p.sz_m, es) && rows4(p.z, p.sz_p, es) &&
                       rows4(p.dz, p.sdz_m, es) && rows4(p.dz, p.sdz_p, es) &&
                       reinterpret_cast<uintptr_t>(p.values) % 2 == 0;
    if (p.values != nullptr) {
        if (aligned) launch_backward<T, GATED, true, kAligned>(p, partial_rows, dev, s);
        else if (words) launch_backward<T, GATED, true, kWords>(p, partial_rows, dev, s);
        else launch_backward<T, GATED, true, kAnywhere>(p, partial_rows, dev, s);
    } else {
        if (aligned) launch_backward<T, GATED, false, kAligned>(p, partial_rows, dev, s);
        else if (words) launch_backward<T, GATED, false, kWords>(p, partial_rows, dev, s);
        else launch_backward<T, GATED, false, kAnywhere>(p, partial_rows, dev, s);
    }
}

#define TPB_DISPATCH_FFN(dtype, what, ...)                                        \
    switch (dtype) {                                                              \
        case TPB_F16: { using scalar_t = __half; __VA_ARGS__; break; }            \
        case TPB_F32: { using scalar_t = float; __VA_ARGS__; break; }             \
        case TPB_BF16: { using scalar_t = __nv_bfloat16; __VA_ARGS__; break; }    \
        default: TPB_CHECK(false, "%s: unsupported dtype %s", what, dtype_name(dtype)); \
    }

template <typename T>
void launch_unpack(const UnpackParams<T>& p, cudaStream_t s) {
    const bool aligned = p.n % 8 == 0 && rows16(p.y, p.sy_m, sizeof(T)) && reinterpret_cast<uintptr_t>(p.values) % 8 == 0;
    const bool words = p.n % 2 == 0 && rows4(p.y, p.sy_m, sizeof(T)) && reinterpret_cast<uintptr_t>(p.values) % 2 == 0;
    const auto go = [&](auto kernel, int v) {
        launch_pdl(kernel, unit_blocks(p.units, kCkptBlock / v, 32 / v), kThreads, 0, s, p);
    };
    if (aligned && p.n % 16 == 0 && aligned16(p.values)) go(checkpoint_unpack_kernel<T, 16, kAligned>, 16);
    else if (aligned) go(checkpoint_unpack_kernel<T, 8, kAligned>, 8);
    else if (words) go(checkpoint_unpack_kernel<T, 8, kWords>, 8);
    else go(checkpoint_unpack_kernel<T, 8, kAnywhere>, 8);
    check_launch("checkpoint_unpack");
}

void require_layer(int dtype, int act, int parts, int64_t m, int64_t n, int64_t k, const char* what) {
    TPB_CHECK(dtype == TPB_BF16 || dtype == TPB_F16 || dtype == TPB_F32,
              "%s: expected bfloat16, float16 or float32, got %s", what, dtype_name(dtype));
    require_act(act, what);
    TPB_CHECK(parts == 1 || parts == 2, "%s: one part, or a gate and an up part; got %d", what, parts);
    const int64_t limit = int64_t(1) << 30;
    TPB_CHECK(m >= 0 && n >= 0 && k >= 0 && m < limit && n < limit && k < limit,
              "%s: sizes %lld, %lld, %lld out of range", what, (long long)m, (long long)n, (long long)k);
    // The products count rows and columns in 32 bits, a tile of 256 past the end
    // included; the gradients' contract over, and have rows for, both parts.
    TPB_CHECK(parts * n <= INT32_MAX - 256, "%s: %lld rows of the weight are out of range", what, (long long)(parts * n));
}

// A checkpoint entry point: its checks, then body(T{}, device, stream).
template <typename F>
int checkpoint_call(const tpb_checkpoint* a, const char* what, bool reads, bool writes, void* stream, F&& body) {
    return guarded([&] {
        TPB_CHECK(a != nullptr, "%s: null arguments", what);
        require_layer(a->dtype, a->act, 1, 0, 0, 0, what);
        TPB_CHECK(a->rows >= 0 && a->n >= 0 && a->n < (int64_t(1) << 40) && a->rows < (int64_t(1) << 40),
                  "%s: sizes %lld, %lld out of range", what, (long long)a->rows, (long long)a->n);
        if (a->rows == 0 || a->n == 0) return;
        TPB_CHECK(a->values != nullptr && a->exponents != nullptr && (!reads || a->x != nullptr) &&
                      (!writes || a->y != nullptr),
                  "%s: null operand", what);
        const int dev = device_of(a->values);
        DeviceGuard guard(dev);
        cudaStream_t s = resolve_stream(stream, dev);
        TPB_DISPATCH_FFN(a->dtype, what, body(scalar_t(0.0f), dev, s));
    });
}

// An operand of a product, copied into `work` (rows of n elements rounded up
// to 128 bytes) where its rows start off 16-byte boundaries.  Rows that start
// inside a 32-byte sector cost the tensor-map loads a fifth sector for every
// four (dx of 1001 x 5460 -> 1000: 37 us on 16-byte boundaries).
struct Aligned {
    const void* data;
    int64_t pitch;
};
Aligned align_rows(const void* src, int64_t pitch, int64_t rows, int64_t n, int es, void* work, const char* what,
                   cudaStream_t s) {
    const int64_t per = 16 / es, line = 128 / es, aligned = (n + line - 1) / line * line;
    if (aligned16(src) && pitch > 0 && pitch % per == 0) return {src, pitch};
    if (aligned16(src) && rows == 1) return {src, aligned};  // there is no second row
    TPB_CHECK(work != nullptr && aligned16(work), "%s: rows off 16-byte boundaries need an aligned workspace", what);
    const int64_t row_chunks = aligned / per, chunks = rows * row_chunks;
    const int64_t blocks = (chunks + kThreads * 4 - 1) / (kThreads * 4);
    TPB_CHECK(blocks < (int64_t(1) << 31), "%s: too many elements", what);
    const FastDiv div(static_cast<uint32_t>(std::min<int64_t>(row_chunks, 0xffffffffll)));
    if (es == 2) {
        launch_pdl(align_rows_kernel<uint16_t>, unsigned(blocks), kThreads, 0, s, static_cast<uint16_t*>(work), aligned,
                   static_cast<const uint16_t*>(src), pitch, n, chunks, row_chunks, div);
    } else {
        launch_pdl(align_rows_kernel<uint32_t>, unsigned(blocks), kThreads, 0, s, static_cast<uint32_t*>(work), aligned,
                   static_cast<const uint32_t*>(src), pitch, n, chunks, row_chunks, div);
    }
    check_launch("align_rows");
    return {work, aligned};
}

// x w^T without an epilogue, for the plain products' kernels: gradients with a
// dimension of 2^30 or more, which the feed-forward products leave.
GemmProblem plain_product(const FfnProblem& q) {
    GemmProblem g{};
    g.dtype = q.dtype;
    g.M = q.M;
    g.N = q.N;
    g.K = q.K;
    g.batch = 1;
    g.a = q.x;
    g.sa_m = q.sx_m;
    g.sa_k = q.sx_k;
    g.b = q.w;
    g.sb_k = q.sw_k;
    g.sb_n = q.sw_n;
    g.c = q.y;
    g.sc_m = q.sy_m;
    g.alpha = 1.0;
    g.flags = q.flags;
    return g;
}

void run_gemm(const GemmProblem& p, int dev, cudaStream_t s) {
    if (!gemm_tc(p, dev, s)) gemm_simt(p, dev, s);
}

}  // namespace
}  // namespace tpb

using namespace tpb;

extern "C" {

int tp_b200_checkpoint_pack(const tpb_checkpoint* a, void* stream) {
    return checkpoint_call(a, "checkpoint_pack", true, false, stream, [&](auto zero, int, cudaStream_t s) {
        using T = decltype(zero);
        ForwardParams<T> p{};
        p.z = static_cast<const T*>(a->x);
        p.sz_m = a->x_stride;
        p.values = static_cast<int8_t*>(a->values);
        p.exponents = static_cast<uint8_t*>(a->exponents);
        p.n = a->n;
        p.units = make_units(a->rows, a->n);
        launch_forward<T, false>(p, s);
    });
}

int tp_b200_checkpoint_unpack(const tpb_checkpoint* a, void* stream) {
    return checkpoint_call(a, "checkpoint_unpack", false, true, stream, [&](auto zero, int, cudaStream_t s) {
        using T = decltype(zero);
        UnpackParams<T> p{};
        p.y = static_cast<T*>(a->y);
        p.sy_m = a->y_stride;
        p.values = static_cast<const int8_t*>(a->values);
        p.exponents = static_cast<const uint8_t*>(a->exponents);
        p.n = a->n;
        p.units = make_units(a->rows, a->n);
        launch_unpack<T>(p, s);
    });
}

int tp_b200_checkpoint_backward(const tpb_checkpoint* a, void* stream) {
    return checkpoint_call(a, "checkpoint_backward", true, true, stream, [&](auto zero, int dev, cudaStream_t s) {
        using T = decltype(zero);
        BackwardParams<T> p{};
        p.dy = static_cast<const T*>(a->x);
        p.sdy_m = a->x_stride;
        p.values = static_cast<const int8_t*>(a->values);
        p.exponents = static_cast<const uint8_t*>(a->exponents);
        p.nb = (a->n + kCkptBlock - 1) / kCkptBlock;
        p.dz = static_cast<T*>(a->y);
        p.sdz_m = a->y_stride;
        p.m = a->rows;
        p.n = a->n;
        p.act = a->act;
        dispatch_backward<T, false>(p, 0, dev, s);
    });
}

int tp_b200_layer_forward(const tpb_layer* a, void* stream) {
    return guarded([&] {
        TPB_CHECK(a != nullptr, "layer_forward: null arguments");
        require_layer(a->dtype, a->act, a->parts, a->m, a->n, a->k, "layer_forward");
        const int es = int(dtype_size(a->dtype));
        const int64_t m = a->m, n = a->n, k = a->k;
        TPB_CHECK((a->values == nullptr) == (a->exponents == nullptr), "layer_forward: a checkpoint is values and exponents");
        if (m == 0 || n == 0) return;
        const bool fused = k > 0;
        TPB_CHECK(a->y != nullptr && (k == 0 || (a->x != nullptr && a->w != nullptr)), "layer_forward: null operand");
        TPB_CHECK(a->parts == 1 || a->residual == nullptr, "layer_forward: the gated block takes no residual");
        TPB_CHECK(fused || a->saved != nullptr, "layer_forward: a layer without input features needs `saved`");
        const int dev = device_of(a->y);
        DeviceGuard guard(dev);
        cudaStream_t s = resolve_stream(stream, dev);
        if (fused) {
            Aligned x{a->x, a->x_stride}, w{a->w, a->w_stride};
            // float32 operands are read with plain loads; only products that
            // asked for the copies get them.
            if (a->dtype != TPB_F32 || a->x_work != nullptr) x = align_rows(x.data, x.pitch, m, k, es, a->x_work, "layer_forward", s);
            if (a->dtype != TPB_F32 || a->w_work != nullptr) {
                w = align_rows(w.data, w.pitch, a->parts * n, k, es, a->w_work, "layer_forward", s);
            }
            FfnProblem q{};
            q.dtype = a->dtype;
            q.M = m;
            q.N = n;
            q.K = k;
            q.parts = a->parts;
            q.x = x.data;
            q.sx_m = x.pitch;
            q.sx_k = 1;
            q.w = w.data;
            q.sw_n = w.pitch;
            q.sw_k = 1;
            q.flags = a->flags;
            q.y = a->y;
            q.sy_m = a->y_stride;
            q.bias = a->bias;
            q.residual = a->residual;
            q.sres_m = a->residual_stride;
            q.saved = a->saved;
            q.values = static_cast<int8_t*>(a->values);
            q.exponents = static_cast<uint8_t*>(a->exponents);
            q.act = a->act;
            if (a->dtype == TPB_F32) gemm_f32(q, dev, s);
            else TPB_CHECK(gemm_ffn(q, dev, s), "layer_forward: operands do not fit the tensor maps");
            return;
        }
        // No input features: the bias is the pre-activation.
        GemmProblem g{};
        g.dtype = a->dtype;
        g.M = m;
        g.N = a->parts * n;
        g.batch = 1;
        g.a = g.b = a->saved;  // not read
        g.c = a->saved;
        g.sc_m = a->parts * n;
        if (a->bias != nullptr) {
            g.cin = a->bias;
            g.sci_n = 1;
            g.beta = 1.0;
        }
        gemm_simt(g, dev, s);
        TPB_DISPATCH_FFN(a->dtype, "layer_forward", {
            ForwardParams<scalar_t> p{};
            p.z = static_cast<const scalar_t*>(a->saved);
            p.sz_m = a->parts * n;
            p.sz_p = n;
            p.residual = static_cast<const scalar_t*>(a->residual);
            p.sr_m = a->residual_stride;
            p.y = static_cast<scalar_t*>(a->y);
            p.sy_m = a->y_stride;
            p.values = static_cast<int8_t*>(a->values);
            p.exponents = static_cast<uint8_t*>(a->exponents);
            p.n = n;
            p.act = a->act;
            p.units = make_units(m, n);
            if (a->parts == 2) launch_forward<scalar_t, true>(p, s);
            else launch_forward<scalar_t, false>(p, s);
        });
    });
}

int tp_b200_layer_backward(const tpb_layer_grad* a, void* stream) {
    return guarded([&] {
        TPB_CHECK(a != nullptr, "layer_backward: null arguments");
        require_layer(a->dtype, a->act, a->parts, a->m, a->n, a->k, "layer_backward");
        const int es = int(dtype_size(a->dtype));
        const int64_t m = a->m, n = a->n, k = a->k, wide = a->parts * n;
        TPB_CHECK((a->values == nullptr) == (a->exponents == nullptr), "layer_backward: a checkpoint is values and exponents");
        TPB_CHECK(a->saved == nullptr || a->values == nullptr, "layer_backward: the pre-activations are given in one form");
        TPB_CHECK(a->db == nullptr || (a->partial != nullptr && a->groups >= 1 && a->groups <= 65535),
                  "layer_backward: db needs a workspace of 1 to 65535 groups");
        if (m == 0 || n == 0) {
            // Nothing was summed: the gradients are zero.
            const void* any = a->dw != nullptr ? a->dw : a->db != nullptr ? a->db : a->dx;
            if (any == nullptr) return;
            const int dev = device_of(any);
            DeviceGuard guard(dev);
            cudaStream_t s = resolve_stream(stream, dev);
            if (a->dx != nullptr && m * k > 0) TPB_CUDA(cudaMemsetAsync(a->dx, 0, size_t(m * k) * es, s));
            if (a->dw != nullptr && wide * k > 0) TPB_CUDA(cudaMemsetAsync(a->dw, 0, size_t(wide * k) * es, s));
            if (a->db != nullptr && wide > 0) TPB_CUDA(cudaMemsetAsync(a->db, 0, size_t(wide) * es, s));
            return;
        }
        const bool linear = a->parts == 1 && a->act == TPB_ACT_NONE;  // dz = dy, whatever z is
        TPB_CHECK(a->dy != nullptr && a->dz != nullptr && (linear || a->saved != nullptr || a->values != nullptr),
                  "layer_backward: null operand");
        TPB_CHECK(a->dz_stride >= wide, "layer_backward: the workspace's rows hold %lld elements, not %lld",
                  (long long)a->dz_stride, (long long)wide);
        TPB_CHECK(k == 0 || ((a->dx == nullptr || a->w != nullptr) && (a->dw == nullptr || a->x != nullptr)),
                  "layer_backward: null operand");
        const int dev = device_of(a->dz);
        DeviceGuard guard(dev);
        cudaStream_t s = resolve_stream(stream, dev);
        const void* dz = a->dz;
        int64_t dz_stride = a->dz_stride;
        if (linear && a->db == nullptr && (a->dtype == TPB_F32 || (rows16(a->dy, a->dy_stride, es) && a->dy_stride > 0))) {
            dz = a->dy;  // as it lies
            dz_stride = a->dy_stride;
        } else TPB_DISPATCH_FFN(a->dtype, "layer_backward", {
            BackwardParams<scalar_t> p{};
            p.dy = static_cast<const scalar_t*>(a->dy);
            p.sdy_m = a->dy_stride;
            if (linear) {  // any readable rows
                p.z = p.dy;
                p.sz_m = p.sdy_m;
            } else {
                p.z = static_cast<const scalar_t*>(a->saved);
                p.sz_m = wide;
                p.sz_p = n;
                p.values = static_cast<const int8_t*>(a->values);
                p.exponents = static_cast<const uint8_t*>(a->exponents);
            }
            p.nb = (n + kCkptBlock - 1) / kCkptBlock;
            p.dz = static_cast<scalar_t*>(a->dz);
            p.sdz_m = a->dz_stride;
            p.sdz_p = n;
            p.partial = a->db != nullptr ? a->partial : nullptr;
            p.m = m;
            p.n = n;
            p.act = a->act;
            if (a->parts == 2) dispatch_backward<scalar_t, true>(p, a->groups, dev, s);
            else dispatch_backward<scalar_t, false>(p, a->groups, dev, s);
        });
        if (a->db != nullptr) {
            const unsigned grid = static_cast<unsigned>((wide + 31) / 32);
            TPB_DISPATCH_FFN(a->dtype, "layer_backward", {
                launch_pdl(column_sum_kernel<scalar_t>, grid, kThreads, 0, s, static_cast<const float*>(a->partial),
                           static_cast<scalar_t*>(a->db), static_cast<int>(a->groups), wide);
            });
            check_launch("column_sum");
        }
        if (k == 0) return;
        Aligned x{a->x, a->x_stride}, w{a->w, a->w_stride};
        if (a->dw != nullptr && (a->dtype != TPB_F32 || a->x_work != nullptr)) {
            x = align_rows(x.data, x.pitch, m, k, es, a->x_work, "layer_backward", s);
        }
        if (a->dx != nullptr && (a->dtype != TPB_F32 || a->w_work != nullptr)) {
            w = align_rows(w.data, w.pitch, wide, k, es, a->w_work, "layer_backward", s);
        }
        FfnProblem q{};
        q.dtype = a->dtype;
        q.parts = 1;
        q.flags = a->flags;
        if (a->dx != nullptr) {
            // dx = dz w, the weight read in place.
            q.M = m;
            q.N = k;
            q.K = wide;
            q.x = dz;
            q.sx_m = dz_stride;
            q.sx_k = 1;
            q.w = w.data;
            q.sw_n = 1;
            q.sw_k = w.pitch;
            q.y = a->dx;
            q.sy_m = k;
            if (a->dtype == TPB_F32) gemm_f32(q, dev, s);
            else if (!gemm_ffn(q, dev, s)) run_gemm(plain_product(q), dev, s);
        }
        if (a->dw != nullptr) {
            // dw = dz^T x: its rows are dz's columns, its columns x's.
            q.M = wide;
            q.N = k;
            q.K = m;
            q.x = dz;
            q.sx_m = 1;
            q.sx_k = dz_stride;
            q.w = x.data;
            q.sw_n = 1;
            q.sw_k = x.pitch;
            q.y = a->dw;
            q.sy_m = k;
            if (a->dtype == TPB_F32) gemm_f32(q, dev, s);
            else if (!gemm_ffn(q, dev, s)) run_gemm(plain_product(q), dev, s);
        }
    });
}

}  // extern "C"
