// The linear layer with its epilogue, and its backward products.
//
//   y = act(x W^T + bias) + residual
//   dz = dy act'(z);  dx = dz W;  dW = dz^T x;  dbias = sum over rows of dz
//
// Sums are held in fp32 by the matrix cores; z, y, dz and the gradients are rounded once, to
// the tensors' dtype, as they are stored.  z is stored for the backward pass: dz is formed
// from its rounded values, which moves act' by at most one rounding of its argument.
#include "hbt_matmul.hpp"

namespace hbt {
namespace mm {
namespace {

// ---- activations ---------------------------------------------------------------------
// 1 / (1 + exp(-t)).  2-byte results take the hardware exponential and reciprocal (about one
// fp32 ulp each, far below their rounding); fp32 results the accurate functions.
template <int D>
__device__ __forceinline__ float sigmoid(float t) {
    if constexpr (D == HBT_DTYPE_F32) return 1.0f / (1.0f + expf(-t));
    else return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(t * -1.44269504f));
}
constexpr float kGeluC = 0.79788456f;  // sqrt(2 / pi)
constexpr float kGeluA = 0.044715f;

template <int D>
__device__ __forceinline__ float activate(float z, int act) {
    switch (act) {
        case HBT_ACT_RELU: return z < 0.0f ? 0.0f : z;  // a NaN stays one
        case HBT_ACT_GELU: return 0.5f * z * (1.0f + erff(z * 0.70710678f));
        // (1 + tanh(u)) / 2 = sigmoid(2 u)
        case HBT_ACT_GELU_TANH: return z * sigmoid<D>(2.0f * kGeluC * (z + kGeluA * z * z * z));
        case HBT_ACT_SILU: return z * sigmoid<D>(z);
        default: return z;
    }
}
// act'(z) of a stored z.  A z past its dtype's range is stored as an infinity, whose products
// with the zeros around it would be NaN; the slopes have reached 0 and 1 long before kFar, which
// stands in for everything past it (a NaN stays one), and whose square and cube stay finite.
constexpr float kFar = 1e4f;
template <int D>
__device__ __forceinline__ float slope(float z, int act) {
    z = z > kFar ? kFar : (z < -kFar ? -kFar : z);
    switch (act) {
        case HBT_ACT_RELU: return z > 0.0f ? 1.0f : (z <= 0.0f ? 0.0f : z);
        case HBT_ACT_GELU:
            return 0.5f * (1.0f + erff(z * 0.70710678f)) + z * expf(-0.5f * z * z) * 0.39894228f;
        case HBT_ACT_GELU_TANH: {
            const float s = sigmoid<D>(2.0f * kGeluC * (z + kGeluA * z * z * z));
            return s + z * s * (1.0f - s) * 2.0f * kGeluC * (1.0f + 3.0f * kGeluA * z * z);
        }
        case HBT_ACT_SILU: {
            const float s = sigmoid<D>(z);
            return s * (1.0f + z * (1.0f - s));
        }
        default: return 1.0f;
    }
}

// ---- the product ---------------------------------------------------------------------
struct ProductArgs {
    const void* a;
    const void* b;
    const void* bias;
    const void* residual;
    void* y;
    void* z;
    float* partial;  // [splits][m][ldp], when the sum over k is split
    int64_t lda, ldb, ldr, ldy, ldz, ldp, m, n, k, k_split;
    int tiles_m, tiles_n, act;
};

// What finishes results: bias, activation, residual, each store rounded once.  Offsets from a
// tile's first element (m0, n0) fit 32 bits.
template <int D>
struct TileEpilogue {
    const char* bias;
    const char* from;
    char* y;
    char* z;
    int ldr, ldy, ldz, act;

    __device__ __forceinline__ TileEpilogue(const ProductArgs& p, int64_t m0, int64_t n0) {
        constexpr int B = elem_bytes<D>();
        bias = p.bias == nullptr ? nullptr : static_cast<const char*>(p.bias) + n0 * B;
        from = p.residual == nullptr ? nullptr : static_cast<const char*>(p.residual) + (m0 * p.ldr + n0) * B;
        y = static_cast<char*>(p.y) + (m0 * p.ldy + n0) * B;
        z = p.z == nullptr ? nullptr : static_cast<char*>(p.z) + (m0 * p.ldz + n0) * B;
        ldr = static_cast<int>(p.ldr), ldy = static_cast<int>(p.ldy), ldz = static_cast<int>(p.ldz), act = p.act;
    }
    // `have`: results left in the row from column j, of which four are taken.
    __device__ __forceinline__ f32x4 residual(int i, int j, int have) const {
        return from == nullptr ? f32x4{0.f, 0.f, 0.f, 0.f} : load_row<D>(from, i * ldr + j, have);
    }
    __device__ __forceinline__ void store(int i, int j, int have, f32x4 v, f32x4 residual) const {
        if (bias != nullptr) v += load_row<D>(bias, j, have);
        if (z != nullptr) store_row<D>(z, i * ldz + j, have, v);
        if (act != HBT_ACT_NONE) {
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = activate<D>(v[e], act);
        }
        if (from != nullptr) v += residual;
        store_row<D>(y, i * ldy + j, have, v);
    }
};

template <int D, bool kA, bool kB, class T, bool kAsync>
__global__ __launch_bounds__(T::kThreads, 2) void product_kernel(ProductArgs p) {
    extern __shared__ __align__(16) char lds[];
    const int t = xcd_tile(blockIdx.x, gridDim.x);
    int tm, tn;
    band_order<8>(t, p.tiles_m, p.tiles_n, tm, tn);
    const int64_t m0 = int64_t(tm) * T::BM, n0 = int64_t(tn) * T::BN;
    const int64_t k0 = blockIdx.y * p.k_split, k1 = min(p.k, k0 + p.k_split);
    f32x4 acc[T::TM][T::TN];
    tile_product<D, kA, kB, T, kAsync>(p.a, p.lda, m0, p.m, p.b, p.ldb, n0, p.n, k0, k1, lds, acc);
    const int rows = static_cast<int>(min<int64_t>(p.m - m0, T::BM)), cols = static_cast<int>(min<int64_t>(p.n - n0, T::BN));
    const TileEpilogue<D> tile(p, m0, n0);
    float* partial = p.partial == nullptr ? nullptr : p.partial + (blockIdx.y * p.m + m0) * p.ldp + n0;
    const int ldp = static_cast<int>(p.ldp);
    finish_tile<T, kAsync, 2>(
        lds, acc,
        [&](int i, int j) {
            return i < rows && j < cols && partial == nullptr ? tile.residual(i, j, cols - j) : f32x4{0.f, 0.f, 0.f, 0.f};
        },
        [&](int i, int j, f32x4 v, f32x4 residual) {
            if (i >= rows || j >= cols) return v;
            if (partial != nullptr) *reinterpret_cast<f32x4*>(partial + i * ldp + j) = v;
            else tile.store(i, j, cols - j, v, residual);
            return v;
        });
}

// Joins the parts of a split sum, in their order, and finishes the result.
template <int D>
__global__ __launch_bounds__(256) void join_kernel(ProductArgs p, int splits) {
    const int64_t units = p.ldp / 4, total = p.m * units;
    for (int64_t u = blockIdx.x * int64_t(256) + threadIdx.x; u < total; u += int64_t(gridDim.x) * 256) {
        const int64_t m = u / units, n = u % units * 4;
        f32x4 v = *reinterpret_cast<const f32x4*>(p.partial + m * p.ldp + n);
        for (int s = 1; s < splits; ++s)
            v += *reinterpret_cast<const f32x4*>(p.partial + (s * p.m + m) * p.ldp + n);
        const TileEpilogue<D> tile(p, m, n);
        const int have = static_cast<int>(min<int64_t>(p.n - n, 4));
        tile.store(0, 0, have, v, tile.residual(0, 0, have));
    }
}

// ---- few rows ------------------------------------------------------------------------
// At most 16 rows of x: the product is the read of W.  A workgroup of 8 waves forms 16
// columns of y; its waves take k-steps in turn straight from global memory, each wave
// instruction covering 64 bytes of 16 rows of W, and their sums meet in LDS.
template <int D>
__global__ __launch_bounds__(512) void thin_kernel(ProductArgs p) {
    constexpr int E = unit_elems<D>(), kStep = 4 * E, kWaves = 8, kUnroll = 4, B = elem_bytes<D>();
    __shared__ f32x4 sums[kWaves][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, row = lane & 15, q = lane >> 4;
    const int64_t n0 = int64_t(blockIdx.x) * 16;
    const bool w_in = n0 + row < p.n, x_in = row < p.m;
    const char* w = static_cast<const char*>(p.b) + ((n0 + (w_in ? row : 0)) * p.ldb + q * E) * B;
    const char* x = static_cast<const char*>(p.a) + ((x_in ? row : 0) * p.lda + q * E) * B;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    const int64_t whole = p.k / kStep;
    int64_t s = wave * kUnroll;  // kUnroll consecutive steps a turn: 256 bytes of each row
    for (; s + kUnroll <= whole; s += kUnroll * kWaves) {
        u32x4 fw[kUnroll], fx[kUnroll];
#pragma unroll
        for (int i = 0; i < kUnroll; ++i) {
            fw[i] = load16(w + (s + i) * kStep * B);
            fx[i] = load16(x + (s + i) * kStep * B);
        }
#pragma unroll
        for (int i = 0; i < kUnroll; ++i) {
            if (!x_in) fx[i] = u32x4{0, 0, 0, 0};
            acc = mma<D>(fw[i], fx[i], acc);
        }
    }
    for (; s < whole; ++s) {  // the one wave whose turn is cut short
        const u32x4 fw = load16(w + s * kStep * B);
        u32x4 fx = load16(x + s * kStep * B);
        if (!x_in) fx = u32x4{0, 0, 0, 0};
        acc = mma<D>(fw, fx, acc);
    }
    if (wave == whole % kWaves && whole * kStep < p.k) {  // the last, partial step
        u32x4 fw = {0, 0, 0, 0}, fx = {0, 0, 0, 0};
        const int64_t at = whole * kStep;
        for (int e = 0; e < E; ++e) {
            if (at + q * E + e >= p.k) break;
            if constexpr (B == 4) {
                fw[e] = reinterpret_cast<const uint32_t*>(w)[at + e];
                if (x_in) fx[e] = reinterpret_cast<const uint32_t*>(x)[at + e];
            } else {
                fw[e / 2] |= uint32_t(reinterpret_cast<const uint16_t*>(w)[at + e]) << (16 * (e % 2));
                if (x_in) fx[e / 2] |= uint32_t(reinterpret_cast<const uint16_t*>(x)[at + e]) << (16 * (e % 2));
            }
        }
        acc = mma<D>(fw, fx, acc);
    }
    sums[wave][lane] = acc;
    __syncthreads();
    if (wave == 0) {
#pragma unroll
        for (int i = 1; i < kWaves; ++i) acc += sums[i][lane];
        const int64_t n = n0 + 4 * q;
        if (x_in && n < p.n) {
            const TileEpilogue<D> tile(p, row, n);
            const int have = static_cast<int>(min<int64_t>(p.n - n, 4));
            tile.store(0, 0, have, acc, tile.residual(0, 0, have));
        }
    }
}

// ---- the gradient before the products ---------------------------------------------------
struct SlopeArgs {
    const void* dy;
    const void* z;
    void* dz;
    float* partial;  // [row blocks][ldp] column sums, or null
    void* dbias;     // or the sums of the only block
    int64_t lddy, ldz, lddz, ldp, m, n;
    int rows_per_block, act;
};

// dz = dy act'(z) over a block of rows by 64 units of 16 bytes, one a lane, and the block's
// column sums in row order: each of four waves adds every fourth row, and the four meet in LDS.
// Bound by memory: 8192 x 14336 in bf16 takes 125 to 129 us (705 MB, 5.5 TB/s).  kStream, for dy and z
// past the memory-side cache's 256 MB, reads them past it: 127 us against 146 there, but 11.8
// against 10.1 on 1537 x 777, whose z the forward pass has left in it.
template <int D, bool kStream>
__global__ __launch_bounds__(256) void slope_kernel(SlopeArgs p) {
    constexpr int E = unit_elems<D>(), B = elem_bytes<D>();
    __shared__ float sums[4][E][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t j = (int64_t(blockIdx.x) * 64 + lane) * E;
    const int64_t first = int64_t(blockIdx.y) * p.rows_per_block, last = min(p.m, first + p.rows_per_block);
    float sum[E];
#pragma unroll
    for (int e = 0; e < E; ++e) sum[e] = 0.0f;
    if (j + E <= p.n) {
        const char* dy = static_cast<const char*>(p.dy) + j * B;
        const char* z = static_cast<const char*>(p.z) + j * B;
        char* dz = static_cast<char*>(p.dz) + j * B;
        constexpr int kRows = 2;  // rows whose loads are in flight together
        for (int64_t at = first + wave; at < last; at += 4 * kRows) {
            u32x4 gs[kRows], zs[kRows];
#pragma unroll
            for (int k = 0; k < kRows; ++k) {
                const int64_t i = min(at + 4 * k, last - 1);
                const auto read = [](const char* from) { return kStream ? stream16(from) : load16(from); };
                gs[k] = read(dy + i * p.lddy * B);
                zs[k] = p.act == HBT_ACT_NONE ? u32x4{0, 0, 0, 0} : read(z + i * p.ldz * B);
            }
#pragma unroll
            for (int k = 0; k < kRows; ++k) {
                const int64_t i = at + 4 * k;
                if (i >= last) break;
                float g[E];
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    g[e] = element<D>(gs[k], e);
                    if (p.act != HBT_ACT_NONE) g[e] *= slope<D>(element<D>(zs[k], e), p.act);
                    sum[e] += g[e];
                }
                if (p.dz != nullptr) {
#pragma unroll
                    for (int e = 0; e < E; e += 4)
                        store4<D>(dz + i * p.lddz * B, e, f32x4{g[e], g[e + 1], g[e + 2], g[e + 3]});
                }
            }
        }
    } else if (j < p.n) {
        for (int64_t i = first + wave; i < last; i += 4) {
#pragma unroll
            for (int e = 0; e < E - 1; ++e) {
                if (j + e >= p.n) continue;
                float g = load_elem<D>(p.dy, i * p.lddy + j + e);
                if (p.act != HBT_ACT_NONE) g *= slope<D>(load_elem<D>(p.z, i * p.ldz + j + e), p.act);
                if (p.dz != nullptr) store_elem<D>(p.dz, i * p.lddz + j + e, g);
                sum[e] += g;
            }
        }
    }
    if (p.partial == nullptr && p.dbias == nullptr) return;
#pragma unroll
    for (int e = 0; e < E; ++e) sums[wave][e][lane] = sum[e];
    __syncthreads();
    if (wave != 0 || j >= p.n) return;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        if (j + e >= p.n) break;
        const float total = ((sums[0][e][lane] + sums[1][e][lane]) + sums[2][e][lane]) + sums[3][e][lane];
        if (p.dbias != nullptr) store_elem<D>(p.dbias, j + e, total);
        else p.partial[blockIdx.y * p.ldp + j + e] = total;
    }
}

// dbias: the row blocks' column sums, added in their order.
template <int D>
__global__ __launch_bounds__(256) void bias_kernel(const float* partial, int64_t ldp, int blocks, void* db, int64_t n) {
    __shared__ float sums[4][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t j = int64_t(blockIdx.x) * 64 + lane;
    float sum = 0.0f;
    if (j < n) {
#pragma unroll 8
        for (int b = wave; b < blocks; b += 4) sum += partial[b * ldp + j];
    }
    sums[wave][lane] = sum;
    __syncthreads();
    if (wave == 0 && j < n)
        store_elem<D>(db, j, ((sums[0][lane] + sums[1][lane]) + sums[2][lane]) + sums[3][lane]);
}

// ---- small layers ----------------------------------------------------------------------
// A layer whose three sizes are at most 64 has its whole backward pass in one workgroup and one
// launch (the parts above are four, and such a pass is launch latency): dz, x and W in LDS in
// fp32, a lane per result.
constexpr int kSmall = 64, kSmallLd = kSmall + 1;
inline bool is_small(int64_t tokens, int64_t inner, int64_t outer) {
    return tokens > 0 && inner > 0 && outer > 0 && tokens <= kSmall && inner <= kSmall && outer <= kSmall;
}

struct SmallArgs {
    const void *dy, *x, *w, *z;
    void *dx, *dw, *dbias;
    int lddy, ldx, ldw, ldz, lddx, lddw, tokens, inner, outer, act;
};

template <int D>
__global__ __launch_bounds__(512) void small_backward_kernel(SmallArgs p) {
    __shared__ float dz[kSmall * kSmallLd], x[kSmall * kSmallLd], w[kSmall * kSmallLd];
    const int tid = threadIdx.x;
    for (int i = tid; i < p.tokens * p.outer; i += 512) {
        const int t = i / p.outer, o = i % p.outer;
        float g = load_elem<D>(p.dy, int64_t(t) * p.lddy + o);
        if (p.act != HBT_ACT_NONE) g *= slope<D>(load_elem<D>(p.z, int64_t(t) * p.ldz + o), p.act);
        dz[t * kSmallLd + o] = g;
    }
    if (p.dw != nullptr)
        for (int i = tid; i < p.tokens * p.inner; i += 512)
            x[i / p.inner * kSmallLd + i % p.inner] = load_elem<D>(p.x, int64_t(i / p.inner) * p.ldx + i % p.inner);
    if (p.dx != nullptr)
        for (int i = tid; i < p.outer * p.inner; i += 512)
            w[i / p.inner * kSmallLd + i % p.inner] = load_elem<D>(p.w, int64_t(i / p.inner) * p.ldw + i % p.inner);
    __syncthreads();
    if (p.dx != nullptr)
        for (int i = tid; i < p.tokens * p.inner; i += 512) {
            const int t = i / p.inner, k = i % p.inner;
            float sum = 0.0f;
            for (int o = 0; o < p.outer; ++o) sum = fmaf(dz[t * kSmallLd + o], w[o * kSmallLd + k], sum);
            store_elem<D>(p.dx, int64_t(t) * p.lddx + k, sum);
        }
    if (p.dw != nullptr)
        for (int i = tid; i < p.outer * p.inner; i += 512) {
            const int o = i / p.inner, k = i % p.inner;
            float sum = 0.0f;
            for (int t = 0; t < p.tokens; ++t) sum = fmaf(dz[t * kSmallLd + o], x[t * kSmallLd + k], sum);
            store_elem<D>(p.dw, int64_t(o) * p.lddw + k, sum);
        }
    if (p.dbias != nullptr && tid < p.outer) {
        float sum = 0.0f;
        for (int t = 0; t < p.tokens; ++t) sum += dz[t * kSmallLd + tid];
        store_elem<D>(p.dbias, tid, sum);
    }
}

// ---- host ----------------------------------------------------------------------------
template <int D, bool kA, bool kB, class T, bool kAsync>
int32_t launch_tile(const char* who, ProductArgs& p, int splits, hipStream_t stream) {
    constexpr int kLds = lds_bytes<T, kAsync>();
    p.tiles_m = static_cast<int>((p.m + T::BM - 1) / T::BM);
    p.tiles_n = static_cast<int>((p.n + T::BN - 1) / T::BN);
    const auto kernel = product_kernel<D, kA, kB, T, kAsync>;
    if constexpr (kLds > 65536) {
        static std::atomic<uint64_t> done{0};
        const int32_t status = allow_lds(who, reinterpret_cast<const void*>(kernel), kLds, done);
        if (status != HBT_OK) return status;
    }
    kernel<<<dim3(p.tiles_m * p.tiles_n, splits), T::kThreads, kLds, stream>>>(p);
    return check_launch(who);
}

template <int D, bool kA, bool kB>
int32_t launch_large(const char* who, const ProductArgs& p, hipStream_t stream) {
    constexpr int64_t B = elem_bytes<D>();
    const Cut cut = cut_of(p.m, p.n, p.k);
    ProductArgs first = p, last = p;
    first.m = cut.m, first.n = cut.n;
    const int32_t status = launch_tile<D, kA, kB, Tile256, true>(who, first, 1, stream);
    if (status != HBT_OK || (cut.m == p.m && cut.n == p.n)) return status;
    const int64_t m0 = cut.m < p.m ? cut.m : 0, n0 = cut.n < p.n ? cut.n : 0;
    const auto moved = [](auto* at, int64_t elements) {
        using Byte = std::conditional_t<std::is_const_v<std::remove_pointer_t<decltype(at)>>, const char, char>;
        return at == nullptr ? at : static_cast<decltype(at)>(static_cast<Byte*>(at) + elements * B);
    };
    last.m = p.m - m0, last.n = p.n - n0;
    last.a = moved(p.a, kA ? m0 * p.lda : m0);
    last.b = moved(p.b, kB ? n0 * p.ldb : n0);
    last.bias = moved(p.bias, n0);
    last.residual = moved(p.residual, m0 * p.ldr + n0);
    last.y = moved(p.y, m0 * p.ldy + n0);
    last.z = moved(p.z, m0 * p.ldz + n0);
    return launch_tile<D, kA, kB, Tile128, true>(who, last, 1, stream);
}

template <int D, bool kA, bool kB>
int32_t launch_product(const char* who, ProductArgs& p, void* workspace, int64_t workspace_bytes, hipStream_t stream) {
    constexpr int BK = tile_k<D>();
    const bool aligned = is_aligned(p.a, p.lda, kA ? p.k : p.m, D) && is_aligned(p.b, p.ldb, kB ? p.k : p.n, D);
    Choice c = choose(p.m, p.n, p.k, D, aligned);
    p.ldp = (p.n + 3) / 4 * 4;
    while (c.splits > 1 && 4 * c.splits * p.m * p.ldp > workspace_bytes) --c.splits;
    p.k_split = p.k;
    p.partial = nullptr;
    if (c.splits > 1) {
        p.k_split = ((p.k + c.splits - 1) / c.splits + BK - 1) / BK * BK;
        c.splits = static_cast<int>((p.k + p.k_split - 1) / p.k_split);
        if (c.splits > 1) p.partial = static_cast<float*>(workspace);
    }
    int32_t status = HBT_OK;
    if (c.tile == 64) {
        status = aligned ? launch_tile<D, kA, kB, Tile64, true>(who, p, c.splits, stream)
                         : launch_tile<D, kA, kB, Tile64, false>(who, p, c.splits, stream);
    } else if (c.tile == 128) {
        status = aligned ? launch_tile<D, kA, kB, Tile128, true>(who, p, c.splits, stream)
                         : launch_tile<D, kA, kB, Tile128, false>(who, p, c.splits, stream);
    } else if constexpr (D != HBT_DTYPE_F32) {
        status = c.splits > 1 ? launch_tile<D, kA, kB, Tile256, true>(who, p, c.splits, stream)
                              : launch_large<D, kA, kB>(who, p, stream);
    }
    if (status != HBT_OK || c.splits == 1) return status;
    const int64_t blocks = std::min<int64_t>((p.m * (p.ldp / 4) + 255) / 256, 4096);
    join_kernel<D><<<dim3(static_cast<unsigned>(blocks)), 256, 0, stream>>>(p, c.splits);
    return check_launch(who);
}

int32_t fail(const char* who, const char* what) {
    set_error("%s: %s", who, what);
    return HBT_ERR_INVALID_ARGUMENT;
}

int32_t check_matrix(const char* who, const void* p, int64_t rows, int64_t cols, int64_t ld, const char* name) {
    if (rows == 0 || cols == 0) return HBT_OK;
    if (p == nullptr) {
        set_error("%s: %s is null", who, name);
        return HBT_ERR_INVALID_ARGUMENT;
    }
    if (ld < cols) {
        set_error("%s: rows of %s overlap (%lld elements apart, %lld long)", who, name, static_cast<long long>(ld),
                  static_cast<long long>(cols));
        return HBT_ERR_INVALID_ARGUMENT;
    }
    if (ld > kMaxLd) {
        set_error("%s: rows of %s are %lld elements apart; at most %lld", who, name, static_cast<long long>(ld),
                  static_cast<long long>(kMaxLd));
        return HBT_ERR_UNSUPPORTED;
    }
    return HBT_OK;
}

int32_t check_sizes(const char* who, int64_t m, int64_t n, int64_t k, int32_t dtype) {
    if (m < 0 || n < 0 || k < 0) return fail(who, "a size is negative");
    if (dtype != HBT_DTYPE_F32 && dtype != HBT_DTYPE_BF16 && dtype != HBT_DTYPE_F16) {
        set_error("%s: dtype %d is not F32, BF16 or F16", who, dtype);
        return HBT_ERR_INVALID_ARGUMENT;
    }
    if (m > kMaxSide || n > kMaxSide || k > kMaxSide || tile_items(m, n, 128) > kGridMaxItems ||
        tile_items(n, k, 128) > kGridMaxItems || tile_items(m, k, 128) > kGridMaxItems) {
        set_error("%s: sizes %lld x %lld x %lld are past the launch limits", who, static_cast<long long>(m),
                  static_cast<long long>(n), static_cast<long long>(k));
        return HBT_ERR_UNSUPPORTED;
    }
    return HBT_OK;
}

// What the split of a product's sum can use, aligned or not.
int64_t split_bytes(int64_t m, int64_t n, int64_t k, int32_t dtype) {
    if (m <= 0 || n <= 0 || k <= 0) return 0;
    const int splits = std::max(choose(m, n, k, dtype, true).splits, choose(m, n, k, dtype, false).splits);
    return splits == 1 ? 0 : 4 * splits * m * ((n + 3) / 4 * 4);
}

int64_t columns_per_block(int dtype) { return dtype == HBT_DTYPE_F32 ? 256 : 512; }

// Rows per block of the slope pass: enough blocks for the device, few enough partial sums.
int rows_per_block(int64_t m, int64_t n, int dtype) {
    const int64_t columns = (n + columns_per_block(dtype) - 1) / columns_per_block(dtype);
    int64_t rows = m * columns / 2048;
    rows = std::min<int64_t>(std::max<int64_t>(rows, 16), 256);
    while ((m + rows - 1) / rows > 65535) rows *= 2;
    return static_cast<int>(rows);
}

// The backward pass's working storage: dz with rows on 16-byte boundaries when an activation
// makes it differ from dy, then a region that the bias sums and each product's split take in
// turn.
struct BackwardSpace {
    int64_t lddz, dz_bytes, shared_bytes;
};

BackwardSpace backward_space(int64_t tokens, int64_t inner, int64_t outer, int32_t dtype, int32_t activation,
                             int32_t wants) {
    BackwardSpace b{};
    if (tokens <= 0 || outer <= 0) return b;
    const int64_t unit = dtype == HBT_DTYPE_F32 ? 4 : 8, size = dtype == HBT_DTYPE_F32 ? 4 : 2;
    if (activation != HBT_ACT_NONE && (wants & (HBT_LINEAR_DX | HBT_LINEAR_DW)) != 0) {
        b.lddz = (outer + unit - 1) / unit * unit;
        b.dz_bytes = (tokens * b.lddz * size + 255) / 256 * 256;
    }
    if (is_small(tokens, inner, outer)) return BackwardSpace{};
    if ((wants & HBT_LINEAR_DBIAS) && tokens > rows_per_block(tokens, outer, dtype)) {
        const int64_t rows = rows_per_block(tokens, outer, dtype);
        b.shared_bytes = 4 * ((tokens + rows - 1) / rows) * ((outer + 3) / 4 * 4);
    }
    if (wants & HBT_LINEAR_DX)
        b.shared_bytes = std::max(b.shared_bytes, split_bytes(tokens, inner, outer, dtype));
    if (wants & HBT_LINEAR_DW)
        b.shared_bytes = std::max(b.shared_bytes, split_bytes(outer, inner, tokens, dtype));
    return b;
}

template <typename F>
int32_t by_dtype(int32_t dtype, F&& f) {
    if (dtype == HBT_DTYPE_F32) return f(std::integral_constant<int, HBT_DTYPE_F32>{});
    if (dtype == HBT_DTYPE_BF16) return f(std::integral_constant<int, HBT_DTYPE_BF16>{});
    return f(std::integral_constant<int, HBT_DTYPE_F16>{});
}

}  // namespace
}  // namespace mm
}  // namespace hbt

using namespace hbt;
using namespace hbt::mm;

extern "C" {

int64_t hbt_linear_workspace(int64_t tokens, int64_t inner, int64_t outer, int32_t dtype) {
    clear_error();
    if (check_sizes("hbt_linear_workspace", tokens, outer, inner, dtype) != HBT_OK) return -1;
    return tokens <= 16 ? 0 : split_bytes(tokens, outer, inner, dtype);
}

int64_t hbt_linear_backward_workspace(int64_t tokens, int64_t inner, int64_t outer, int32_t dtype, int32_t activation,
                                      int32_t wants) {
    clear_error();
    const char* who = "hbt_linear_backward_workspace";
    if (check_sizes(who, tokens, outer, inner, dtype) != HBT_OK) return -1;
    if (activation < HBT_ACT_NONE || activation > HBT_ACT_SILU) return fail(who, "unknown activation");
    if (wants < 0 || wants > 7) return fail(who, "unknown results are wanted");
    const BackwardSpace b = backward_space(tokens, inner, outer, dtype, activation, wants);
    return b.dz_bytes + b.shared_bytes;
}

int32_t hbt_linear(const void* x, int64_t ldx, const void* w, int64_t ldw, const void* bias, const void* residual,
                   int64_t ldr, void* y, int64_t ldy, void* z, int64_t ldz, int64_t tokens, int64_t inner,
                   int64_t outer, int32_t dtype, int32_t activation, void* workspace, int64_t workspace_bytes,
                   void* stream) {
    clear_error();
    const char* who = "hbt_linear";
    int32_t status = check_sizes(who, tokens, outer, inner, dtype);
    if (status != HBT_OK) return status;
    if (activation < HBT_ACT_NONE || activation > HBT_ACT_SILU) return fail(who, "unknown activation");
    if (tokens == 0 || outer == 0) return HBT_OK;
    if ((status = check_matrix(who, x, tokens, inner, ldx, "x")) != HBT_OK ||
        (status = check_matrix(who, w, outer, inner, ldw, "w")) != HBT_OK ||
        (status = check_matrix(who, y, tokens, outer, ldy, "y")) != HBT_OK)
        return status;
    if (residual != nullptr && (status = check_matrix(who, residual, tokens, outer, ldr, "residual")) != HBT_OK)
        return status;
    if (z != nullptr && (status = check_matrix(who, z, tokens, outer, ldz, "z")) != HBT_OK) return status;
    ProductArgs p{};
    p.a = x, p.b = w, p.bias = bias, p.residual = residual, p.y = y, p.z = z;
    p.lda = ldx, p.ldb = ldw, p.ldr = ldr, p.ldy = ldy, p.ldz = ldz;
    p.m = tokens, p.n = outer, p.k = inner, p.act = activation;
    const hipStream_t s = as_stream(stream);
    return by_dtype(dtype, [&](auto d) -> int32_t {
        constexpr int D = decltype(d)::value;
        if (tokens <= 16) {
            thin_kernel<D><<<dim3(static_cast<unsigned>((outer + 15) / 16)), 512, 0, s>>>(p);
            return check_launch(who);
        }
        return launch_product<D, true, true>(who, p, workspace, workspace == nullptr ? 0 : workspace_bytes, s);
    });
}

int32_t hbt_linear_backward(const void* dy, int64_t lddy, const void* x, int64_t ldx, const void* w, int64_t ldw,
                            const void* z, int64_t ldz, void* dx, int64_t lddx, void* dw, int64_t lddw, void* dbias,
                            int64_t tokens, int64_t inner, int64_t outer, int32_t dtype, int32_t activation,
                            void* workspace, int64_t workspace_bytes, void* stream) {
    clear_error();
    const char* who = "hbt_linear_backward";
    int32_t status = check_sizes(who, tokens, outer, inner, dtype);
    if (status != HBT_OK) return status;
    if (activation < HBT_ACT_NONE || activation > HBT_ACT_SILU) return fail(who, "unknown activation");
    if ((status = check_matrix(who, dy, tokens, outer, lddy, "dy")) != HBT_OK) return status;
    if (activation != HBT_ACT_NONE && (status = check_matrix(who, z, tokens, outer, ldz, "z")) != HBT_OK)
        return status;
    if (dx != nullptr && ((status = check_matrix(who, dx, tokens, inner, lddx, "dx")) != HBT_OK ||
                          (status = check_matrix(who, w, outer, inner, ldw, "w")) != HBT_OK))
        return status;
    if (dw != nullptr && ((status = check_matrix(who, dw, outer, inner, lddw, "dw")) != HBT_OK ||
                          (status = check_matrix(who, x, tokens, inner, ldx, "x")) != HBT_OK))
        return status;
    const int32_t wants = (dx != nullptr ? HBT_LINEAR_DX : 0) | (dw != nullptr ? HBT_LINEAR_DW : 0) |
                          (dbias != nullptr ? HBT_LINEAR_DBIAS : 0);
    const BackwardSpace space = backward_space(tokens, inner, outer, dtype, activation, wants);
    const int64_t need = space.dz_bytes + space.shared_bytes;
    if (need > 0 && (workspace == nullptr || workspace_bytes < need))
        return fail(who, "the workspace is smaller than hbt_linear_backward_workspace's");
    char* shared = static_cast<char*>(workspace) + space.dz_bytes;
    const hipStream_t s = as_stream(stream);
    return by_dtype(dtype, [&](auto d) -> int32_t {
        constexpr int D = decltype(d)::value;
        if (is_small(tokens, inner, outer)) {
            if (wants == 0) return HBT_OK;
            const auto i = [](int64_t v) { return static_cast<int>(v); };
            small_backward_kernel<D><<<dim3(1), 512, 0, s>>>({dy, x, w, z, dx, dw, dbias, i(lddy), i(ldx), i(ldw), i(ldz),
                                                              i(lddx), i(lddw), i(tokens), i(inner), i(outer), activation});
            return check_launch(who);
        }
        SlopeArgs p{};
        p.dy = dy, p.z = z, p.dz = space.dz_bytes > 0 ? workspace : nullptr;
        p.lddy = lddy, p.ldz = ldz, p.lddz = space.lddz, p.ldp = (outer + 3) / 4 * 4;
        p.m = tokens, p.n = outer, p.act = activation;
        int64_t blocks = 0;
        if (tokens > 0 && outer > 0 && (p.dz != nullptr || dbias != nullptr)) {
            p.rows_per_block = rows_per_block(tokens, outer, dtype);
            blocks = (tokens + p.rows_per_block - 1) / p.rows_per_block;
            if (dbias != nullptr && blocks > 1) p.partial = reinterpret_cast<float*>(shared);
            else p.dbias = dbias;
            const dim3 grid(static_cast<unsigned>((outer + columns_per_block(dtype) - 1) / columns_per_block(dtype)),
                            static_cast<unsigned>(blocks));
            const int64_t bytes = tokens * outer * elem_bytes<D>() * (activation != HBT_ACT_NONE ? 2 : 1);
            if (bytes > int64_t(256) << 20) slope_kernel<D, true><<<grid, 256, 0, s>>>(p);
            else slope_kernel<D, false><<<grid, 256, 0, s>>>(p);
            const int32_t launched = check_launch(who);
            if (launched != HBT_OK) return launched;
        }
        if (dbias != nullptr && outer > 0 && blocks != 1) {
            bias_kernel<D><<<dim3(static_cast<unsigned>((outer + 63) / 64)), 256, 0, s>>>(
                p.partial, p.ldp, static_cast<int>(blocks), dbias, outer);
            const int32_t launched = check_launch(who);
            if (launched != HBT_OK) return launched;
        }
        const void* dz = p.dz != nullptr ? p.dz : dy;
        const int64_t lddz = p.dz != nullptr ? space.lddz : lddy;
        if (dx != nullptr && tokens > 0 && inner > 0) {
            ProductArgs q{};
            q.a = dz, q.b = w, q.y = dx, q.lda = lddz, q.ldb = ldw, q.ldy = lddx;
            q.m = tokens, q.n = inner, q.k = outer;
            const int32_t launched = launch_product<D, true, false>(who, q, shared, space.shared_bytes, s);
            if (launched != HBT_OK) return launched;
        }
        if (dw != nullptr && outer > 0 && inner > 0) {
            ProductArgs q{};
            q.a = dz, q.b = x, q.y = dw, q.lda = lddz, q.ldb = ldx, q.ldy = lddw;
            q.m = outer, q.n = inner, q.k = tokens;
            return launch_product<D, false, false>(who, q, shared, space.shared_bytes, s);
        }
        return HBT_OK;
    });
}

}  // extern "C"
