// Orthogonalised updates: momentum, Newton-Schulz products, the step.
//
//   v' = mu v + (1 - mu) g;  u = (1 - mu) g + mu v' (Nesterov) or v';  x = u / max(|u|, eps)
//   `steps` times:  A = x x^T (or x^T x, over the shorter side),  B = b A + c A A,  x = a x + B x
//   w' = decay w - lr scale x
//
// The iterate x is held in 32 bits: fp32, or, beside fp16 products, the fp16 value they read and
// what it leaves of x, 2^11 times as large and in fp16 itself (22 bits of mantissa down to elements
// of 2^-14, below them steps of 2^-36).  The products read copies of x, A and B rounded to the
// product type: fp16 (11 bits, and the values are bounded: singular values stay below 1.3, and x
// is scaled by a power of two near the square root of its longer side, which puts its elements
// near 1 and the first iterate's above fp16's subnormals) or, on request, fp32.  Rounding x itself
// to 16 bits would be amplified by 3.4 a step in the directions that start small: on matrices with
// a decaying spectrum fp16 products then end 6e-3 to 9e-3 off, and 3e-4 to 2e-3 with x in 32.
//
// Every phase takes all matrices in one launch: the tiles of up to 32
// matrices of any sizes, found in a table in the launch's arguments.
#include <tuple>

#include "hbt_matmul.hpp"

namespace hbt {
namespace mm {
namespace {

constexpr int kMaxMatrices = HBT_MAX_MATRICES;
constexpr int kChunk = 4096;  // elements per norm partial
constexpr int kMaxSteps = 64;

// The first workgroup of every matrix of a launch, the unused ones past every workgroup.
struct FirstBlocks {
    int first[kMaxMatrices];
    void clear() {
        for (int& f : first) f = 0x7FFFFFFF;
    }
};
// The matrix of a workgroup: one wide scalar load and a sum of comparisons.
__device__ __forceinline__ int find_entry(const FirstBlocks& blocks, int block) {
    int e = -1;
#pragma unroll
    for (int i = 0; i < kMaxMatrices; ++i) e += blocks.first[i] <= block ? 1 : 0;
    return e;
}

// ---- the direction and its norm --------------------------------------------------------
struct DirectionEntry {
    const void* g;
    float* v;        // null: u is the input itself
    double* partial;
    void* x;         // the first iterate in the product type, [rows][ld]
    void* low;       // the rest of it beside fp16 values, times kLowScale
    const float* factor;
    int64_t rows, cols, ld;
};
struct DirectionArgs {
    FirstBlocks blocks;
    DirectionEntry entry[kMaxMatrices];
    const float* grad_mul;
    const float* slot;  // null, or the momentum and its complement are its third and fourth float
    float unscale, momentum, rest;
    int nesterov;
};

// The fp16 value of x and what it leaves, itself in fp16: at most 2^-11 of x, so 2^11 times that keeps
// fp16's range and its 11 bits, where the remainder of an element below 1/4 is a subnormal.
constexpr float kLowScale = 2048.0f;
__device__ __forceinline__ void split(f32x4 x, u32x2& high, u32x2& low) {
    high = u32x2{pack2_rounded<HBT_DTYPE_F16>(x[0], x[1]), pack2_rounded<HBT_DTYPE_F16>(x[2], x[3])};
    f32x4 left;
#pragma unroll
    for (int e = 0; e < 4; ++e) left[e] = (x[e] - f16_to_f32((high[e / 2] >> (16 * (e % 2))) & 0xFFFFu)) * kLowScale;
    low = u32x2{pack2_rounded<HBT_DTYPE_F16>(left[0], left[1]), pack2_rounded<HBT_DTYPE_F16>(left[2], left[3])};
}

// Two passes over the gradients and momenta, which lie dense, at any alignment; a lane takes four
// columns of a row at a time.  kNorm: v' is stored and the squares of u are summed in fp64.
// Otherwise u is formed again from v', by the same operations, and x = factor u is stored on
// padded rows: reading g and v' twice moves no more than storing u between the passes would.
template <int GD, int D, bool kNorm>
__global__ __launch_bounds__(256) void direction_kernel(DirectionArgs p) {
    const int block = blockIdx.x, entry = find_entry(p.blocks, block);
    const DirectionEntry& t = p.entry[entry];
    const int chunk = block - p.blocks.first[entry];
    const uint32_t units = static_cast<uint32_t>(t.ld / 4);
    const int64_t first = int64_t(chunk) * (kChunk / 4), row0 = first / units;
    const uint32_t unit0 = static_cast<uint32_t>(first - row0 * units);
    const float mul = p.grad_mul != nullptr ? *p.grad_mul : 1.0f;
    const float mu = p.slot != nullptr ? p.slot[2] : p.momentum, rest = p.slot != nullptr ? p.slot[3] : p.rest;
    const float factor = kNorm ? 0.0f : *t.factor;
    constexpr int kUnits = kChunk / 1024;
    int64_t at[kUnits], to[kUnits];
    int have[kUnits];
    f32x4 g[kUnits], v[kUnits];
#pragma unroll
    for (int k = 0; k < kUnits; ++k) {
        const uint32_t local = unit0 + k * 256 + threadIdx.x, down = local / units;
        const int64_t row = row0 + down;
        const int col = static_cast<int>(local - down * units) * 4;
        // at most 0 in a row's padding, whose x is zero; -8 past the last row
        have[k] = row < t.rows ? static_cast<int>(min<int64_t>(t.cols - col, 4)) : -8;
        at[k] = row * t.cols + col;
        to[k] = row * t.ld + col;
        g[k] = v[k] = f32x4{0.f, 0.f, 0.f, 0.f};
        if (have[k] > 0) {
            g[k] = load_row<GD>(t.g, at[k], have[k]);
            if (t.v != nullptr) v[k] = load_row<HBT_DTYPE_F32>(t.v, at[k], have[k]);
        }
    }
    double sum = 0.0;
#pragma unroll
    for (int k = 0; k < kUnits; ++k) {
        if (have[k] <= (kNorm ? 0 : -8)) continue;
        f32x4 u = g[k] * p.unscale * mul;
        if (t.v != nullptr) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if constexpr (kNorm) v[k][e] = mu * v[k][e] + rest * u[e];
                u[e] = p.nesterov ? mu * v[k][e] + rest * u[e] : v[k][e];
            }
            if constexpr (kNorm) store_row<HBT_DTYPE_F32>(t.v, at[k], have[k], v[k]);
        }
        if constexpr (kNorm) {
#pragma unroll
            for (int e = 0; e < 4; ++e) sum += double(u[e]) * double(u[e]);
        } else if constexpr (D == HBT_DTYPE_F32) {
            *reinterpret_cast<f32x4*>(static_cast<float*>(t.x) + to[k]) = u * factor;
        } else {
            u32x2 high, low;
            split(u * factor, high, low);
            *reinterpret_cast<u32x2*>(static_cast<uint16_t*>(t.x) + to[k]) = high;
            *reinterpret_cast<u32x2*>(static_cast<uint16_t*>(t.low) + to[k]) = low;
        }
    }
    if constexpr (kNorm) {
        const double total = block_sum<256>(sum);
        if (threadIdx.x == 0) t.partial[chunk] = total;
    }
}

struct NormEntry {
    const double* partial;
    float* factor;
    int64_t chunks;
    float scale;  // the power of two the iterate is held at
};
struct NormArgs {
    NormEntry entry[kMaxMatrices];
    double eps;
};

// scale / norm within float's range; 0 for a zero norm, whose u is 0 and stays 0.
__device__ __forceinline__ float factor_of(float scale, double norm) {
    const double f = scale / norm;
    return norm == 0.0 ? 0.0f : (f > 3.4028234e38 ? 3.4028234e38f : static_cast<float>(f));
}

// factor = scale / max(|u|, eps), one workgroup a matrix, partials in a fixed order.
__global__ __launch_bounds__(1024) void norm_kernel(NormArgs p) {
    const NormEntry& t = p.entry[blockIdx.x];
    double sum = 0.0;
    for (int64_t i = threadIdx.x; i < t.chunks; i += 1024) sum += t.partial[i];
    const double total = block_sum<1024>(sum);
    if (threadIdx.x == 0) {
        const double norm = sqrt(total);
        const double floor = norm < p.eps ? p.eps : norm;  // a NaN norm stays one
        *t.factor = factor_of(t.scale, floor);
    }
}

// ---- the products ----------------------------------------------------------------------
// kFinish: the last iterate, into the result; kGramParts: a Gram product whose sum is split.
enum Phase { kGram, kSquare, kIterate, kFinish, kGramParts };
constexpr bool is_gram(Phase phase) { return phase == kGram || phase == kGramParts; }

struct Problem {
    const void* x;        // the iterate in the product type, [rows][ldx]
    void* x_next;
    void* gram;           // [side][ldg], side the shorter one
    void* poly;
    void* low;            // what x's fp16 values leave of it, times kLowScale, [rows][ldx], or null
    float* parts;         // [split][side][ldg]: the Gram product's sum in parts
    void* out;            // last step: the parameter or the result, [rows][cols]
    int rows, cols, ldx;
    float gram_scale;     // 1 / scale^2
    float out_scale;      // the step's multiple of x, over scale
    int split;            // the number of parts
};
struct Run {
    int first, count, tiles;  // its matrices, and the workgroups of each
    int parts, part_k;        // a Gram product's sum in parts of part_k
};
struct ProductArgs {
    FirstBlocks blocks;
    Run run[kMaxMatrices];
    Problem problem[kMaxMatrices];
    const float* slot;    // null, or decay and learning rate are its first two floats
    float a, b, c, decay, lr;
    int count, update, out_dtype;
};
static_assert(sizeof(ProductArgs) <= 4096, "kernel arguments");

template <typename F>
__device__ __forceinline__ auto by_dtype(int dtype, F&& f) {
    if (dtype == HBT_DTYPE_F32) return f(std::integral_constant<int, HBT_DTYPE_F32>{});
    if (dtype == HBT_DTYPE_BF16) return f(std::integral_constant<int, HBT_DTYPE_BF16>{});
    return f(std::integral_constant<int, HBT_DTYPE_F16>{});
}

// A wide matrix (rows <= columns) has A = x x^T and x' = a x + B x, a tall one A = x^T x and
// x' = a x + x B.  Every array's rows are padded to 16 bytes with zeros: the products of zeros
// keep the padding zero.
template <int D, class T, Phase kPhase>
__global__ __launch_bounds__(T::kThreads, 2) void newton_schulz_kernel(ProductArgs p) {
    extern __shared__ __align__(16) char lds[];
    // Matrices of one shape share a run of workgroups, which starts at a multiple of 8: each XCD
    // takes consecutive tiles of it, and every XCD its part of each run, whose sums differ in length.
    const int r = find_entry(p.blocks, blockIdx.x), local = blockIdx.x - p.blocks.first[r];
    const Run& run = p.run[r];
    if (local >= run.count * run.tiles) return;
    const int global = xcd_tile(local, run.count * run.tiles);
    const Problem& t = p.problem[run.first + global / run.tiles];
    const bool wide = t.rows <= t.cols;
    const int side = wide ? t.rows : t.cols;
    int tile = global % run.tiles, k0 = 0, k1 = wide ? t.cols : t.rows, part = 0;
    if constexpr (kPhase == kGramParts) {  // the parts of one tile are neighbours
        part = tile % run.parts, tile /= run.parts;
        k0 = part * run.part_k, k1 = min(k1, k0 + run.part_k);
    }
    const int ldg = (side + 7) / 8 * 8;
    int tm, tn;
    constexpr bool kProduct = kPhase == kIterate || kPhase == kFinish;
    if constexpr (kProduct) {
        band_order<8>(tile, (t.rows + T::BM - 1) / T::BM, (t.cols + T::BN - 1) / T::BN, tm, tn);
    } else {  // the lower triangle of a symmetric result, row by row
        tm = static_cast<int>((sqrtf(8.0f * tile + 1.0f) - 1.0f) * 0.5f);
        while (tm * (tm + 1) / 2 > tile) --tm;
        while ((tm + 1) * (tm + 2) / 2 <= tile) ++tm;
        tn = tile - tm * (tm + 1) / 2;
    }
    const int m0 = tm * T::BM, n0 = tn * T::BN;
    f32x4 acc[T::TM][T::TN];
    if constexpr (is_gram(kPhase)) {
        if (wide)
            tile_product<D, true, true, T, true>(t.x, t.ldx, m0, side, t.x, t.ldx, n0, side, k0, k1, lds, acc);
        else
            tile_product<D, false, false, T, true>(t.x, t.ldx, m0, t.ldx, t.x, t.ldx, n0, t.ldx, k0, k1, lds, acc);
    } else if constexpr (kPhase == kSquare) {
        tile_product<D, true, true, T, true>(t.gram, ldg, m0, side, t.gram, ldg, n0, side, 0, side, lds, acc);
    } else if (wide) {
        tile_product<D, true, false, T, true>(t.poly, ldg, m0, side, t.x, t.ldx, n0, t.ldx, 0, side, lds, acc);
    } else {
        tile_product<D, true, true, T, true>(t.x, t.ldx, m0, t.rows, t.poly, ldg, n0, side, 0, side, lds, acc);
    }
    // Offsets from the tile's first element fit 32 bits; loads past an edge repeat the last row or
    // the last four columns, stores stop there.
    if constexpr (kProduct) {
        const int64_t at = int64_t(m0) * t.ldx + n0, dense = int64_t(m0) * t.cols + n0;
        const int rows = t.rows - m0, cols = t.cols - n0, padded = t.ldx - n0, ldx = t.ldx, ldo = t.cols;
        const char* x = static_cast<const char*>(t.x) + at * elem_bytes<D>();
        const char* low = static_cast<const char*>(t.low) + at * 2;
        const auto old = [&](int i, int j) {
            const int from = min(i, rows - 1) * ldx + min(j, padded - 4);
            f32x4 v = load4<D>(x, from);
            if constexpr (D != HBT_DTYPE_F32) {
                const u32x2 r = *reinterpret_cast<const u32x2*>(low + int64_t(from) * 2);
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    v[e] = fmaf(f16_to_f32((r[e / 2] >> (16 * (e % 2))) & 0xFFFFu), 1.0f / kLowScale, v[e]);
            }
            return v;
        };
        if constexpr (kPhase == kIterate) {
            char* to_x = static_cast<char*>(t.x_next) + at * elem_bytes<D>();
            char* to_low = static_cast<char*>(t.low) + at * 2;
            finish_tile<T, true, 16>(lds, acc, old, [&](int i, int j, f32x4 v, f32x4 l) {
                v += l * p.a;
                if (i < rows && j < padded) {
                    const int to = i * ldx + j;
                    if constexpr (D == HBT_DTYPE_F32) {
                        store4<D>(to_x, to, v);
                    } else {
                        u32x2 high, rest;
                        split(v, high, rest);
                        *reinterpret_cast<u32x2*>(to_x + int64_t(to) * 2) = high;
                        *reinterpret_cast<u32x2*>(to_low + int64_t(to) * 2) = rest;
                    }
                }
                return v;
            });
        } else {
            const float decay = p.slot != nullptr ? p.slot[0] : p.decay, lr = p.slot != nullptr ? p.slot[1] : p.lr;
            const float step = p.update ? -lr * t.out_scale : t.out_scale;
            by_dtype(p.out_dtype, [&](auto d) {
                constexpr int PD = decltype(d)::value;
                char* out = static_cast<char*>(t.out) + dense * elem_bytes<PD>();
                finish_tile<T, true, 2>(lds, acc, old, [&](int i, int j, f32x4 v, f32x4 l) {
                    if (i >= rows || j >= cols) return v;
                    const int to = i * ldo + j;
                    // w' = decay w - lr out_scale x, or the result out_scale x itself
                    v = (v + l * p.a) * step;
                    if (p.update) v += load_row<PD>(out, to, cols - j) * decay;
                    store_row<PD>(out, to, cols - j, v);
                    return v;
                });
            });
        }
    } else {
        const int rows = side - m0, cols = side - n0, padded_rows = ldg - m0, padded_cols = ldg - n0;
        char* out = static_cast<char*>(is_gram(kPhase) ? t.gram : t.poly);
        char* direct = out + (int64_t(m0) * ldg + n0) * elem_bytes<D>();
        char* mirror = out + (int64_t(n0) * ldg + m0) * elem_bytes<D>();
        const char* gram = static_cast<const char*>(t.gram) + (int64_t(m0) * ldg + n0) * elem_bytes<D>();
        float* sums = kPhase == kGramParts && run.parts > 1 ? t.parts + (int64_t(part) * side + m0) * ldg + n0 : nullptr;
        // Off the diagonal the mirror image is stored too: the products are bitwise symmetric.
        finish_tile<T, true, 8>(
            lds, acc,
            [&](int i, int j) {
                if constexpr (is_gram(kPhase)) return f32x4{0.f, 0.f, 0.f, 0.f};
                else return load4<D>(gram, min(i, rows - 1) * ldg + min(j, padded_cols - 4));
            },
            [&](int i, int j, f32x4 v, f32x4 l) {
                if constexpr (kPhase == kGramParts) {
                    if (sums != nullptr) {
                        if (i < rows && j < padded_cols) *reinterpret_cast<f32x4*>(sums + i * ldg + j) = v;
                        return v;
                    }
                }
                v = is_gram(kPhase) ? v * t.gram_scale : l * p.b + v * p.c;
                if (i >= rows) v = f32x4{0.f, 0.f, 0.f, 0.f};  // the mirror image's padding
                if (i < rows && j < padded_cols) store4<D>(direct, i * ldg + j, v);
                return v;
            },
            tm != tn && sums == nullptr,
            [&](int j, int i, f32x4 v) {
                if (j < cols && i < padded_rows) store4<D>(mirror, j * ldg + i, v);
            });
    }
}

// A Gram product from its parts, added in their order: four columns of a row a lane, read from the
// lower triangle of tiles of `size` that the parts hold.
template <int D>
__global__ __launch_bounds__(256) void gram_join_kernel(ProductArgs p, int size) {
    const int r = find_entry(p.blocks, blockIdx.x), local = blockIdx.x - p.blocks.first[r];
    const Run& run = p.run[r];
    const Problem& t = p.problem[run.first + local / run.tiles];
    const int side = min(t.rows, t.cols), ldg = (side + 7) / 8 * 8, units = ldg / 4;
    const int u = local % run.tiles * 256 + threadIdx.x, i = u / units, j = u % units * 4;
    if (i >= side) return;
    const int64_t part = int64_t(side) * ldg;
    f32x4 sum = {0.f, 0.f, 0.f, 0.f};
    if (i / size >= j / size) {
        const float* at = t.parts + int64_t(i) * ldg + j;
        for (int k = 0; k < run.parts; ++k) sum += *reinterpret_cast<const f32x4*>(at + k * part);
    } else {
        const float* at = t.parts + int64_t(j) * ldg + i;
        for (int k = 0; k < run.parts; ++k)
#pragma unroll
            for (int e = 0; e < 4; ++e) sum[e] += j + e < side ? at[k * part + e * ldg] : 0.0f;
    }
    sum *= t.gram_scale;
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (j + e >= side) sum[e] = 0.0f;
    store4<D>(t.gram, int64_t(i) * ldg + j, sum);
}

// ---- small matrices --------------------------------------------------------------------
// A matrix whose sides are at most 64 and 128 is one workgroup's whole step, in fp32: it stays
// in LDS from its gradient to its parameter, so a model of small matrices is one launch.  The
// products are 16 x 16 tiles of fp32 matrix instructions over LDS, zero-padded to whole tiles.
constexpr int kSmallSide = 64, kSmallLong = 128;
constexpr int kSmallLd = kSmallSide + 4, kSmallXLd = kSmallLong + 4;  // 16 rows by 4 k: distinct banks
constexpr int kSmallLds = 4 * (kSmallSide * kSmallXLd + 2 * kSmallSide * kSmallLd);

struct SmallEntry {
    const void* g;
    float* v;
    void* out;
    int rows, cols;
    float scale;
};
struct SmallArgs {
    SmallEntry entry[kMaxMatrices];
    const float* grad_mul;
    const float* slot;
    double eps;
    float unscale, momentum, rest, a, b, c, decay, lr;
    int nesterov, steps, update, out_dtype;
};

template <int GD>
__global__ __launch_bounds__(512) void small_kernel(SmallArgs p) {
    extern __shared__ __align__(16) char lds[];
    float* x = reinterpret_cast<float*>(lds);
    float* gram = x + kSmallSide * kSmallXLd;
    float* poly = gram + kSmallSide * kSmallLd;
    const SmallEntry& t = p.entry[blockIdx.x];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, row = lane & 15, q = lane >> 4;
    const bool wide = t.rows <= t.cols;
    const int side = wide ? t.rows : t.cols, len = wide ? t.cols : t.rows;
    const int side16 = (side + 15) / 16, len16 = (len + 15) / 16, numel = t.rows * t.cols;
    const float mul = p.grad_mul != nullptr ? *p.grad_mul : 1.0f;
    const float mu = p.slot != nullptr ? p.slot[2] : p.momentum, rest = p.slot != nullptr ? p.slot[3] : p.rest;
    const auto place = [&](int i) {  // element i of the matrix in x, its shorter side as rows
        const int r = i / t.cols, c = i % t.cols;
        return wide ? r * kSmallXLd + c : c * kSmallXLd + r;
    };
    for (int i = tid; i < kSmallSide * kSmallXLd; i += 512) x[i] = 0.0f;
    __syncthreads();
    double sum = 0.0;
    for (int i = tid; i < numel; i += 512) {
        float u = load_elem<GD>(t.g, i) * p.unscale * mul;
        if (t.v != nullptr) {
            const float v = mu * t.v[i] + rest * u;
            u = p.nesterov ? mu * v + rest * u : v;
            t.v[i] = v;
        }
        x[place(i)] = u;
        sum += double(u) * double(u);
    }
    const double total = block_sum<512>(sum);
    __shared__ float factor;
    if (tid == 0) {
        const double norm = sqrt(total);
        const double floor = norm < p.eps ? p.eps : norm;
        factor = factor_of(1.0f, floor);
    }
    __syncthreads();
    for (int i = tid; i < numel; i += 512) x[place(i)] *= factor;
    __syncthreads();
    for (int s = 0; s < p.steps; ++s) {
        for (int tile = wave; tile < side16 * side16; tile += 8) {  // A = x x^T
            const float* a = x + (tile / side16 * 16 + row) * kSmallXLd + q;
            const float* b = x + (tile % side16 * 16 + row) * kSmallXLd + q;
            f32x4 acc = {0.f, 0.f, 0.f, 0.f};
            for (int k = 0; k < len16 * 16; k += 4) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a[k], b[k], acc, 0, 0, 0);
#pragma unroll
            for (int e = 0; e < 4; ++e) gram[(tile / side16 * 16 + 4 * q + e) * kSmallLd + tile % side16 * 16 + row] = acc[e];
        }
        __syncthreads();
        for (int tile = wave; tile < side16 * side16; tile += 8) {  // B = b A + c A A, A symmetric
            const float* a = gram + (tile / side16 * 16 + row) * kSmallLd + q;
            const float* b = gram + (tile % side16 * 16 + row) * kSmallLd + q;
            f32x4 acc = {0.f, 0.f, 0.f, 0.f};
            for (int k = 0; k < side16 * 16; k += 4) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a[k], b[k], acc, 0, 0, 0);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int at = (tile / side16 * 16 + 4 * q + e) * kSmallLd + tile % side16 * 16 + row;
                poly[at] = p.b * gram[at] + p.c * acc[e];
            }
        }
        __syncthreads();
        for (int col = wave; col < len16; col += 8) {  // 16 columns of x = a x + B x, this wave's alone
            f32x4 acc[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
            for (int k = 0; k < side16 * 16; k += 4) {
                const float b = x[(k + q) * kSmallXLd + col * 16 + row];
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (i < side16)
                        acc[i] = __builtin_amdgcn_mfma_f32_16x16x4f32(poly[(i * 16 + row) * kSmallLd + k + q], b, acc[i],
                                                                      0, 0, 0);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (i >= side16) continue;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float* at = x + (i * 16 + 4 * q + e) * kSmallXLd + col * 16 + row;
                    *at = p.a * *at + acc[i][e];
                }
            }
        }
        __syncthreads();
    }
    const float decay = p.slot != nullptr ? p.slot[0] : p.decay, lr = p.slot != nullptr ? p.slot[1] : p.lr;
    const auto finish_all = [&](auto d) {
        constexpr int PD = decltype(d)::value;
        for (int i = tid; i < numel; i += 512) {
            float w = x[place(i)] * t.scale;
            if (p.update) w = load_elem<PD>(t.out, i) * decay - lr * w;
            store_elem<PD>(t.out, i, w);
        }
    };
    if (p.out_dtype == HBT_DTYPE_F32) finish_all(std::integral_constant<int, HBT_DTYPE_F32>{});
    else if (p.out_dtype == HBT_DTYPE_BF16) finish_all(std::integral_constant<int, HBT_DTYPE_BF16>{});
    else finish_all(std::integral_constant<int, HBT_DTYPE_F16>{});
}

// ---- host ----------------------------------------------------------------------------
struct Plan {
    int64_t low, x0, x1, gram, poly, parts, partial, factor, end;  // offsets of one matrix's storage
    int64_t chunks, ldx, ldg;
    int split;
};

// The parts a Gram product's sum over the longer side is split into.  Long thin matrices have few
// tiles, whose sums the parts spread over the device: up to 64 workgroups a matrix, eight k-tiles
// or more each, where that is at least three parts (joining them is one more launch).  Five steps on
// one 50257 x 64 matrix take 330 us, with whole sums 5490; on 24 of 4096 x 64 270 and 609.  The rule
// sees one matrix, so that its bits do not depend on what shares its launches.
int parts_of(int64_t rows, int64_t cols, int product) {
    const int64_t n = (std::min(rows, cols) + 63) / 64, tiles = n * (n + 1) / 2;
    const int64_t steps = std::max(rows, cols) / (product == HBT_DTYPE_F32 ? 32 : 64);
    const int64_t parts = std::min(64 / tiles, steps / 8);
    return parts < 3 ? 1 : static_cast<int>(parts);
}

Plan plan_of(int64_t rows, int64_t cols, int product, int64_t at) {
    const auto take = [&](int64_t bytes) {
        const int64_t here = at;
        at += (bytes + 255) / 256 * 256;
        return here;
    };
    const int64_t size = product == HBT_DTYPE_F32 ? 4 : 2, side = std::min(rows, cols);
    Plan p{};
    p.ldx = (cols + 7) / 8 * 8;
    p.ldg = (side + 7) / 8 * 8;
    p.chunks = (rows * p.ldx + kChunk - 1) / kChunk;
    p.low = product == HBT_DTYPE_F32 ? at : take(rows * p.ldx * 2);
    p.x0 = take(rows * p.ldx * size);
    p.x1 = take(rows * p.ldx * size);
    p.gram = take(side * p.ldg * size);
    p.poly = take(side * p.ldg * size);
    p.split = parts_of(rows, cols, product);
    p.parts = p.split == 1 ? at : take(p.split * side * p.ldg * 4);
    p.partial = take(p.chunks * 8);
    p.factor = take(4);
    p.end = at;
    return p;
}

// The power of two that brings an orthogonal matrix's elements near 1 in fp16.
float iterate_scale(int64_t rows, int64_t cols, int product) {
    if (product == HBT_DTYPE_F32) return 1.0f;
    float s = 1.0f;
    while (s * s * 4.0f <= static_cast<float>(std::max(rows, cols))) s *= 2.0f;
    return s;
}

// A matrix's own product type: fp16's rounding errors average over long sides (5 of 1402 x 100
// came out 2.0e-3 off, 24 of 768 x 768 1.1e-3), and a short side's products cost little beside
// its memory traffic, so those are formed in fp32.
int product_of(int64_t rows, int64_t cols, int product) {
    return std::min(rows, cols) <= 128 ? HBT_DTYPE_F32 : product;
}

bool is_small(int64_t rows, int64_t cols) {
    return std::min(rows, cols) <= kSmallSide && std::max(rows, cols) <= kSmallLong;
}

struct Matrices {
    const void* const* grads;
    float* const* momenta;
    void* const* outs;
    const int64_t* rows;
    const int64_t* cols;
    const float* scales;
    int count;
};

int64_t tiles_of(const Problem& t, int size, Phase phase) {
    const auto n = [&](int64_t extent) { return (extent + size - 1) / size; };
    if (phase == kIterate || phase == kFinish) return n(t.rows) * n(t.cols);
    const int64_t s = n(std::min(t.rows, t.cols));
    return s * (s + 1) / 2;
}

template <int D, class T, Phase kPhase>
int32_t launch_phase_tile(const char* who, ProductArgs& p, int size, hipStream_t stream) {
    constexpr int kLds = lds_bytes<T, true>();
    int64_t blocks = 0;
    p.blocks.clear();
    for (int i = 0, r = 0; i < p.count; i += p.run[r++].count) {
        const Problem& t = p.problem[i];
        int n = 1;
        while (i + n < p.count && p.problem[i + n].rows == t.rows && p.problem[i + n].cols == t.cols) ++n;
        Run& run = p.run[r];
        run = {i, n, static_cast<int>(tiles_of(t, size, kPhase)), 1, 0};
        if (kPhase == kGramParts) {
            const int length = std::max(t.rows, t.cols);
            run.part_k = ((length + t.split - 1) / t.split + tile_k<D>() - 1) / tile_k<D>() * tile_k<D>();
            run.parts = (length + run.part_k - 1) / run.part_k;
            run.tiles *= run.parts;
        }
        p.blocks.first[r] = static_cast<int>(blocks);
        blocks += (int64_t(n) * run.tiles + 7) / 8 * 8;
    }
    const auto kernel = newton_schulz_kernel<D, T, kPhase>;
    if constexpr (kLds > 65536) {
        static std::atomic<uint64_t> done{0};
        const int32_t status = allow_lds(who, reinterpret_cast<const void*>(kernel), kLds, done);
        if (status != HBT_OK) return status;
    }
    kernel<<<dim3(static_cast<unsigned>(blocks)), T::kThreads, kLds, stream>>>(p);
    int32_t status = check_launch(who);
    if (kPhase != kGramParts || status != HBT_OK) return status;
    int64_t joins = 0;
    for (int i = 0, r = 0; i < p.count; i += p.run[r++].count) {
        const Problem& t = p.problem[i];
        const int64_t side = std::min(t.rows, t.cols), units = (side + 7) / 8 * 2;
        p.run[r].tiles = static_cast<int>((side * units + 255) / 256);
        p.blocks.first[r] = static_cast<int>(joins);
        if (p.run[r].parts > 1) joins += int64_t(p.run[r].count) * p.run[r].tiles;
    }
    if (joins == 0) return HBT_OK;
    gram_join_kernel<D><<<dim3(static_cast<unsigned>(joins)), 256, 0, stream>>>(p, size);
    return check_launch(who);
}

template <int D, Phase kPhase>
int32_t launch_phase(const char* who, ProductArgs& p, hipStream_t stream) {
    if (p.count == 0) return HBT_OK;
    int best = 64;
    double least = 0.0;
    for (const int size : {64, 128, 256}) {
        if (size == 256 && D == HBT_DTYPE_F32) continue;
        int64_t tiles = 0;
        double steps = 0.0;
        for (int i = 0; i < p.count; ++i) {
            const Problem& t = p.problem[i];
            const int64_t count = tiles_of(t, size, kPhase);
            const int k = is_gram(kPhase) ? std::max(t.rows, t.cols) : std::min(t.rows, t.cols);
            tiles += count * (is_gram(kPhase) ? t.split : 1);
            steps += static_cast<double>(count) * k / tile_k<D>();
        }
        // Mirror images, and the reads and writes of the iterate, make rounds longer than a layer's.
        const double cost = round_cost(size, tiles, steps / tiles, D == HBT_DTYPE_F32,
                                       size == 256 ? 20.0 : (size == 128 ? 13.0 : 4.0));
        if (least == 0.0 || cost < least) least = cost, best = size;
    }
    if constexpr (D != HBT_DTYPE_F32) {
        if (best == 256) return launch_phase_tile<D, Tile256, kPhase>(who, p, 256, stream);
    }
    if (best == 128) return launch_phase_tile<D, Tile128, kPhase>(who, p, 128, stream);
    return launch_phase_tile<D, Tile64, kPhase>(who, p, 64, stream);
}

// The small matrices of a call, all in one launch.
int32_t run_small(const char* who, const Matrices& t, int32_t grad_dtype, const DirectionArgs& direction,
                  const ProductArgs& common, int steps, double eps, hipStream_t stream) {
    SmallArgs p{};
    int n = 0;
    for (int i = 0; i < t.count; ++i) {
        if (t.rows[i] * t.cols[i] == 0 || !is_small(t.rows[i], t.cols[i])) continue;
        p.entry[n++] = {t.grads[i], t.momenta == nullptr ? nullptr : t.momenta[i], t.outs[i],
                        static_cast<int>(t.rows[i]), static_cast<int>(t.cols[i]),
                        t.scales == nullptr ? 1.0f : t.scales[i]};
    }
    if (n == 0) return HBT_OK;
    p.grad_mul = direction.grad_mul, p.slot = direction.slot, p.eps = eps;
    p.unscale = direction.unscale, p.momentum = direction.momentum, p.rest = direction.rest;
    p.a = common.a, p.b = common.b, p.c = common.c, p.decay = common.decay, p.lr = common.lr;
    p.nesterov = direction.nesterov, p.steps = steps, p.update = common.update, p.out_dtype = common.out_dtype;
    const auto launch = [&](auto d) {
        const auto kernel = small_kernel<decltype(d)::value>;
        static std::atomic<uint64_t> done{0};
        const int32_t status = allow_lds(who, reinterpret_cast<const void*>(kernel), kSmallLds, done);
        if (status != HBT_OK) return status;
        kernel<<<dim3(n), 512, kSmallLds, stream>>>(p);
        return check_launch(who);
    };
    if (grad_dtype == HBT_DTYPE_F32) return launch(std::integral_constant<int, HBT_DTYPE_F32>{});
    if (grad_dtype == HBT_DTYPE_BF16) return launch(std::integral_constant<int, HBT_DTYPE_BF16>{});
    return launch(std::integral_constant<int, HBT_DTYPE_F16>{});
}

// The matrices whose products read type D.
template <int D>
int32_t run(const char* who, const Matrices& t, int32_t grad_dtype, int32_t product, DirectionArgs& direction,
            ProductArgs& common, int steps, double eps, char* workspace, hipStream_t stream) {
    NormArgs norm{};
    // Longest sums first, so that a launch's last workgroups are its shortest: over the longer
    // sides for the Gram products, over the shorter ones for the others.
    ProductArgs by_length = common, by_side = common;
    by_length.count = by_side.count = 0;
    norm.eps = eps;
    direction.blocks.clear();
    int64_t at = 0, direction_blocks = 0;
    int n = 0;
    bool split = false;
    for (int i = 0; i < t.count; ++i) {
        const int64_t rows = t.rows[i], cols = t.cols[i];
        if (rows == 0 || cols == 0 || is_small(rows, cols)) continue;
        const int kind = product_of(rows, cols, product);
        const Plan plan = plan_of(rows, cols, kind, at);
        at = plan.end;
        if (kind != D) continue;
        const float scale = iterate_scale(rows, cols, D);
        void* low = D == HBT_DTYPE_F32 ? nullptr : workspace + plan.low;
        float* factor = reinterpret_cast<float*>(workspace + plan.factor);
        double* partial = reinterpret_cast<double*>(workspace + plan.partial);
        direction.entry[n] = {t.grads[i], t.momenta == nullptr ? nullptr : t.momenta[i], partial, workspace + plan.x0, low,
                              factor, rows, cols, plan.ldx};
        direction.blocks.first[n] = static_cast<int>(direction_blocks);
        direction_blocks += plan.chunks;
        split |= plan.split > 1;
        norm.entry[n] = {partial, factor, plan.chunks, scale};
        ++n;
        by_length.problem[by_length.count++] = {
            workspace + plan.x0, workspace + plan.x1, workspace + plan.gram, workspace + plan.poly, low,
            reinterpret_cast<float*>(workspace + plan.parts), t.outs[i],
            static_cast<int>(rows), static_cast<int>(cols), static_cast<int>(plan.ldx), 1.0f / (scale * scale),
            (t.scales == nullptr ? 1.0f : t.scales[i]) / scale, plan.split};
    }
    if (n == 0) return HBT_OK;
    const dim3 grid(static_cast<unsigned>(direction_blocks));
    const auto pass = [&](auto kNorm) {
        constexpr bool norm_pass = decltype(kNorm)::value;
        if (grad_dtype == HBT_DTYPE_F32) direction_kernel<HBT_DTYPE_F32, D, norm_pass><<<grid, 256, 0, stream>>>(direction);
        else if (grad_dtype == HBT_DTYPE_BF16) direction_kernel<HBT_DTYPE_BF16, D, norm_pass><<<grid, 256, 0, stream>>>(direction);
        else direction_kernel<HBT_DTYPE_F16, D, norm_pass><<<grid, 256, 0, stream>>>(direction);
        return check_launch(who);
    };
    int32_t status = pass(std::true_type{});
    if (status != HBT_OK) return status;
    norm_kernel<<<dim3(n), 1024, 0, stream>>>(norm);
    if ((status = check_launch(who)) != HBT_OK || (status = pass(std::false_type{})) != HBT_OK) return status;
    std::copy_n(by_length.problem, n, by_side.problem);
    by_side.count = n;
    const auto sort = [](ProductArgs& p, auto&& key) {
        std::sort(p.problem, p.problem + p.count, [&](const Problem& a, const Problem& b) {
            return std::make_tuple(-key(a), a.rows, a.cols, a.x) < std::make_tuple(-key(b), b.rows, b.cols, b.x);
        });
    };
    sort(by_length, [](const Problem& t) { return std::max(t.rows, t.cols); });
    sort(by_side, [](const Problem& t) { return std::min(t.rows, t.cols); });
    for (int s = 0; s < steps; ++s) {
        status = split ? launch_phase<D, kGramParts>(who, by_length, stream) : launch_phase<D, kGram>(who, by_length, stream);
        if (status != HBT_OK || (status = launch_phase<D, kSquare>(who, by_side, stream)) != HBT_OK)
            return status;
        if (s + 1 == steps) return launch_phase<D, kFinish>(who, by_side, stream);
        if ((status = launch_phase<D, kIterate>(who, by_side, stream)) != HBT_OK) return status;
        for (ProductArgs* p : {&by_length, &by_side})
            for (int i = 0; i < n; ++i) {
                const void* x = p->problem[i].x;
                p->problem[i].x = p->problem[i].x_next;
                p->problem[i].x_next = const_cast<void*>(x);
            }
    }
    return HBT_OK;
}

int32_t invalid(const char* who, const char* what) {
    set_error("%s: %s", who, what);
    return HBT_ERR_INVALID_ARGUMENT;
}

bool known(int32_t dtype) { return dtype == HBT_DTYPE_F32 || dtype == HBT_DTYPE_BF16 || dtype == HBT_DTYPE_F16; }

// Sides that keep 16-byte units of a tile's rows inside 31-bit offsets, and element counts whose
// workgroups fit one launch.
constexpr int64_t kMaxSide = int64_t(1) << 20;
constexpr int64_t kMaxElements = int64_t(1) << 34;

int32_t check_matrices(const char* who, const Matrices& t, int32_t product, int32_t steps, int64_t* bytes) {
    if (t.count < 0 || t.count > kMaxMatrices) {
        set_error("%s: count %d is outside 0..%d", who, t.count, kMaxMatrices);
        return HBT_ERR_INVALID_ARGUMENT;
    }
    if (t.count > 0 && (t.rows == nullptr || t.cols == nullptr)) return invalid(who, "a table is null");
    if (product != HBT_DTYPE_F16 && product != HBT_DTYPE_F32) {
        set_error("%s: product dtype %d is not F16 or F32", who, product);
        return HBT_ERR_INVALID_ARGUMENT;
    }
    if (steps < 1 || steps > kMaxSteps) {
        set_error("%s: %d steps are outside 1..%d", who, steps, kMaxSteps);
        return HBT_ERR_INVALID_ARGUMENT;
    }
    int64_t at = 0, elements = 0;
    for (int i = 0; i < t.count; ++i) {
        const int64_t rows = t.rows[i], cols = t.cols[i];
        if (rows < 0 || cols < 0) return invalid(who, "a size is negative");
        if (rows == 0 || cols == 0) continue;
        if (rows > kMaxSide || cols > kMaxSide || (elements += rows * cols) > kMaxElements) {
            set_error("%s: matrix %d (%lld x %lld) is past the limits of one call", who, i,
                      static_cast<long long>(rows), static_cast<long long>(cols));
            return HBT_ERR_UNSUPPORTED;
        }
        if (!is_small(rows, cols)) at = plan_of(rows, cols, product_of(rows, cols, product), at).end;
    }
    *bytes = at;
    return HBT_OK;
}

int32_t dispatch(const char* who, const Matrices& t, int32_t grad_dtype, int32_t product, DirectionArgs& direction,
                 ProductArgs& common, int steps, double eps, void* workspace, int64_t workspace_bytes, void* stream) {
    int64_t need = 0;
    const int32_t status = check_matrices(who, t, product, steps, &need);
    if (status != HBT_OK) return status;
    if (!known(grad_dtype) || !known(common.out_dtype)) return invalid(who, "dtypes are F32, BF16 or F16");
    if (!(eps >= 0.0)) return invalid(who, "eps is negative");
    for (int i = 0; i < t.count; ++i) {
        if (t.rows[i] == 0 || t.cols[i] == 0) continue;
        if (t.grads == nullptr || t.outs == nullptr || t.grads[i] == nullptr || t.outs[i] == nullptr ||
            (t.momenta != nullptr && t.momenta[i] == nullptr))
            return invalid(who, "a matrix is null");
    }
    if (need > 0 && (workspace == nullptr || workspace_bytes < need))
        return invalid(who, "the workspace is smaller than hbt_orthogonal_workspace's");
    char* space = static_cast<char*>(workspace);
    const hipStream_t s = as_stream(stream);
    int32_t launched = run_small(who, t, grad_dtype, direction, common, steps, eps, s);
    if (launched == HBT_OK)
        launched = run<HBT_DTYPE_F32>(who, t, grad_dtype, product, direction, common, steps, eps, space, s);
    if (launched == HBT_OK && product != HBT_DTYPE_F32)
        launched = run<HBT_DTYPE_F16>(who, t, grad_dtype, product, direction, common, steps, eps, space, s);
    return launched;
}

}  // namespace
}  // namespace mm
}  // namespace hbt

using namespace hbt;
using namespace hbt::mm;

extern "C" {

int64_t hbt_orthogonal_workspace(const int64_t* rows, const int64_t* cols, int32_t count, int32_t product_dtype) {
    clear_error();
    Matrices t{};
    t.rows = rows, t.cols = cols, t.count = count;
    int64_t bytes = 0;
    return check_matrices("hbt_orthogonal_workspace", t, product_dtype, 1, &bytes) == HBT_OK ? bytes : -1;
}

int32_t hbt_orthogonalize(const void* const* inputs, void* const* outputs, const int64_t* rows, const int64_t* cols,
                          int32_t count, int32_t in_dtype, int32_t out_dtype, int32_t product_dtype, int32_t steps,
                          float a, float b, float c, double eps, void* workspace, int64_t workspace_bytes,
                          void* stream) {
    clear_error();
    Matrices t{inputs, nullptr, outputs, rows, cols, nullptr, count};
    DirectionArgs direction{};
    direction.unscale = 1.0f;
    ProductArgs common{};
    common.a = a, common.b = b, common.c = c, common.out_dtype = out_dtype;
    return dispatch("hbt_orthogonalize", t, in_dtype, product_dtype, direction, common, steps, eps, workspace,
                    workspace_bytes, stream);
}

int32_t hbt_muon_step(void* const* params, const void* const* grads, float* const* momenta, const int64_t* rows,
                      const int64_t* cols, const float* scales, int32_t count, int32_t param_dtype, int32_t grad_dtype,
                      int32_t product_dtype, float unscale, const float* grad_mul, float momentum,
                      float one_minus_momentum, int32_t nesterov, int32_t steps, float a, float b, float c, double eps, float decay, float lr, const float* slot,
                      void* workspace, int64_t workspace_bytes, void* stream) {
    clear_error();
    const char* who = "hbt_muon_step";
    if (count > 0 && momenta == nullptr) return invalid(who, "a table is null");
    Matrices t{grads, momenta, params, rows, cols, scales, count};
    DirectionArgs direction{};
    direction.unscale = unscale, direction.grad_mul = grad_mul, direction.slot = slot;
    direction.momentum = momentum, direction.rest = one_minus_momentum, direction.nesterov = nesterov;
    ProductArgs common{};
    common.a = a, common.b = b, common.c = c, common.out_dtype = param_dtype, common.update = 1;
    common.decay = decay, common.lr = lr, common.slot = slot;
    return dispatch(who, t, grad_dtype, product_dtype, direction, common, steps, eps, workspace, workspace_bytes,
                    stream);
}

}  // extern "C"
