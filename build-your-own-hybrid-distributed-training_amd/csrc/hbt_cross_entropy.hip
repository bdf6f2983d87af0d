// Softmax cross entropy over a large vocabulary from hidden states, with its gradients, without
// the logits in memory.
//
//   z_iv = <x_i, W_v> + b_v;   lse_i = log sum_v exp z_iv
//   loss_i = lse_i - (1 - s) z_i,t(i) - (s / V) sum_v z_iv
//   dz_iv = c_i (exp(z_iv - lse_i) - (1 - s) [v = t(i)] - s / V);  dx = dz W;  dW = dz^T x
//
// The tokens that carry a loss are first gathered into consecutive rows: tokens without one cost
// nothing after that, and whatever their hidden states hold reaches no sum.
//
// The logits of a tile never leave the workgroup that forms them: it takes each row's largest and
// the sum of exp(z - largest) over its columns, and a row's tiles are joined afterwards.  For
// gradients the tile also stores exp(z - largest), which needs only 16 bits (fp16: 2^-11 of a value
// whose gradient is rounded by 2^-8 or 2^-11 next, or 2^-25 of the tile's largest; fp32 for fp32 tensors), for a piece of the rows
// at a time (at most kPieceBytes); one pass over a piece turns them into dz, rounded to the tensors' dtype
// for the matrix cores, and the two products follow.  So the logits are formed once, 6 T V D operations in
// all, where forming them again for the gradients would take 8.
//
// What a sum over pieces needs (dW, db) is carried in fp32.  A target is left out of its tile's largest
// and sum, and its exponential joins the others' in fp64, from its fp32 logit: both the loss and the gradient
// 1 - p of a nearly certain target are the others' sum, which fp32 or fp16 would round off beside a 1, and the
// other words' exponentials would be subnormal in fp16, or zero, beside the target's.
#include "hbt_matmul.hpp"

namespace hbt {
namespace mm {
namespace {

constexpr int F32 = HBT_DTYPE_F32, BF16 = HBT_DTYPE_BF16, F16 = HBT_DTYPE_F16;
constexpr int64_t kPieceBytes = int64_t(2) << 30;  // stored exponentials at a time
constexpr int64_t kStatsBytes = int64_t(1) << 28;  // row statistics at a time, without gradients
// The kernel for few tokens takes up to 16; each of its workgroups reads all of them, which tells past
// so many products: 4 x 4096 x 128256 take 199 us and in tiles 196, 2 tokens 191 and 198, 16 tokens 282 and
// 198, but 16 x 768 x 50257 (0.6e9) 26.5 and 30.7.
constexpr int kThin = 16;
constexpr int64_t kThinProducts = int64_t(1) << 31;
// Tokens from which on a 2-byte W with rows off 16 bytes is copied to rows on them first: its
// products then load straight into LDS, in tiles of 256.  50257 x 765 in bf16: 8192 tokens, evaluated,
// 1324 us without the copy and 641 with it, all gradients 3884 and 2291; 200 tokens 73 either way.  In
// fp32 the matrix cores are the bound and a copy gains nothing (2048 x 1001 x 32003: 3265 and 3185 us).
constexpr int64_t kPadTokens = 256;
constexpr int64_t kMostRows = kMaxLd;               // rows of a piece: a row of the turned hidden states
constexpr int64_t kMostTokens = int64_t(1) << 24;
constexpr int64_t kMostParts = 1024;               // tiles' sums of dx that a call has room for
constexpr float kLog2e = 1.44269504f;

// What the kernels of a call share.
struct Control {
    int32_t count;    // tokens that carry a loss
    float scale_in;   // multiplies dz before it is rounded: keeps fp16 in range
    float scale_out;  // multiplies the products
    int32_t splits;   // parts that the sums of dx are split into
};

// A row's statistics: the largest logit, 1 / sum of exp(z - largest), log p of its target and what
// multiplies its dz.  A target out of range makes the log p, and so the loss and the gradients, NaN.
struct Row {
    float top, inverse, log_p, weight;
};

// The rows of piece `piece` of `pieces`, of at most `most` rows each.
struct Piece {
    const Control* control;
    int piece, pieces;
};
__device__ __forceinline__ int rows_of_a_piece(int count, int pieces) {
    return ((count + pieces - 1) / pieces + 255) / 256 * 256;
}
__device__ __forceinline__ void piece_rows(const Piece& p, int& first, int& rows) {
    const int count = p.control->count, each = rows_of_a_piece(count, p.pieces);
    first = min(p.piece * each, count);
    rows = min(each, count - first);
}

// The largest over the wavefront, in every lane.
__device__ __forceinline__ float wave_max(float x) {
#pragma unroll
    for (int m = 32; m > 0; m >>= 1) x = fmaxf(x, __shfl_xor(x, m));
    return x;
}

// Statistics, and the exponentials under them, are in units of log(2) for 2-byte tensors: their
// logits are multiplied by log2(e) once and the hardware's base-2 exponential takes them (2^-23 or so
// off, far below what 16 bits keep).  fp32 tensors keep the natural unit and the accurate function.
template <int D>
__device__ __forceinline__ float in_units(float z) {
    if constexpr (D == F32) return z;
    else return z * kLog2e;
}
template <int D>
__device__ __forceinline__ float exponential(float t) {
    if constexpr (D == F32) return expf(t);
    else return __builtin_amdgcn_exp2f(t);
}
template <int D>
constexpr double unit() { return D == F32 ? 1.0 : 0.69314718055994531; }

// ---- the tokens that carry a loss ---------------------------------------------------------
// How the sums of dx may be split: tiles of `tile`, tiles_n across, and `steps` k-tiles each; a launch has
// workgroups and room for `most` parts, 0 if none is to be split.
struct SplitArgs {
    int64_t inner;
    int tile, tiles_n, steps, most, f32;
};

struct PrepareArgs {
    const int64_t* target;
    const float* token_grads;  // the loss's gradient for each token, or null for 1
    const float* factor;       // the loss's own gradient, or null for 1
    Control* control;
    int32_t* place;   // token -> row, -1 without a loss
    int32_t* token;   // row -> token
    int32_t* word;    // row -> target, -1 out of range
    float* weight;    // row -> gradient
    int64_t tokens, vocab, ignore;
    int mean, half, pieces;
    SplitArgs split;
};

// The split of dx's sums, by the estimate that chose its tile: only here is it known how many rows
// there are.  Lane s of a wavefront looks at s + 1 parts.  3001 tokens of which 1801 carry a loss, 1000 x 32003
// in fp16: 8 parts and 145 us with their join, where the 4 of 3001 tokens, and 6, take 215 and 172.
__device__ __forceinline__ int pick_splits(const SplitArgs& p, int rows, int lane) {
    if (p.most == 0) return 1;
    int splits = lane % 16 + 1;
    const int tiles = (rows + p.tile - 1) / p.tile * p.tiles_n;
    double cost = INFINITY;
    if (splits == 1 || (p.steps >= 4 * splits && tiles * splits <= p.most))
        cost = split_cost(p.tile, rows, p.inner, tiles, p.steps, splits, p.f32 != 0);
    for (int m = 1; m < 16; m <<= 1) {
        const double other = __shfl_xor(cost, m);
        const int others = __shfl_xor(splits, m);
        if (other < cost || (other == cost && others < splits)) cost = other, splits = others;
    }
    return splits;
}

// `top`: the largest magnitude of a token's gradient.  A wavefront.
__device__ __forceinline__ void write_control(const PrepareArgs& p, int count, float top, int lane) {
    const int splits = pick_splits(p.split, min(count, rows_of_a_piece(count, p.pieces)), lane);
    if (lane != 0) return;
    // fp16 values of dz: the largest gradient comes to 2^13 to 2^14, far from both ends of the
    // range; a power of two, so that nothing is rounded.
    float in = 1.0f;
    if (p.half && top > 0.0f && top < INFINITY) {
        int e = 0;
        frexpf(top, &e);
        in = ldexpf(1.0f, max(-126, min(126, 14 - e)));
    }
    p.control->count = count;
    p.control->splits = splits;
    p.control->scale_in = in;
    // No token carries a loss: no gradient, where 1 / 0 times a sum of nothing would be NaN.
    const float factor = p.factor != nullptr ? *p.factor : 1.0f;
    p.control->scale_out = count == 0 ? 0.0f : (p.mean ? factor / static_cast<float>(count) : factor) / in;
}
__device__ __forceinline__ void write_row(const PrepareArgs& p, int row, int64_t i, int64_t t, float weight) {
    p.token[row] = static_cast<int32_t>(i);
    p.word[row] = t >= 0 && t < p.vocab ? static_cast<int32_t>(t) : -1;
    p.weight[row] = weight;
}

// One workgroup: rows in the order of the tokens, 512 consecutive ones a wavefront at a time (8192: 8 us; a barrier for each 1024 of them took 14).
__global__ __launch_bounds__(1024) void prepare_kernel(PrepareArgs p) {
    constexpr int kEach = 8;
    __shared__ int wave_count[16];
    __shared__ float wave_top[16];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int count = 0;
    float top = 0.0f;
    for (int64_t base = 0; base < p.tokens; base += 1024 * kEach) {
        const int64_t first = base + wave * (64 * kEach) + lane;
        int64_t t[kEach];
        float g[kEach];
        uint64_t votes[kEach];
        int mine = 0;
#pragma unroll
        for (int k = 0; k < kEach; ++k) {
            const int64_t i = first + 64 * k;
            t[k] = i < p.tokens ? p.target[i] : p.ignore;
            g[k] = i < p.tokens && p.token_grads != nullptr ? p.token_grads[i] : 1.0f;
        }
#pragma unroll
        for (int k = 0; k < kEach; ++k) {
            votes[k] = __ballot(t[k] != p.ignore);
            mine += __popcll(votes[k]);
        }
        __syncthreads();
        if (lane == 0) wave_count[wave] = mine;
        __syncthreads();
        int row = count;
        for (int w = 0; w < 16; ++w) {
            if (w < wave) row += wave_count[w];
            count += wave_count[w];
        }
#pragma unroll
        for (int k = 0; k < kEach; ++k) {
            const int64_t i = first + 64 * k;
            const bool valid = (votes[k] >> lane) & 1;
            const int at = row + __popcll(votes[k] & ((uint64_t(1) << lane) - 1));
            if (valid) {
                write_row(p, at, i, t[k], g[k]);
                top = fmaxf(top, fabsf(g[k]));
            }
            if (i < p.tokens) p.place[i] = valid ? at : -1;
            row += __popcll(votes[k]);
        }
    }
    top = wave_max(top);
    if (lane == 0) wave_top[wave] = top;
    __syncthreads();
    if (wave != 0) return;
    for (int w = 1; w < 16; ++w) top = fmaxf(top, wave_top[w]);
    write_control(p, count, top, lane);
}

// `cols` elements from any boundary to a row of `ld`, zeros behind them; a wavefront.
template <int D>
__device__ __forceinline__ void copy_row(const char* from, char* to, int64_t cols, int64_t ld, int lane) {
    constexpr int E = unit_elems<D>(), B = elem_bytes<D>();
    for (int64_t j = lane * E; j < ld; j += 64 * E) {
        u32x4 v = {0, 0, 0, 0};
        if (j + E <= cols) {
            v = load16(from + j * B);
        } else {
#pragma unroll
            for (int e = 0; e < E - 1; ++e) {
                if (j + e >= cols) break;
                if constexpr (B == 4) v[e] = reinterpret_cast<const uint32_t*>(from)[j + e];
                else v[e / 2] |= static_cast<uint32_t>(reinterpret_cast<const uint16_t*>(from)[j + e]) << (16 * (e % 2));
            }
        }
        *reinterpret_cast<u32x4*>(to + j * B) = v;
    }
}

// A matrix whose rows are off 16 bytes, copied to rows that are not.
template <int D>
__global__ __launch_bounds__(256) void pad_kernel(const void* from, int64_t ld_from, void* to, int64_t ld, int64_t rows,
                                                  int64_t cols) {
    constexpr int B = elem_bytes<D>();
    const int64_t row = blockIdx.x * int64_t(4) + (threadIdx.x >> 6);
    if (row >= rows) return;
    copy_row<D>(static_cast<const char*>(from) + row * ld_from * B, static_cast<char*>(to) + row * ld * B, cols, ld,
                threadIdx.x & 63);
}

struct GatherArgs {
    const void* x;
    const int32_t* place;
    void* rows;   // [count][ld], zeros behind the inner size
    void* dx;     // zeros for the tokens without a loss, or null
    float* loss;  // the same, or null
    int64_t ldx, ld, lddx, tokens, inner;
    int dx_wide;  // dx in fp32
};

// The token's row of x to its place, or zeros where it carries no loss; a wavefront.
template <int D>
__device__ __forceinline__ void gather_token(const GatherArgs& p, int64_t token, int row, int lane) {
    constexpr int B = elem_bytes<D>();
    if (row >= 0) {
        copy_row<D>(static_cast<const char*>(p.x) + token * p.ldx * B, static_cast<char*>(p.rows) + row * p.ld * B, p.inner,
                    p.ld, lane);
        return;
    }
    if (p.loss != nullptr && lane == 0) p.loss[token] = 0.0f;
    if (p.dx == nullptr) return;
    if (p.dx_wide) {
        for (int64_t j = lane; j < p.inner; j += 64) store_elem<F32>(p.dx, token * p.lddx + j, 0.0f);
    } else {
        for (int64_t j = lane; j < p.inner; j += 64) store_elem<D>(p.dx, token * p.lddx + j, 0.0f);
    }
}
// A wavefront a token; 8192 x 4096 in bf16: 25 us (5.4 TB/s).
template <int D>
__global__ __launch_bounds__(256) void gather_kernel(GatherArgs p) {
    const int64_t token = blockIdx.x * int64_t(4) + (threadIdx.x >> 6);
    if (token < p.tokens) gather_token<D>(p, token, p.place[token], threadIdx.x & 63);
}

// Both of the above for at most kFewTokens tokens: a launch less, since every workgroup counts the
// rows before its own tokens from the targets.
constexpr int64_t kFewTokens = 2048;
template <int D>
__global__ __launch_bounds__(256) void prepare_few_kernel(PrepareArgs p, GatherArgs g) {
    __shared__ int wave_before[4], wave_count[4];
    __shared__ float wave_top[4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, first = blockIdx.x * 4, tokens = static_cast<int>(p.tokens);
    int before = 0, count = 0;  // of the wavefront's share: valid tokens before `first`, and all
    float top = 0.0f;
    for (int base = 0; base < tokens; base += 256) {
        const int i = base + static_cast<int>(threadIdx.x);
        const bool valid = i < tokens && p.target[i] != p.ignore;
        before += __popcll(__ballot(valid && i < first));
        count += __popcll(__ballot(valid));
        if (blockIdx.x == 0 && valid) top = fmaxf(top, p.token_grads != nullptr ? fabsf(p.token_grads[i]) : 1.0f);
    }
    if (blockIdx.x == 0) top = wave_max(top);
    if (lane == 0) wave_before[wave] = before, wave_count[wave] = count, wave_top[wave] = top;
    __syncthreads();
    if (blockIdx.x == 0 && wave == 0)
        write_control(p, (wave_count[0] + wave_count[1]) + (wave_count[2] + wave_count[3]),
                      fmaxf(fmaxf(wave_top[0], wave_top[1]), fmaxf(wave_top[2], wave_top[3])), lane);
    const int token = first + wave;
    if (token >= tokens) return;
    int row = (wave_before[0] + wave_before[1]) + (wave_before[2] + wave_before[3]);
    for (int i = first; i < token; ++i) row += p.target[i] != p.ignore;
    const int64_t t = p.target[token];
    if (t == p.ignore) row = -1;
    if (row >= 0 && lane == 0) write_row(p, row, token, t, p.token_grads != nullptr ? p.token_grads[token] : 1.0f);
    gather_token<D>(g, token, row, lane);
}

// ---- logits ---------------------------------------------------------------------------------
struct LogitArgs {
    const void* x;      // gathered rows
    const void* w;
    const void* bias;
    const int32_t* word;
    float2* stats;      // [tile][row of the piece]: largest, sum of the other words' exponentials than the target's
    float* sums;        // the same: sum of the logits, or null without smoothing
    float* target;      // row -> its target's logit
    void* kept;         // [row of the piece][ldk] exponentials, or null
    int64_t ldx, ldw, ldk, stride, inner;  // stride: rows of stats
    int64_t column, end;     // the words [column, end) of this launch, whose tiles are first_tile and on
    int tiles_n, first_tile;
    Piece piece;
};

// The larger, or the sum, of a value over the four quarters of a wavefront (lanes l % 16).
__device__ __forceinline__ float quarters_max(float x) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float quarters_sum(float x) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// Two registers of sixteen columns' neighbours: quarter q of a wavefront holds columns 4 q .. + 3 of the
// first sixteen in `a` and of the next sixteen in `b`; afterwards it holds columns 8 q .. + 3 of the
// thirty-two in `a` and 8 q + 4 .. + 7 in `b`.
__device__ __forceinline__ void pair_columns(uint32_t& a, uint32_t& b) {
    const auto half = __builtin_amdgcn_permlane32_swap(a, b, false, false);
    const auto row = __builtin_amdgcn_permlane16_swap(half[0], half[1], false, false);
    a = row[0], b = row[1];
}

// Tiles' logits to statistics and exponentials, in the registers that the matrix cores leave
// them in: lane l holds, of row l % 16 of each sixteen rows, four columns of each sixteen.  The
// largest of a row is taken in the lane, over the quarters, and over the wavefronts through LDS.
//
// A workgroup takes every gridDim.x-th tile.  With tiles of 256, of which a CU holds one, the grid is
// one workgroup a CU, and the first loads of its next tile are in flight while it reduces this one's logits
// (8192 x 768 x 50257: a workgroup a tile takes 7% more).
//
// Bound by the matrix cores: in bf16 8192 x 4096 x 128256 takes 6.86 ms with the exponentials (1.25
// PFLOP/s; the library's product alone 6.06), 8192 x 768 x 50257 763 us, 584 without them, an eighth
// of it the reduction.  Logits passed through LDS, a row a wavefront, take 14 to 16 us a tile more.
template <int D, class T, bool kAsync>
__global__ __launch_bounds__(T::kThreads, 2) void logit_kernel(LogitArgs p) {
    extern __shared__ __align__(16) char lds[];
    int first, count;
    piece_rows(p.piece, first, count);
    const int tiles_m = (count + T::BM - 1) / T::BM, total = tiles_m * p.tiles_n;
    int t = blockIdx.x;
    if (t >= total) return;
    // A thread's places are worked out anew for each tile: kept through the products, they would take
    // registers that those need.
    const auto thread = []() {
        int tid = threadIdx.x;
        asm volatile("" : "+v"(tid));
        return tid;
    };
    const auto row_of = [](int tid) { return (tid >> 6) / T::WN * (T::BM / T::WM) + (tid & 15); };
    const auto column_of = [](int tid) { return __builtin_amdgcn_readfirstlane(tid >> 6) % T::WN * (T::BN / T::WN); };
    const int32_t* words = p.word + first;
    const char* x = static_cast<const char*>(p.x) + first * p.ldx * elem_bytes<D>();
    float* line = reinterpret_cast<float*>(lds + lds_bytes<T, kAsync>());  // [3][WN][BM]: largest, two sums
    constexpr int kLine = T::WN * T::BM;
    TileProduct<D, true, true, T, kAsync> tile;
    int64_t m0, n0;
    int tn;
    int word[T::TM];        // the rows' targets, and once they have arrived a byte for each: the
    uint32_t places[2];     // target's column from the wavefront's first one, 255 outside of its columns
    static_assert(T::TM <= 8 && 16 * T::TN <= 255, "a byte a row");
    const auto begin = [&]() {
        int tm;
        // Tile rows in eights take 6825 and 748 us at the two sizes above, in fours 6753 and 755, in sixteens 7020 and 758.
        band_order<8>(xcd_tile(t, total), tiles_m, p.tiles_n, tm, tn);
        m0 = int64_t(tm) * T::BM, n0 = p.column + int64_t(tn) * T::BN;
        const int tid = thread();
        if (p.inner > 0) {
            tile.init(x, p.ldx, m0, count, p.w, p.ldw, n0, p.end, 0, p.inner, tid);
            tile.begin(lds);
        }
        const int wm = row_of(tid);
#pragma unroll
        for (int i = 0; i < T::TM; ++i) word[i] = words[min(static_cast<int>(m0) + wm + 16 * i, count - 1)];
    };
    const auto place = [&]() {
        const int wn = column_of(thread());
        places[0] = places[1] = 0;
#pragma unroll
        for (int i = 0; i < T::TM; ++i) {
            const int at = word[i] - static_cast<int>(n0) - wn;
            places[i / 4] |= (at >= 0 && at < 16 * T::TN ? static_cast<uint32_t>(at) : 255u) << (8 * (i % 4));
        }
    };
    f32x4 acc[T::TM][T::TN];
    begin();
    for (;;) {
        place();
        if (p.inner > 0) {
            tile.run(lds, acc);
        } else {
#pragma unroll
            for (int i = 0; i < T::TM; ++i)
#pragma unroll
                for (int j = 0; j < T::TN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
            __syncthreads();
        }
        const int64_t m = m0, n = n0;
        const int tid = thread(), q = (tid >> 4) & 3, wm = row_of(tid), wn = column_of(tid), slot = wn / (T::BN / T::WN) * T::BM + wm;
        const int rows = static_cast<int>(min<int64_t>(count - m, T::BM));
        const int left = static_cast<int>(p.end - n) - wn;  // columns from the wavefront's first one
        const int column = tn + p.first_tile;
        const uint32_t targets[2] = {places[0], places[1]};
        if (p.bias != nullptr) {
#pragma unroll
            for (int j = 0; j < T::TN; ++j) {
                const f32x4 b = load_row<D>(p.bias, n + wn + 16 * j + 4 * q, left - 16 * j - 4 * q);
#pragma unroll
                for (int i = 0; i < T::TM; ++i) acc[i][j] += b;
            }
        }
        t += gridDim.x;
        const bool more = T::BM == 256 && t < total;
        if (more) begin();
        if (p.sums != nullptr) {
#pragma unroll
            for (int i = 0; i < T::TM; ++i) {
                float sum = 0.0f;
#pragma unroll
                for (int j = 0; j < T::TN; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) sum += 16 * j + 4 * q + e < left ? acc[i][j][e] : 0.0f;
                sum = quarters_sum(sum);
                if (q == 0) line[2 * kLine + slot + 16 * i] = sum;
            }
        }
#pragma unroll
        for (int i = 0; i < T::TM; ++i)
#pragma unroll
            for (int j = 0; j < T::TN; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[i][j][e] = in_units<D>(acc[i][j][e]);
        if (left < 16 * T::TN) {  // past the last column
#pragma unroll
            for (int i = 0; i < T::TM; ++i)
#pragma unroll
                for (int j = 0; j < T::TN; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (16 * j + 4 * q + e >= left) acc[i][j][e] = -INFINITY;
        }
        // The target leaves before the largest is taken: far above the others, it would push their exponentials
        // under fp16's smallest.
#pragma unroll
        for (int i = 0; i < T::TM; ++i) {
            const int at = (targets[i / 4] >> (8 * (i % 4))) & 255;
            if (__builtin_expect(__any(at != 255), 0)) {  // seldom: a wavefront's columns are a small part of the vocabulary
                float z = 0.0f;
#pragma unroll
                for (int j = 0; j < T::TN; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (at == 16 * j + 4 * q + e) z = acc[i][j][e], acc[i][j][e] = -INFINITY;
                if (at != 255 && ((at >> 2) & 3) == q && wm + 16 * i < rows) p.target[first + m + wm + 16 * i] = z;
            }
        }
#pragma unroll
        for (int i = 0; i < T::TM; ++i) {
            float top = fmaxf(fmaxf(acc[i][0][0], acc[i][0][1]), fmaxf(acc[i][0][2], acc[i][0][3]));
#pragma unroll
            for (int j = 1; j < T::TN; ++j)
                top = fmaxf(top, fmaxf(fmaxf(acc[i][j][0], acc[i][j][1]), fmaxf(acc[i][j][2], acc[i][j][3])));
            top = quarters_max(top);
            if (q == 0) line[slot + 16 * i] = top;
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < T::TM; ++i) {
            float top = line[wm + 16 * i];
#pragma unroll
            for (int w = 1; w < T::WN; ++w) top = fmaxf(top, line[w * T::BM + wm + 16 * i]);
            if (top == -INFINITY) top = 0.0f;  // a tile of nothing but -inf
            float sum = 0.0f;
#pragma unroll
            for (int j = 0; j < T::TN; ++j) {
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[i][j][e] = exponential<D>(acc[i][j][e] - top);
                sum += (acc[i][j][0] + acc[i][j][1]) + (acc[i][j][2] + acc[i][j][3]);
            }
            sum = quarters_sum(sum);
            if (q == 0) line[kLine + slot + 16 * i] = sum;
            // Whole runs of the wavefront's columns lie inside a stored row, whose length is a multiple of 64.
            if (p.kept == nullptr || n + wn >= p.ldk) continue;
            const int64_t to = (m + wm + 16 * i) * p.ldk + n + wn;
            const bool in = wm + 16 * i < rows;
            if constexpr (D == F32) {
#pragma unroll
                for (int j = 0; j < T::TN; ++j)
                    if (in) *reinterpret_cast<f32x4*>(static_cast<float*>(p.kept) + to + 16 * j + 4 * q) = acc[i][j];
            } else {
                uint32_t h[T::TN][2];
#pragma unroll
                for (int j = 0; j < T::TN; ++j) {
                    h[j][0] = pack2_rounded<F16>(acc[i][j][0], acc[i][j][1]);
                    h[j][1] = pack2_rounded<F16>(acc[i][j][2], acc[i][j][3]);
                }
                uint16_t* kept = static_cast<uint16_t*>(p.kept) + to;
#pragma unroll
                for (int j = 0; j < T::TN; j += 2) {  // 64 bytes of a row a quarter: eight columns a lane
                    pair_columns(h[j][0], h[j + 1][0]);
                    pair_columns(h[j][1], h[j + 1][1]);
                    if (in) *reinterpret_cast<u32x4*>(kept + 16 * j + 8 * q) = u32x4{h[j][0], h[j][1], h[j + 1][0], h[j + 1][1]};
                }
            }
            __builtin_amdgcn_sched_barrier(0);  // a row at a time: mixed, they do not fit the registers
        }
        __syncthreads();
        for (int i = threadIdx.x; i < rows; i += T::kThreads) {
            float top = line[i], sum = line[kLine + i];
#pragma unroll
            for (int w = 1; w < T::WN; ++w) top = fmaxf(top, line[w * T::BM + i]), sum += line[kLine + w * T::BM + i];
            p.stats[column * p.stride + m + i] = make_float2(top, sum);
            if (p.sums != nullptr) {
                float logits = line[2 * kLine + i];
#pragma unroll
                for (int w = 1; w < T::WN; ++w) logits += line[2 * kLine + w * T::BM + i];
                p.sums[column * p.stride + m + i] = logits;
            }
        }
        if (!more) return;
        // A barrier above lies between this and the next tile's writes of the lines.
    }
}

// At most 16 tokens, without gradients: the read of W.  A workgroup of 8 waves forms 16 logits of
// every token as the linear layer's thin kernel does, and their statistics.  1 x 4096 x 128256 in
// bf16 takes 175 to 180 us (5.8 to 6.0 TB/s), 183 to 188 with the join; two or four groups of 16 a workgroup 215 and 191.
template <int D>
__global__ __launch_bounds__(512) void thin_logit_kernel(const void* x_, int64_t ldx, const void* w_, int64_t ldw,
                                                         const void* bias, const int64_t* target, int tokens,
                                                         int64_t vocab, int64_t inner, float2* stats, float* sums,
                                                         float* target_logit) {
    constexpr int E = unit_elems<D>(), kStep = 4 * E, kWaves = 8, kUnrolled = 4, B = elem_bytes<D>();
    __shared__ f32x4 parts[kWaves][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, row = lane & 15, q = lane >> 4;
    const int64_t n0 = int64_t(blockIdx.x) * 16;
    const bool w_in = n0 + row < vocab, x_in = row < tokens;
    const char* w = static_cast<const char*>(w_) + ((n0 + (w_in ? row : 0)) * ldw + q * E) * B;
    const char* x = static_cast<const char*>(x_) + ((x_in ? row : 0) * ldx + q * E) * B;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    const int64_t whole = inner / kStep;
    int64_t s = wave * kUnrolled;
    for (; s + kUnrolled <= whole; s += kUnrolled * kWaves) {
        u32x4 fw[kUnrolled], fx[kUnrolled];
#pragma unroll
        for (int i = 0; i < kUnrolled; ++i) {
            fw[i] = load16(w + (s + i) * kStep * B);
            fx[i] = load16(x + (s + i) * kStep * B);
        }
#pragma unroll
        for (int i = 0; i < kUnrolled; ++i) acc = mma<D>(fw[i], fx[i], acc);
    }
    for (; s < whole; ++s) acc = mma<D>(load16(w + s * kStep * B), load16(x + s * kStep * B), acc);
    if (wave == whole % kWaves && whole * kStep < inner) {  // the last, partial step
        u32x4 fw = {0, 0, 0, 0}, fx = {0, 0, 0, 0};
        const int64_t at = whole * kStep;
        for (int e = 0; e < E; ++e) {
            if (at + q * E + e >= inner) break;
            if constexpr (B == 4) {
                fw[e] = reinterpret_cast<const uint32_t*>(w)[at + e];
                fx[e] = reinterpret_cast<const uint32_t*>(x)[at + e];
            } else {
                fw[e / 2] |= uint32_t(reinterpret_cast<const uint16_t*>(w)[at + e]) << (16 * (e % 2));
                fx[e / 2] |= uint32_t(reinterpret_cast<const uint16_t*>(x)[at + e]) << (16 * (e % 2));
            }
        }
        acc = mma<D>(fw, fx, acc);
    }
    parts[wave][lane] = acc;
    __syncthreads();
    if (wave != 0) return;
#pragma unroll
    for (int i = 1; i < kWaves; ++i) acc += parts[i][lane];
    // The lane holds logits n0 + 4 q .. + 3 of token `row`.
    const int64_t n = n0 + 4 * q;
    const int have = static_cast<int>(min<int64_t>(vocab - n, 4));
    if (bias != nullptr) acc += load_row<D>(bias, n, have);
    const int64_t at = x_in ? target[row] - n : -1;
    float sum = 0.0f, top = -INFINITY;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if (e < have) sum += acc[e];
        acc[e] = e < have ? in_units<D>(acc[e]) : -INFINITY;
        if (at == e && e < have) target_logit[row] = acc[e], acc[e] = -INFINITY;
        top = fmaxf(top, acc[e]);
    }
    top = fmaxf(top, __shfl_xor(top, 16));
    top = fmaxf(top, __shfl_xor(top, 32));
    const float base = top == -INFINITY ? 0.0f : top;
    float part = 0.0f;
#pragma unroll
    for (int e = 0; e < 4; ++e) part += exponential<D>(acc[e] - base);
    part += __shfl_xor(part, 16);
    part += __shfl_xor(part, 32);
    sum += __shfl_xor(sum, 16);
    sum += __shfl_xor(sum, 32);
    if (x_in && q == 0) {
        stats[row * int64_t(gridDim.x) + blockIdx.x] = make_float2(top, part);
        if (sums != nullptr) sums[row * int64_t(gridDim.x) + blockIdx.x] = sum;
    }
}

// ---- a row's tiles joined ----------------------------------------------------------------
struct JoinArgs {
    const float2* stats;
    const float* sums;
    const float* target;       // row -> target's logit
    const int32_t* word;       // row -> target, or null: `raw` names it
    const int32_t* token;      // row -> token, or null: the same
    const float* weight;       // row -> gradient, or null
    const int64_t* raw;        // token -> target, without gathered rows
    Row* row;                  // for the gradients, or null
    float* loss;               // token -> loss, or null
    double* row_loss;          // row -> loss, or null
    int64_t ignore, vocab, stride;
    double unit;               // of the largest and the targets' logits
    int tiles;
    float smoothing;
    Piece piece;
};

// A running log-sum: the largest so far and the sum of exponentials over it.  An empty tile (sum 0)
// adds nothing, a NaN sum stays one.
struct Running {
    float top = -INFINITY;
    double sum = 0.0;
    __device__ __forceinline__ void add(float t, double s, float unit) {
        if (s == 0.0) return;
        const float high = fmaxf(top, t);
        sum = (sum == 0.0 ? 0.0 : sum * expf((top - high) * unit)) + s * expf((t - high) * unit);
        top = high;
    }
};

__device__ __forceinline__ void finish_row(const JoinArgs& p, int row, Running r, double logits) {
    const int64_t token = p.token != nullptr ? p.token[row] : row;
    bool known;
    if (p.word != nullptr) {
        known = p.word[row] >= 0;
    } else {
        const int64_t t = p.raw[token];
        if (t == p.ignore) {
            if (p.loss != nullptr) p.loss[token] = 0.0f;
            if (p.row_loss != nullptr) p.row_loss[row] = 0.0;
            return;
        }
        known = t >= 0 && t < p.vocab;
    }
    const float unit = static_cast<float>(p.unit), z = known ? p.target[row] : NAN;
    const Running others = r;
    if (known) r.add(z, 1.0, unit);
    const double log_sum = log(r.sum);
    double log_p = (static_cast<double>(z) - r.top) * p.unit - log_sum;
    if (z >= others.top && fabsf(z) < INFINITY)  // the others beside a 1, which would round them off
        log_p = others.sum == 0.0 ? 0.0 : -log1p(others.sum * expf((others.top - z) * unit));
    double loss = -(1.0 - p.smoothing) * log_p;
    if (p.smoothing != 0.0f) loss += p.smoothing * ((r.top * p.unit + log_sum) - logits / static_cast<double>(p.vocab));
    if (p.loss != nullptr) p.loss[token] = static_cast<float>(loss);
    if (p.row_loss != nullptr) p.row_loss[row] = loss;
    if (p.row != nullptr)
        p.row[row] = Row{r.top, static_cast<float>(1.0 / r.sum), static_cast<float>(log_p),
                         p.weight[row] * p.piece.control->scale_in};
}

// Statistics [tile][row]: a workgroup joins 16 rows, 128 bytes of a tile's; its 32 groups of 16 lanes
// take tiles in turn.  8192 rows of 501 tiles: 15 us, where 64 rows a workgroup take 26.
constexpr int kJoinRows = 16, kJoinGroups = 32;
__global__ __launch_bounds__(kJoinRows * kJoinGroups) void join_kernel(JoinArgs p) {
    __shared__ float tops[kJoinGroups][kJoinRows];
    __shared__ double totals[kJoinGroups][kJoinRows], logit_sums[kJoinGroups][kJoinRows];
    int first, count;
    piece_rows(p.piece, first, count);
    if (static_cast<int>(blockIdx.x) * kJoinRows >= count) return;
    const int lane = threadIdx.x % kJoinRows, group = threadIdx.x / kJoinRows;
    const int i = blockIdx.x * kJoinRows + lane, at = min(i, count - 1);
    const float unit = static_cast<float>(p.unit);
    Running r;
    double logits = 0.0;
    for (int t = group; t < p.tiles; t += 4 * kJoinGroups) {
        float2 s[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {  // four loads in flight
            const int tile = t + k * kJoinGroups;
            s[k] = tile < p.tiles ? p.stats[tile * p.stride + at] : make_float2(0.0f, 0.0f);
            if (p.sums != nullptr && tile < p.tiles) logits += p.sums[tile * p.stride + at];
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) r.add(s[k].x, s[k].y, unit);
    }
    for (int half = kJoinGroups / 2; half > 0; half >>= 1) {
        tops[group][lane] = r.top, totals[group][lane] = r.sum, logit_sums[group][lane] = logits;
        __syncthreads();
        if (group < half) {
            r.add(tops[group + half][lane], totals[group + half][lane], unit);
            logits += logit_sums[group + half][lane];
        }
        __syncthreads();
    }
    if (group == 0 && i < count) finish_row(p, first + i, r, logits);
}

// Statistics [row][tile], many tiles and few rows: a workgroup a row, its lanes' parts joined in a tree
// (8016 tiles: 9 us, where 256 lanes take 25).
__global__ __launch_bounds__(1024) void thin_join_kernel(JoinArgs p) {
    __shared__ float tops[1024];
    __shared__ double totals[1024], logit_sums[1024];
    const int row = blockIdx.x, tid = threadIdx.x;
    const float unit = static_cast<float>(p.unit);
    Running r;
    double logits = 0.0;
    for (int t = tid; t < p.tiles; t += 4096) {
        float2 s[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int tile = t + k * 1024;
            s[k] = tile < p.tiles ? p.stats[row * p.stride + tile] : make_float2(0.0f, 0.0f);
            if (p.sums != nullptr && tile < p.tiles) logits += p.sums[row * p.stride + tile];
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) r.add(s[k].x, s[k].y, unit);
    }
    tops[tid] = r.top, totals[tid] = r.sum, logit_sums[tid] = logits;
    for (int half = 512; half > 0; half >>= 1) {
        __syncthreads();
        if (tid < half) {
            r.add(tops[tid + half], totals[tid + half], unit);
            logits += logit_sums[tid + half];
            tops[tid] = r.top, totals[tid] = r.sum, logit_sums[tid] = logits;
        }
    }
    if (tid == 0) finish_row(p, row, r, logits);
}

// The rows' losses added up in a fixed order; `divide`: their mean (0 / 0 without any).
__global__ __launch_bounds__(1024) void total_kernel(const double* row_loss, const Control* control,
                                                     const int64_t* raw, int64_t ignore, int64_t rows, int divide,
                                                     float* loss) {
    const int64_t count = control != nullptr ? control->count : rows;
    double sum = 0.0, valid = 0.0;
    for (int64_t i = threadIdx.x; i < count; i += 1024) {
        sum += row_loss[i];
        if (raw == nullptr || raw[i] != ignore) valid += 1.0;
    }
    sum = block_sum<1024>(sum);
    __syncthreads();
    valid = block_sum<1024>(valid);
    if (threadIdx.x == 0) loss[0] = static_cast<float>(divide ? sum / valid : sum);
}

// ---- hidden states with the tokens along a row ---------------------------------------------
// A dW in tiles of 256 reads its piece's hidden states so: of its operands, dz and x, both lie with the
// sum's index down the columns, and the transposing reads from LDS that this takes are slower than straight ones:
// dW at 8192 x 4096 x 128256 6970 us and 27 for this copy, 7290 without; at 8192 x 768 x 50257 551, 7 and 580.
// 64 x 64 values a workgroup; the tokens are filled up with zeros to a multiple of 64, of which the k-tiles are made.
struct TurnArgs {
    const uint16_t* rows;
    uint16_t* turned;    // [inner][ldt]
    int64_t ld, ldt, inner;
    Piece piece;
};
__device__ __forceinline__ int whole_tiles(int count) { return (count + 63) / 64 * 64; }
__global__ __launch_bounds__(256) void turn_kernel(TurnArgs p) {
    constexpr int kStride = 33;  // words of a row: a column's values fall on distinct banks
    __shared__ uint32_t tile[64 * kStride];
    int first, count;
    piece_rows(p.piece, first, count);
    const int r0 = blockIdx.x * 64, c0 = blockIdx.y * 64;
    if (r0 >= count) return;
    for (int u = threadIdx.x; u < 512; u += 256) {
        const int r = u / 8, at = u % 8;
        u32x4 v = {0, 0, 0, 0};  // rows end in zeros, at a multiple of 64
        if (r0 + r < count) v = *reinterpret_cast<const u32x4*>(p.rows + (first + r0 + r) * p.ld + c0 + at * 8);
#pragma unroll
        for (int e = 0; e < 4; ++e) tile[r * kStride + at * 4 + e] = v[e];
    }
    __syncthreads();
    for (int u = threadIdx.x; u < 512; u += 256) {
        const int c = u / 8, at = u % 8;
        if (c0 + c >= p.inner) break;
        u32x4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const uint32_t* word = tile + (at * 8 + 2 * e) * kStride + c / 2;
            const int shift = c % 2 * 16;
            v[e] = ((word[0] >> shift) & 0xFFFFu) | ((word[kStride] >> shift) << 16);
        }
        *reinterpret_cast<u32x4*>(p.turned + (c0 + c) * p.ldt + r0 + at * 8) = v;
    }
}

// ---- exponentials to dz, in place ----------------------------------------------------------
struct SoftmaxArgs {
    void* kept;
    const float2* stats;
    const Row* row;
    const int32_t* word;
    int64_t ldk, vocab, stride;
    int64_t cut;  // the words before it are in tiles of `tile` columns, the others in tiles of `last`
    int tile, last;
    float smoothing;
    const double* row_loss;
    float* loss;  // the call's, of which the first workgroup takes the sum, or null
    int mean;
    int whole;    // the rows are filled up with zeros to a multiple of 64
    Piece piece;
};

// Up to so many tokens the losses are added up beside the pass that follows them, a launch less (777 x 501
// x 5003 in fp32: 175 us for 178); by one workgroup of 256 more would outlast it.
constexpr int64_t kTotalTokens = 16384;
constexpr int kSoftmaxUnits = 2;  // 16-byte units a lane
// Bound by memory: a read and a write of 2 bytes (fp32: 4) an element, 8192 x 128256 in bf16 in 741 us
// (5.6 TB/s), 8192 x 50257 in 293.  Two units a lane, read past the caches: as they are written 780 and 307;
// four in a loop 815 and 317; one 710 and 315, but 52 for 44 where two fifths of the rows are none.
template <int D>
__global__ __launch_bounds__(256) void softmax_kernel(SoftmaxArgs p) {
    constexpr int E = unit_elems<D>(), B = elem_bytes<D>(), S = D == F32 ? F32 : F16;
    int block = blockIdx.x;
    if (p.loss != nullptr) {
        if (block == 0) {
            double sum = 0.0;
            const int rows = p.piece.control->count;
            for (int i = threadIdx.x; i < rows; i += 256) sum += p.row_loss[i];
            sum = block_sum<256>(sum);
            if (threadIdx.x == 0) p.loss[0] = static_cast<float>(p.mean ? sum / rows : sum);
            return;
        }
        --block;
    }
    int first, count;
    piece_rows(p.piece, first, count);
    constexpr int kSegment = 256 * kSoftmaxUnits * E;  // words a workgroup takes
    const int segments = static_cast<int>((p.ldk + kSegment - 1) / kSegment);
    const int i = block / segments, part = block % segments;
    char* line = static_cast<char*>(p.kept) + int64_t(i) * p.ldk * B;
    const int64_t first_word = (int64_t(part) * 256 * kSoftmaxUnits + threadIdx.x) * E;
    if (i >= count) {
        if (!p.whole || i >= whole_tiles(count)) return;
#pragma unroll
        for (int u = 0; u < kSoftmaxUnits; ++u) {
            const int64_t j = first_word + u * 256 * E;
            if (j < p.ldk) *reinterpret_cast<u32x4*>(line + j * B) = u32x4{0, 0, 0, 0};
        }
        return;
    }
    const Row row = p.row[first + i];
    const int word = p.word[first + i];
    const float even = p.smoothing / static_cast<float>(p.vocab) * row.weight;
    const float hit = (expm1f(row.log_p) + p.smoothing) * row.weight - even;
    const bool known = word >= 0;
    const float2* stats = p.stats + i;
    u32x4 units[kSoftmaxUnits];
#pragma unroll
    for (int u = 0; u < kSoftmaxUnits; ++u) {
        const int64_t j = first_word + u * 256 * E;
        if (j < p.ldk) units[u] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(line + j * B));
    }
#pragma unroll
    for (int u = 0; u < kSoftmaxUnits; ++u) {
        const int64_t j = first_word + u * 256 * E;
        if (j >= p.ldk) break;
        const int64_t word_at = min<int64_t>(j, p.vocab - 1);
        const int64_t at = word_at < p.cut ? word_at / p.tile : p.cut / p.tile + (word_at - p.cut) / p.last;
        const float factor = exponential<D>(stats[at * p.stride].x - row.top) * row.inverse * row.weight;
        float v[E];
#pragma unroll
        for (int e = 0; e < E; ++e) {
            v[e] = element<S>(units[u], e) * factor - even;
            if (j + e == word) v[e] = hit;
            if (!known) v[e] = NAN;
            if (j + e >= p.vocab) v[e] = 0.0f;
        }
#pragma unroll
        for (int e = 0; e < E; e += 4) store4<D>(line, j + e, f32x4{v[e], v[e + 1], v[e + 2], v[e + 3]});
    }
}

// ---- the gradients' products ---------------------------------------------------------------
struct GradArgs {
    const void* a;
    const void* b;
    const float* before;   // sums of the earlier pieces, or null
    void* y;
    const int32_t* token;  // y's row for a row of the piece, or null: its own
    float* partial;        // [splits][m][ldp]
    int64_t lda, ldb, ldy, ldbefore, ldp, m, n, k, m_in, n_in;  // m_in, n_in: rows that the operands hold
    int tiles_n, splits;   // splits: of dW, those of dx are the call's control's
    Piece piece;
};

// y = a b (dx: the rows of a are the piece's; dW: the sum runs over them, kTurned along b's rows), times the
// call's scale.
template <int D, int OD, bool kRows>
struct GradEpilogue {
    const GradArgs& p;
    float scale;
    int first;
    __device__ __forceinline__ f32x4 before(int64_t i, int64_t j, int have) const {
        return p.before == nullptr ? f32x4{0.f, 0.f, 0.f, 0.f} : load_row<F32>(p.before, i * p.ldbefore + j, have);
    }
    __device__ __forceinline__ void store(int64_t i, int64_t j, int have, f32x4 v, f32x4 before) const {
        v = v * scale + before;
        const int64_t row = kRows ? p.token[first + i] : i;
        store_row<OD>(p.y, row * p.ldy + j, have, v);
    }
};

// Bound by the matrix cores: at 8192 x 4096 x 128256 in bf16 dx takes 6.66 ms (1.29 PFLOP/s; the
// library 6.54) and dW 7.09 (1.21; the library 7.58).
template <int D, int OD, bool kRows, bool kTurned, class T, bool kAsync>
__global__ __launch_bounds__(T::kThreads, 2) void grad_kernel(GradArgs p) {
    extern __shared__ __align__(16) char lds[];
    int first, count;
    piece_rows(p.piece, first, count);
    const int64_t m = kRows ? count : p.m, k = kRows ? p.k : kTurned ? whole_tiles(count) : count;
    const int tiles_m = static_cast<int>((m + T::BM - 1) / T::BM), splits = kRows ? p.piece.control->splits : p.splits;
    const int total = tiles_m * p.tiles_n, split = total > 0 ? static_cast<int>(blockIdx.x) / total : splits;
    int tm, tn;
    if (split >= splits) return;
    // Tile rows walked together, in us (8192 x 4096 x 128256, 8192 x 768 x 50257): dW in twos 7120 and 552, in
    // fours 7175 and 556, in eights 7420 and 560; dx in fours 6540 and 586, in eights 6455 and 600, 1801 x 1000 x 32003
    // 138 and 133.
    const int at = xcd_tile(static_cast<int>(blockIdx.x) - split * total, total);
    if (!kRows) band_order<2>(at, tiles_m, p.tiles_n, tm, tn);
    else if (p.tiles_n < 4) band_order<4>(at, tiles_m, p.tiles_n, tm, tn);
    else band_order<8>(at, tiles_m, p.tiles_n, tm, tn);
    const int64_t m0 = int64_t(tm) * T::BM, n0 = int64_t(tn) * T::BN;
    constexpr int BK = tile_k<D>();
    const int64_t part = ((k + splits - 1) / splits + BK - 1) / BK * BK;
    const int64_t k0 = min<int64_t>(k, split * part), k1 = min<int64_t>(k, k0 + part);
    f32x4 acc[T::TM][T::TN];
    const char* b = static_cast<const char*>(p.b) + (kRows || kTurned ? 0 : first * p.ldb * elem_bytes<D>());
    tile_product<D, kRows, kTurned, T, kAsync>(p.a, p.lda, m0, kRows ? m : p.m_in, b, p.ldb, n0, p.n_in, k0, k1, lds, acc);
    const int rows = static_cast<int>(min<int64_t>(m - m0, T::BM)), cols = static_cast<int>(min<int64_t>(p.n - n0, T::BN));
    const GradEpilogue<D, OD, kRows> tile{p, p.piece.control->scale_out, first};
    float* partial = splits == 1 ? nullptr : p.partial + (split * m + m0) * p.ldp + n0;
    finish_tile<T, kAsync, 2>(
        lds, acc,
        [&](int i, int j) {
            return i < rows && j < cols && partial == nullptr ? tile.before(m0 + i, n0 + j, cols - j)
                                                              : f32x4{0.f, 0.f, 0.f, 0.f};
        },
        [&](int i, int j, f32x4 v, f32x4 before) {
            if (i >= rows || j >= cols) return v;
            if (partial != nullptr) *reinterpret_cast<f32x4*>(partial + i * p.ldp + j) = v;
            else tile.store(m0 + i, n0 + j, cols - j, v, before);
            return v;
        });
}

// Joins the parts of a split sum, in their order.
template <int D, int OD, bool kRows>
__global__ __launch_bounds__(256) void grad_join_kernel(GradArgs p) {
    int first, count;
    piece_rows(p.piece, first, count);
    const int64_t m = kRows ? count : p.m, units = p.ldp / 4, total = m * units;
    const int splits = kRows ? p.piece.control->splits : p.splits;
    if (splits == 1) return;
    const GradEpilogue<D, OD, kRows> tile{p, p.piece.control->scale_out, first};
    for (int64_t u = blockIdx.x * int64_t(256) + threadIdx.x; u < total; u += int64_t(gridDim.x) * 256) {
        const int64_t i = u / units, j = u % units * 4;
        f32x4 v = *reinterpret_cast<const f32x4*>(p.partial + i * p.ldp + j);
        for (int s = 1; s < splits; ++s) v += *reinterpret_cast<const f32x4*>(p.partial + (s * m + i) * p.ldp + j);
        const int have = static_cast<int>(min<int64_t>(p.n - j, 4));
        tile.store(i, j, have, v, tile.before(i, j, have));
    }
}

// ---- the bias gradient: column sums of dz ------------------------------------------------
// Bound by memory: 1801 x 32003 in fp16 24 us and 5 for the join (4.8 TB/s).
constexpr int kBiasBlocks = 64;  // parts that the rows of a piece are summed in
template <int D>
__global__ __launch_bounds__(256) void bias_part_kernel(const void* dz, int64_t ld, int64_t vocab, float* parts,
                                                        Piece piece) {
    int first, count;
    piece_rows(piece, first, count);
    const int64_t j = blockIdx.x * int64_t(256) + threadIdx.x;
    if (j >= vocab) return;
    const int each = (count + kBiasBlocks - 1) / kBiasBlocks, from = blockIdx.y * each, to = min(count, from + each);
    float sum = 0.0f;
#pragma unroll 4
    for (int i = from; i < to; ++i) sum += load_elem<D>(dz, i * ld + j);
    parts[blockIdx.y * vocab + j] = sum;
}
// The parts in order, and the earlier pieces' sum; the last piece rounds it to `db`.
template <int OD>
__global__ __launch_bounds__(256) void bias_join_kernel(const float* parts, float* sums, void* db, int64_t vocab,
                                                        Piece piece) {
    const int64_t j = blockIdx.x * int64_t(256) + threadIdx.x;
    if (j >= vocab) return;
    float sum = 0.0f;
    for (int b = 0; b < kBiasBlocks; ++b) sum += parts[b * vocab + j];
    sum *= piece.control->scale_out;
    if (piece.piece > 0) sum += sums[j];
    if (piece.piece + 1 < piece.pieces) sums[j] = sum;
    else store_elem<OD>(db, j, sum);
}

// ---- small calls --------------------------------------------------------------------------
// Few tokens of a small model over a small vocabulary are launch latency: one workgroup does all of
// a call in LDS, in fp32, where the kernels above are ten launches (16 x 32 x 97 with a bias: 11 us on
// the device; forward and backward by the host's clock 62 to 112, where eleven launches took 156).
constexpr int kSmallTokens = 64, kSmallLds = 128 << 10;
constexpr int64_t kSmallProduct = int64_t(1) << 17;  // multiplications of each product
int64_t small_lds(int64_t tokens, int64_t inner, int64_t vocab) {
    return 4 * (tokens * (inner + 1) + vocab * (inner + 1) + tokens * (vocab + 1));
}
bool is_small(int64_t tokens, int64_t inner, int64_t vocab) {
    return tokens <= kSmallTokens && tokens * inner * vocab <= kSmallProduct && small_lds(tokens, inner, vocab) <= kSmallLds;
}

struct SmallArgs {
    const void *x, *w, *bias;
    const int64_t* target;
    const float *token_grads, *factor;
    float* loss;
    void *dx, *dw, *db;
    int64_t ldx, ldw, lddx, lddw, ignore;
    int tokens, inner, vocab, reduction;
    float smoothing;
};

template <int D, int OD>
__global__ __launch_bounds__(1024) void small_kernel(SmallArgs p) {
    extern __shared__ __align__(16) char lds[];
    __shared__ double losses[kSmallTokens];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, across = p.inner + 1, wide = p.vocab + 1;
    float* x = reinterpret_cast<float*>(lds);   // [tokens][across], zeros for a token without a loss
    float* w = x + p.tokens * across;           // [vocab][across]
    float* z = w + p.vocab * across;            // [tokens][wide]: logits, then dz
    const int64_t mine = lane < p.tokens ? p.target[lane] : p.ignore;  // every wavefront has all targets
    const uint64_t valid = __ballot(mine != p.ignore);
    const int count = __popcll(valid);
    for (int i = tid; i < p.tokens * p.inner; i += 1024) {
        const int t = i / p.inner, k = i % p.inner;
        x[t * across + k] = (valid >> t) & 1 ? load_elem<D>(p.x, t * p.ldx + k) : 0.0f;
    }
    for (int i = tid; i < p.vocab * p.inner; i += 1024) {
        const int v = i / p.inner, k = i % p.inner;
        w[v * across + k] = load_elem<D>(p.w, v * p.ldw + k);
    }
    __syncthreads();
    for (int i = tid; i < p.tokens * p.vocab; i += 1024) {
        const int t = i / p.vocab, v = i % p.vocab;
        float sum = 0.0f;
        for (int k = 0; k < p.inner; ++k) sum = fmaf(x[t * across + k], w[v * across + k], sum);
        z[t * wide + v] = p.bias != nullptr ? sum + load_elem<D>(p.bias, v) : sum;
    }
    __syncthreads();
    const float even = p.smoothing / static_cast<float>(p.vocab);
    for (int t = wave; t < p.tokens; t += 16) {  // a wavefront a row
        float* row = z + t * wide;
        if (((valid >> t) & 1) == 0) {
            if (lane == 0) losses[t] = 0.0;
            for (int v = lane; v < p.vocab; v += 64) row[v] = 0.0f;
            continue;
        }
        const int64_t word = __shfl(mine, t);
        const bool known = word >= 0 && word < p.vocab;
        float top = -INFINITY;
        for (int v = lane; v < p.vocab; v += 64) top = fmaxf(top, row[v]);
        top = wave_max(top);
        if (top == -INFINITY) top = 0.0f;
        const float z_t = known ? row[word] : NAN;
        double others = 0.0, logits = 0.0;  // without the target's exponential, which would round them off
        for (int v = lane; v < p.vocab; v += 64) others += v == word ? 0.0f : expf(row[v] - top), logits += row[v];
        others = wave_sum(others), logits = wave_sum(logits);
        const double sum = known ? others + expf(z_t - top) : others, log_sum = log(sum);
        const double log_p = z_t == top && top < INFINITY ? -log1p(others) : (static_cast<double>(z_t) - top) - log_sum;
        if (lane == 0) {
            losses[t] = -(1.0 - p.smoothing) * log_p;
            if (p.smoothing != 0.0f) losses[t] += p.smoothing * ((top + log_sum) - logits / p.vocab);
        }
        const float weight = p.token_grads != nullptr ? p.token_grads[t] : 1.0f, inverse = static_cast<float>(1.0 / sum);
        const float missing = expm1f(static_cast<float>(log_p)) + p.smoothing;
        for (int v = lane; v < p.vocab; v += 64) {
            const float part = v == word ? missing : expf(row[v] - top) * inverse;
            row[v] = known ? (part - even) * weight : NAN;
        }
    }
    __syncthreads();
    const bool mean = p.reduction == HBT_LOSS_MEAN;
    if (p.loss != nullptr) {
        if (p.reduction == HBT_LOSS_NONE) {
            if (tid < p.tokens) p.loss[tid] = static_cast<float>(losses[tid]);
        } else if (wave == 0) {
            const double sum = wave_sum(lane < p.tokens ? losses[lane] : 0.0);
            if (lane == 0) p.loss[0] = static_cast<float>(mean ? sum / count : sum);
        }
    }
    const float factor = p.factor != nullptr ? *p.factor : 1.0f;
    const float scale = count == 0 ? 0.0f : (mean ? factor / static_cast<float>(count) : factor);
    if (p.dx != nullptr)
        for (int i = tid; i < p.tokens * p.inner; i += 1024) {
            const int t = i / p.inner, k = i % p.inner;
            float sum = 0.0f;
            if ((valid >> t) & 1)
                for (int v = 0; v < p.vocab; ++v) sum = fmaf(z[t * wide + v], w[v * across + k], sum);
            store_elem<OD>(p.dx, t * p.lddx + k, sum * scale);
        }
    if (p.dw != nullptr)
        for (int i = tid; i < p.vocab * p.inner; i += 1024) {
            const int v = i / p.inner, k = i % p.inner;
            float sum = 0.0f;
            for (int t = 0; t < p.tokens; ++t) sum = fmaf(z[t * wide + v], x[t * across + k], sum);
            store_elem<OD>(p.dw, v * p.lddw + k, sum * scale);
        }
    if (p.db != nullptr)
        for (int v = tid; v < p.vocab; v += 1024) {
            float sum = 0.0f;
            for (int t = 0; t < p.tokens; ++t) sum += z[t * wide + v];
            store_elem<OD>(p.db, v, sum * scale);
        }
}

// ---- the loss's own gradient -----------------------------------------------------------------
struct ScaleArgs {
    const void* src[HBT_MAX_SCALED];
    void* dst[HBT_MAX_SCALED];
    int64_t n[HBT_MAX_SCALED];
    int count;
    const float* factor;
};
// In place (SD == OD) nothing is to be done for a factor of 1, which is known on the device alone:
// the workgroups are few and walk the tensors, so that such a launch ends at once (525 million bf16
// elements: 3 us, where a workgroup for each 1024 elements takes 230).
template <int SD, int OD>
__global__ __launch_bounds__(256) void scale_round_kernel(ScaleArgs p) {
    const float f = *p.factor;
    if (SD == OD && f == 1.0f && p.src[0] == p.dst[0]) return;
    for (int t = 0; t < p.count; ++t) {
        const int64_t n = p.n[t];
        for (int64_t i = (blockIdx.x * int64_t(256) + threadIdx.x) * 8; i < n; i += int64_t(gridDim.x) * 2048) {
            const int have = static_cast<int>(min<int64_t>(n - i, 8));
            const f32x4 a = load_row<SD>(p.src[t], i, have), b = load_row<SD>(p.src[t], i + 4, have - 4);
            store_row<OD>(p.dst[t], i, have, a * f);
            store_row<OD>(p.dst[t], i + 4, have - 4, b * f);
        }
    }
}

// ---- host ------------------------------------------------------------------------------------
int64_t up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }

// dW in tiles of 256, its last rows or columns apart where that is estimated to be shorter: a round that
// is mostly empty takes as long as a full one.  They are formed in tiles of 128 (splits 1), or in tiles of 256
// whose sums are split so that they fill a round: 50257 x 768 over 8192 rows are two rounds and 79 tiles,
// which take 94 us in three parts with their join, and 134 in tiles of 128 (bf16).
struct DwCut {
    int64_t m, n;  // the part in whole tiles of 256
    int splits;
};
DwCut dw_cut(int64_t m, int64_t n, int64_t k) {
    const int64_t rows = (m + 255) / 256, cols = (n + 255) / 256, steps = (k + 63) / 64;
    DwCut best{m, n, 1};
    double least = 0.97 * round_cost(256, rows * cols, steps, false, 9.0);
    const auto consider = [&](int64_t whole, int64_t left, int64_t m_left, int64_t n_left, int64_t m_whole, int64_t n_whole) {
        const double before = round_cost(256, whole, steps, false, 9.0) + 3.0;
        if (before >= least) return;
        const double small = before + round_cost(128, ((m_left + 127) / 128) * ((n_left + 127) / 128), steps, false, 6.0);
        if (small < least) least = small, best = {m_whole, n_whole, 1};
        const int splits = static_cast<int>(std::min<int64_t>(256 / left, 16));
        if (splits < 2 || steps < 4 * splits) return;
        const double split = before + split_cost(256, m_left, n_left, left, steps, splits, false);
        if (split < least) least = split, best = {m_whole, n_whole, splits};
    };
    for (int64_t less = 1; less < 256; ++less) {  // tile rows or columns left to the second launch
        if (less < rows && less * cols < 256)
            consider((rows - less) * cols, less * cols, m - (rows - less) * 256, n, (rows - less) * 256, n);
        if (less < cols && less * rows < 256)
            consider(rows * (cols - less), less * rows, m, n - (cols - less) * 256, m, (cols - less) * 256);
    }
    return best;
}

// Everything a call's launches and working storage follow from.
struct Plan {
    bool thin, grads, pad;  // pad: W is copied to rows on 16 bytes first
    int size;               // logit tiles
    int64_t cut;            // the words from here on are in tiles of 128 instead
    int tiles, pieces;
    int64_t most;           // rows of a piece, at most
    int64_t ld, ldk;        // gathered rows; exponentials
    SplitArgs split;        // of dx
    Choice dw;
    DwCut cut_dw;
    bool turned;            // dW reads hidden states with the tokens along a row
    int64_t control, place, token, word, weight, target, row, row_loss, rows, padded, stats, sums, kept, dw_sums, db_sums,
        parts, partial, turned_rows, bytes;
};

// Where the last, mostly empty round of tiles of 256 is better formed in tiles of 128: the words from
// which on they are.  788 tiles (1024 tokens over 50257 words) are three rounds and 20 tiles.
int64_t column_cut(int64_t rows, int64_t vocab, double steps) {
    const int64_t high = (rows + 255) / 256, wide = (vocab + 255) / 256, high128 = (rows + 127) / 128;
    int64_t best = vocab;
    double least = 0.97 * round_cost(256, high * wide, steps, false, 9.0);
    for (int64_t less = 1; less < std::min<int64_t>(wide, 256) && less * high < 256; ++less) {
        const int64_t cut = (wide - less) * 256;
        const double cost = round_cost(256, high * (wide - less), steps, false, 9.0) +
                            round_cost(128, high128 * ((vocab - cut + 127) / 128), steps, false, 6.0) + 3.0;
        if (cost < least) least = cost, best = cut;
    }
    return best;
}

// `aligned`: W's rows load straight into LDS, which tiles of 256 need.
Plan plan_of(int64_t tokens, int64_t inner, int64_t vocab, int dtype, int wants, int grad_dtype, bool smooth,
             bool aligned) {
    Plan p{};
    if (is_small(tokens, inner, vocab)) return p;
    const int64_t size = dtype == F32 ? 4 : 2;
    p.grads = wants != 0;
    p.thin = tokens <= kThin && tokens * inner * vocab <= kThinProducts && !p.grads;
    p.pad = !aligned && dtype != F32 && tokens >= kPadTokens;
    aligned = aligned || p.pad;
    p.ld = up(std::max<int64_t>(inner, 1), 64);
    p.ldk = up(vocab, 64);
    int64_t at = 0;
    const auto take = [&](int64_t bytes) {
        const int64_t here = at;
        at += up(bytes, 256);
        return here;
    };
    if (p.thin) {
        p.tiles = static_cast<int>((vocab + 15) / 16);
        p.pieces = 1, p.most = tokens;
    } else {
        p.size = 0;
        double least = 0.0;
        const double steps = static_cast<double>((inner + (dtype == F32 ? 31 : 63)) / (dtype == F32 ? 32 : 64));
        const int64_t rows = std::min<int64_t>(tokens, std::max<int64_t>(256, kPieceBytes / (p.ldk * size)));
        for (const int s : {64, 128, 256}) {
            if (s == 256 && (dtype == F32 || !aligned)) continue;
            const double cost = round_cost(s, ((rows + s - 1) / s) * ((vocab + s - 1) / s), steps, dtype == F32,
                                           s == 256 ? 9.0 : (s == 128 ? 6.0 : 3.5));
            if (least == 0.0 || cost < least) least = cost, p.size = s;
        }
        p.cut = p.size == 256 ? column_cut(rows, vocab, steps) : vocab;
        p.tiles = static_cast<int>((p.cut + p.size - 1) / p.size + (vocab - p.cut + 127) / 128);
        const int64_t row_bytes = p.grads ? p.ldk * size : 12 * p.tiles;
        p.most = std::max<int64_t>(256, (p.grads ? kPieceBytes : kStatsBytes) / row_bytes / 256 * 256);
        p.most = std::min(p.most, kMostRows);
        p.pieces = static_cast<int>((tokens + p.most - 1) / p.most);
        p.most = std::min(up(up(tokens, p.pieces) / p.pieces, 256), tokens);
    }
    p.target = take(4 * tokens);
    p.row_loss = take(8 * tokens);
    p.stats = take(8 * p.most * p.tiles);
    p.sums = smooth ? take(4 * p.most * p.tiles) : 0;
    if (!p.thin) {
        p.control = take(sizeof(Control));
        p.place = take(4 * tokens);
        p.token = take(4 * tokens);
        p.word = take(4 * tokens);
        p.weight = take(4 * tokens);
        p.rows = take(size * tokens * p.ld);
        if (p.pad) p.padded = take(size * vocab * p.ld);
    }
    if (p.grads) {
        p.row = take(sizeof(Row) * tokens);
        p.kept = take(size * up(p.most, 64) * p.ldk);
        const bool carried = p.pieces > 1;
        if ((wants & HBT_LINEAR_DW) && carried && grad_dtype != F32) p.dw_sums = take(4 * vocab * inner);
        if (wants & HBT_LINEAR_DBIAS) {
            p.parts = take(4 * kBiasBlocks * vocab);
            p.db_sums = take(4 * vocab);
        }
        int64_t partial = 0;
        if ((wants & HBT_LINEAR_DX) && inner > 0) {
            const int64_t tile = choose(p.most, inner, vocab, dtype, aligned).tile, across = (inner + tile - 1) / tile;
            const int64_t tiles = (p.most + tile - 1) / tile * across, steps = (vocab + (size == 4 ? 31 : 63)) / (size == 4 ? 32 : 64);
            const int64_t most = steps >= 8 && tiles <= kMostParts ? std::min(kMostParts, tiles * 16) : 0;
            p.split = SplitArgs{inner, static_cast<int>(tile), static_cast<int>(across), static_cast<int>(steps),
                                static_cast<int>(most), size == 4};
            partial = 4 * most * tile * tile;
        }
        if ((wants & HBT_LINEAR_DW) && inner > 0) {
            p.dw = choose(vocab, inner, p.most, dtype, true);
            p.turned = p.dw.tile == 256;
            if (p.turned) p.turned_rows = take(size * inner * up(p.most, 64));
            if (p.dw.splits > 1) {
                partial = std::max(partial, 4 * p.dw.splits * up(vocab, 256) * up(inner, 4));
            } else if (p.dw.tile == 256) {
                p.cut_dw = dw_cut(vocab, inner, p.most);
                const int64_t m = p.cut_dw.m < vocab ? vocab - p.cut_dw.m : vocab, n = p.cut_dw.n < inner ? inner - p.cut_dw.n : inner;
                if (p.cut_dw.splits > 1) partial = std::max(partial, 4 * p.cut_dw.splits * up(m, 256) * up(n, 4));
            }
        }
        p.partial = take(partial);
    }
    p.bytes = at;
    return p;
}

template <class T, bool kAsync, int kLds = lds_bytes<T, kAsync>(), class Kernel, class Args>
int32_t launch(const char* who, Kernel kernel, const Args& args, int64_t blocks, std::atomic<uint64_t>& done, hipStream_t s) {
    if constexpr (kLds > 65536) {
        const int32_t status = allow_lds(who, reinterpret_cast<const void*>(kernel), kLds, done);
        if (status != HBT_OK) return status;
    }
    kernel<<<dim3(static_cast<unsigned>(blocks)), T::kThreads, kLds, s>>>(args);
    return check_launch(who);
}

// The words [column, end), whose statistics are tiles first_tile and on.
template <int D, class T, bool kAsync>
int32_t launch_logits(const char* who, LogitArgs p, int64_t rows, int64_t column, int64_t end, int first_tile,
                      hipStream_t s) {
    static std::atomic<uint64_t> done{0};
    constexpr int kLds = lds_bytes<T, kAsync>() + 3 * 4 * T::WN * T::BM;
    p.column = column, p.end = end, p.first_tile = first_tile;
    p.tiles_n = static_cast<int>((end - column + T::BN - 1) / T::BN);
    int64_t tiles = (rows + T::BM - 1) / T::BM * p.tiles_n;
    if (T::BM == 256) tiles = std::min<int64_t>(tiles, device_cu_count());
    return launch<T, kAsync, kLds>(who, logit_kernel<D, T, kAsync>, p, tiles, done, s);
}

template <int D, int OD, bool kRows>
int32_t join_parts(const char* who, const GradArgs& p, hipStream_t s) {
    const int64_t blocks = std::min<int64_t>((p.m * (p.ldp / 4) + 255) / 256, 4096);
    grad_join_kernel<D, OD, kRows><<<dim3(static_cast<unsigned>(blocks)), 256, 0, s>>>(p);
    return check_launch(who);
}

template <int D, int OD, bool kRows, bool kTurned, class T, bool kAsync>
int32_t launch_grad_tile(const char* who, GradArgs& p, int64_t most_parts, hipStream_t s) {
    static std::atomic<uint64_t> done{0};
    p.tiles_n = static_cast<int>((p.n + T::BN - 1) / T::BN);
    const int64_t blocks = std::max((p.m + T::BM - 1) / T::BM * p.tiles_n * p.splits, most_parts);
    return launch<T, kAsync>(who, grad_kernel<D, OD, kRows, kTurned, T, kAsync>, p, blocks, done, s);
}

// dW in tiles of 256, its last rows or columns in a launch of their own: in parts of their sums, or
// in tiles of 128.
template <int D, int OD>
int32_t launch_cut(const char* who, const GradArgs& p, const DwCut& cut, hipStream_t s) {
    GradArgs first = p, last = p;
    first.m = cut.m, first.n = cut.n;
    int32_t status = launch_grad_tile<D, OD, false, true, Tile256, true>(who, first, 0, s);
    if (status != HBT_OK || (cut.m == p.m && cut.n == p.n)) return status;
    const int64_t m0 = cut.m < p.m ? cut.m : 0, n0 = cut.n < p.n ? cut.n : 0;
    last.m -= m0, last.m_in -= m0, last.n -= n0, last.n_in -= n0;
    last.a = static_cast<const char*>(p.a) + m0 * elem_bytes<D>();
    last.b = static_cast<const char*>(p.b) + n0 * p.ldb * elem_bytes<D>();
    last.y = static_cast<char*>(p.y) + (m0 * p.ldy + n0) * elem_bytes<OD>();
    if (p.before != nullptr) last.before = p.before + m0 * p.ldbefore + n0;
    if (cut.splits == 1) return launch_grad_tile<D, OD, false, true, Tile128, true>(who, last, 0, s);
    last.splits = cut.splits;
    last.ldp = up(last.n, 4);
    status = launch_grad_tile<D, OD, false, true, Tile256, true>(who, last, 0, s);
    return status != HBT_OK ? status : join_parts<D, OD, false>(who, last, s);
}

// p.m or p.k is the most that the piece's rows may be.  dx: `split` has its tile, and how many parts
// there may be; dW: its choice, and its cut in tiles of 256.
template <int D, int OD, bool kRows>
int32_t launch_grad(const char* who, GradArgs& p, const SplitArgs& split, const Choice& dw, const DwCut& cut, bool aligned,
                    void* space, hipStream_t s) {
    const Choice c = kRows ? Choice{split.tile, 1} : dw;
    const int64_t parts = kRows ? split.most : 0;
    p.splits = c.splits;
    p.ldp = up(p.n, 4);
    p.partial = static_cast<float*>(space);
    int32_t status = HBT_OK;
    if (c.tile == 64) {
        status = aligned ? launch_grad_tile<D, OD, kRows, false, Tile64, true>(who, p, parts, s)
                         : launch_grad_tile<D, OD, kRows, false, Tile64, false>(who, p, parts, s);
    } else if (c.tile == 128) {
        status = aligned ? launch_grad_tile<D, OD, kRows, false, Tile128, true>(who, p, parts, s)
                         : launch_grad_tile<D, OD, kRows, false, Tile128, false>(who, p, parts, s);
    } else if constexpr (D != F32) {
        if constexpr (!kRows) {
            status = c.splits == 1 ? launch_cut<D, OD>(who, p, cut, s)
                                   : launch_grad_tile<D, OD, kRows, true, Tile256, true>(who, p, 0, s);
        } else {
            status = launch_grad_tile<D, OD, kRows, false, Tile256, true>(who, p, parts, s);
        }
    }
    if (status != HBT_OK || (c.splits == 1 && parts == 0)) return status;
    return join_parts<D, OD, kRows>(who, p, s);
}

int32_t refuse(const char* who, const char* what) {
    set_error("%s: %s", who, what);
    return HBT_ERR_INVALID_ARGUMENT;
}

int32_t check_sizes(const char* who, int64_t tokens, int64_t inner, int64_t vocab, int32_t dtype, int32_t wants,
                    int32_t grad_dtype) {
    if (tokens < 0 || inner < 0) return refuse(who, "a size is negative");
    if (vocab < 1) return refuse(who, "the vocabulary is empty");
    if (dtype != F32 && dtype != BF16 && dtype != F16) {
        set_error("%s: dtype %d is not F32, BF16 or F16", who, dtype);
        return HBT_ERR_INVALID_ARGUMENT;
    }
    if (wants < 0 || wants > 7) return refuse(who, "unknown results are wanted");
    if (wants != 0 && grad_dtype != dtype && grad_dtype != F32) return refuse(who, "gradients are of the tensors' dtype or F32");
    if (vocab > kMaxLd - 64 || inner > kMaxLd - 64 || tokens > kMostTokens) {
        set_error("%s: %lld tokens of %lld over %lld words are past the limits", who, static_cast<long long>(tokens),
                  static_cast<long long>(inner), static_cast<long long>(vocab));
        return HBT_ERR_UNSUPPORTED;
    }
    return HBT_OK;
}

int32_t check_rows(const char* who, const void* p, int64_t rows, int64_t cols, int64_t ld, const char* name) {
    if (rows == 0 || cols == 0) return HBT_OK;
    if (p == nullptr || ld < cols || ld > kMaxLd) {
        set_error("%s: %s is null, or its rows are %lld elements apart (from %lld to %lld)", who, name,
                  static_cast<long long>(ld), static_cast<long long>(cols), static_cast<long long>(kMaxLd));
        return HBT_ERR_INVALID_ARGUMENT;
    }
    return HBT_OK;
}

struct Call {
    const void *x, *w, *bias;
    const int64_t* target;
    const float *token_grads, *factor;
    float* loss;
    void *dx, *dw, *db;
    int64_t ldx, ldw, lddx, lddw, tokens, inner, vocab, ignore;
    int reduction, wants;
    float smoothing;
};

template <int D, int OD>
int32_t run(const char* who, const Call& c, const Plan& plan, char* space, hipStream_t s) {
    const auto at = [&](int64_t offset) { return static_cast<void*>(space + offset); };
    float2* stats = static_cast<float2*>(at(plan.stats));
    float* sums = c.smoothing != 0.0f ? static_cast<float*>(at(plan.sums)) : nullptr;
    float* target = static_cast<float*>(at(plan.target));
    double* row_loss = c.reduction == HBT_LOSS_NONE || c.loss == nullptr ? nullptr : static_cast<double*>(at(plan.row_loss));
    float* token_loss = c.reduction == HBT_LOSS_NONE ? c.loss : nullptr;
    const int mean = c.reduction == HBT_LOSS_MEAN;
    int32_t status = HBT_OK;
    if (is_small(c.tokens, c.inner, c.vocab)) {
        static std::atomic<uint64_t> done{0};
        const int bytes = static_cast<int>(small_lds(c.tokens, c.inner, c.vocab));
        if (bytes > 65536 &&
            (status = allow_lds(who, reinterpret_cast<const void*>(small_kernel<D, OD>), kSmallLds, done)) != HBT_OK)
            return status;
        small_kernel<D, OD><<<1, 1024, bytes, s>>>({c.x, c.w, c.bias, c.target, c.token_grads, c.factor, c.loss, c.dx, c.dw, c.db, c.ldx,
                                                    c.ldw, c.lddx, c.lddw, c.ignore, static_cast<int>(c.tokens),
                                                    static_cast<int>(c.inner), static_cast<int>(c.vocab), c.reduction,
                                                    c.smoothing});
        return check_launch(who);
    }
    JoinArgs join{};
    join.stats = stats, join.sums = sums, join.target = target, join.loss = token_loss, join.row_loss = row_loss;
    join.ignore = c.ignore, join.vocab = c.vocab, join.tiles = plan.tiles, join.smoothing = c.smoothing;
    join.unit = unit<D>();
    if (plan.thin) {
        thin_logit_kernel<D><<<dim3(plan.tiles), 512, 0, s>>>(c.x, c.ldx, c.w, c.ldw, c.bias, c.target,
                                                              static_cast<int>(c.tokens), c.vocab, c.inner, stats, sums, target);
        if ((status = check_launch(who)) != HBT_OK) return status;
        join.raw = c.target, join.stride = plan.tiles;
        thin_join_kernel<<<dim3(static_cast<unsigned>(c.tokens)), 1024, 0, s>>>(join);
        if ((status = check_launch(who)) != HBT_OK || row_loss == nullptr) return status;
        total_kernel<<<1, 1024, 0, s>>>(row_loss, nullptr, c.target, c.ignore, c.tokens, mean, c.loss);
        return check_launch(who);
    }
    Control* control = static_cast<Control*>(at(plan.control));
    int32_t* token = static_cast<int32_t*>(at(plan.token));
    int32_t* word = static_cast<int32_t*>(at(plan.word));
    int32_t* place = static_cast<int32_t*>(at(plan.place));
    float* weight = static_cast<float*>(at(plan.weight));
    void* rows = at(plan.rows);
    const PrepareArgs prepare{c.target, c.token_grads, c.factor, control, place, token, word, weight, c.tokens, c.vocab, c.ignore, mean,
                              D == F16 && plan.grads, plan.pieces, plan.split};
    const GatherArgs gather{c.x, place, rows, c.dx, token_loss, c.ldx, plan.ld, c.lddx, c.tokens, c.inner, OD == F32};
    const dim3 gathers(static_cast<unsigned>((c.tokens + 3) / 4));
    if (c.tokens <= kFewTokens) {
        prepare_few_kernel<D><<<gathers, 256, 0, s>>>(prepare, gather);
    } else {
        prepare_kernel<<<1, 1024, 0, s>>>(prepare);
        if ((status = check_launch(who)) != HBT_OK) return status;
        gather_kernel<D><<<gathers, 256, 0, s>>>(gather);
    }
    if ((status = check_launch(who)) != HBT_OK) return status;
    const bool aligned = plan.pad || is_aligned(c.w, c.ldw, c.inner, D);
    const void* w = plan.pad ? at(plan.padded) : c.w;
    const int64_t ldw = plan.pad ? plan.ld : c.ldw;
    if (plan.pad) {
        pad_kernel<D><<<dim3(static_cast<unsigned>((c.vocab + 3) / 4)), 256, 0, s>>>(c.w, c.ldw, at(plan.padded), plan.ld,
                                                                                   c.vocab, c.inner);
        if ((status = check_launch(who)) != HBT_OK) return status;
    }
    void* kept = plan.grads ? at(plan.kept) : nullptr;
    Row* row = plan.grads ? static_cast<Row*>(at(plan.row)) : nullptr;
    for (int i = 0; i < plan.pieces; ++i) {
        const Piece piece{control, i, plan.pieces};
        LogitArgs l{};
        l.x = rows, l.w = w, l.bias = c.bias, l.word = word, l.stats = stats, l.sums = sums, l.target = target;
        l.kept = kept, l.ldx = plan.ld, l.ldw = ldw, l.ldk = plan.ldk, l.inner = c.inner, l.stride = plan.most;
        l.piece = piece;
        const int64_t most = plan.most, vocab = c.vocab;
        if (plan.size == 64) {
            status = aligned ? launch_logits<D, Tile64, true>(who, l, most, 0, vocab, 0, s)
                             : launch_logits<D, Tile64, false>(who, l, most, 0, vocab, 0, s);
        } else if (plan.size == 128) {
            status = aligned ? launch_logits<D, Tile128, true>(who, l, most, 0, vocab, 0, s)
                             : launch_logits<D, Tile128, false>(who, l, most, 0, vocab, 0, s);
        } else if constexpr (D != F32) {
            status = launch_logits<D, Tile256, true>(who, l, most, 0, plan.cut, 0, s);
            if (status == HBT_OK && plan.cut < vocab)
                status = launch_logits<D, Tile128, true>(who, l, most, plan.cut, vocab, static_cast<int>(plan.cut / 256), s);
        }
        if (status != HBT_OK) return status;
        join.word = word, join.token = token, join.weight = weight, join.row = row, join.piece = piece;
        join.stride = plan.most;
        join_kernel<<<dim3(static_cast<unsigned>((plan.most + kJoinRows - 1) / kJoinRows)), kJoinRows * kJoinGroups, 0, s>>>(join);
        if ((status = check_launch(who)) != HBT_OK) return status;
        if (!plan.grads) continue;
        const bool last = i + 1 == plan.pieces, totals = last && row_loss != nullptr && c.tokens <= kTotalTokens;
        const int64_t segment = 256 * kSoftmaxUnits * unit_elems<D>();
        const int64_t blocks = (plan.ldk + segment - 1) / segment * (plan.turned ? up(plan.most, 64) : plan.most) + totals;
        softmax_kernel<D><<<dim3(static_cast<unsigned>(blocks)), 256, 0, s>>>(
            {kept, stats, row, word, plan.ldk, c.vocab, plan.most, plan.cut, plan.size, 128, c.smoothing, row_loss,
             totals ? c.loss : nullptr, mean, plan.turned, piece});
        if ((status = check_launch(who)) != HBT_OK) return status;
        if (totals) row_loss = nullptr;
        if ((c.wants & HBT_LINEAR_DX) && c.inner > 0) {
            GradArgs g{};
            g.a = kept, g.b = w, g.y = c.dx, g.token = token, g.lda = plan.ldk, g.ldb = ldw, g.ldy = c.lddx;
            g.m = plan.most, g.n = c.inner, g.k = c.vocab, g.m_in = plan.most, g.n_in = plan.pad ? up(c.inner, 8) : c.inner, g.piece = piece;
            if ((status = launch_grad<D, OD, true>(who, g, plan.split, plan.dw, plan.cut_dw, aligned, at(plan.partial), s)) != HBT_OK) return status;
        }
        if ((c.wants & HBT_LINEAR_DW) && c.inner > 0) {
            GradArgs g{};
            g.a = kept, g.b = rows, g.lda = plan.ldk, g.ldb = plan.ld;
            g.m = c.vocab, g.n = c.inner, g.k = plan.most, g.m_in = up(c.vocab, 8), g.n_in = up(c.inner, 8), g.piece = piece;
            if (plan.turned) {
                g.b = at(plan.turned_rows), g.ldb = up(plan.most, 64), g.n_in = c.inner;
                const dim3 grid(static_cast<unsigned>(g.ldb / 64), static_cast<unsigned>((c.inner + 63) / 64));
                turn_kernel<<<grid, 256, 0, s>>>({static_cast<const uint16_t*>(rows), static_cast<uint16_t*>(at(plan.turned_rows)),
                                                  plan.ld, g.ldb, c.inner, piece});
                if ((status = check_launch(who)) != HBT_OK) return status;
            }
            // Between pieces the sums stand dense in fp32: in working storage, or in an fp32 result.
            float* carried = OD == F32 ? static_cast<float*>(c.dw) : static_cast<float*>(at(plan.dw_sums));
            const int64_t ldcarried = OD == F32 ? c.lddw : c.inner;
            g.before = i > 0 ? carried : nullptr, g.ldbefore = ldcarried;
            if (last) {
                g.y = c.dw, g.ldy = c.lddw;
                status = launch_grad<D, OD, false>(who, g, plan.split, plan.dw, plan.cut_dw, true, at(plan.partial), s);
            } else {
                g.y = carried, g.ldy = ldcarried;
                status = launch_grad<D, F32, false>(who, g, plan.split, plan.dw, plan.cut_dw, true, at(plan.partial), s);
            }
            if (status != HBT_OK) return status;
        }
        if (c.wants & HBT_LINEAR_DBIAS) {
            float* parts = static_cast<float*>(at(plan.parts));
            const unsigned blocks = static_cast<unsigned>((c.vocab + 255) / 256);
            bias_part_kernel<D><<<dim3(blocks, kBiasBlocks), 256, 0, s>>>(kept, plan.ldk, c.vocab, parts, piece);
            if ((status = check_launch(who)) != HBT_OK) return status;
            bias_join_kernel<OD><<<dim3(blocks), 256, 0, s>>>(parts, static_cast<float*>(at(plan.db_sums)), c.db, c.vocab, piece);
            if ((status = check_launch(who)) != HBT_OK) return status;
        }
    }
    if (row_loss == nullptr) return HBT_OK;
    total_kernel<<<1, 1024, 0, s>>>(row_loss, control, nullptr, c.ignore, 0, mean, c.loss);
    return check_launch(who);
}

}  // namespace
}  // namespace mm
}  // namespace hbt

using namespace hbt;
using namespace hbt::mm;

extern "C" {

int64_t hbt_linear_cross_entropy_workspace(int64_t tokens, int64_t inner, int64_t vocab, int32_t dtype, int32_t wants,
                                           int32_t grad_dtype, float smoothing, int32_t aligned) {
    clear_error();
    const char* who = "hbt_linear_cross_entropy_workspace";
    if (check_sizes(who, tokens, inner, vocab, dtype, wants, grad_dtype) != HBT_OK) return -1;
    if (tokens == 0) return 0;
    const bool smooth = smoothing != 0.0f;
    return plan_of(tokens, inner, vocab, dtype, wants, grad_dtype, smooth, aligned != 0).bytes;
}

int32_t hbt_linear_cross_entropy(const void* x, int64_t ldx, const void* w, int64_t ldw, const void* bias,
                                 const int64_t* target, const float* token_grads, const float* factor, float* loss,
                                 void* dx, int64_t lddx, void* dw, int64_t lddw, void* dbias, int64_t tokens, int64_t inner, int64_t vocab,
                                 int32_t dtype, int32_t grad_dtype, int64_t ignore_index, float smoothing,
                                 int32_t reduction, void* workspace, int64_t workspace_bytes, void* stream) {
    clear_error();
    const char* who = "hbt_linear_cross_entropy";
    const int32_t wants = (dx != nullptr ? HBT_LINEAR_DX : 0) | (dw != nullptr ? HBT_LINEAR_DW : 0) |
                          (dbias != nullptr ? HBT_LINEAR_DBIAS : 0);
    int32_t status = check_sizes(who, tokens, inner, vocab, dtype, wants, grad_dtype);
    if (status != HBT_OK) return status;
    if (!(smoothing >= 0.0f && smoothing <= 1.0f)) return refuse(who, "smoothing lies outside [0, 1]");
    if (reduction < HBT_LOSS_NONE || reduction > HBT_LOSS_SUM) return refuse(who, "unknown reduction");
    if (reduction != HBT_LOSS_NONE && token_grads != nullptr) return refuse(who, "token_grads belong to separate losses");
    if (tokens == 0) return refuse(who, "there are no tokens");
    if (loss == nullptr && wants == 0) return refuse(who, "nothing is wanted");
    if (target == nullptr) return refuse(who, "target is null");
    if ((status = check_rows(who, x, tokens, inner, ldx, "x")) != HBT_OK ||
        (status = check_rows(who, w, vocab, inner, ldw, "w")) != HBT_OK ||
        (dx != nullptr && (status = check_rows(who, dx, tokens, inner, lddx, "dx")) != HBT_OK) ||
        (dw != nullptr && (status = check_rows(who, dw, vocab, inner, lddw, "dw")) != HBT_OK))
        return status;
    const Plan plan = plan_of(tokens, inner, vocab, dtype, wants, grad_dtype, smoothing != 0.0f,
                              is_aligned(w, ldw, inner, dtype));
    if (plan.bytes > 0 &&
        (workspace == nullptr || workspace_bytes < plan.bytes || reinterpret_cast<uintptr_t>(workspace) % 256 != 0))
        return refuse(who, "the workspace is smaller than hbt_linear_cross_entropy_workspace's, or off 256 bytes");
    const Call c{x, w, bias, target, token_grads, factor, loss, dx, dw, dbias, ldx, ldw, lddx, lddw, tokens, inner, vocab,
                 ignore_index, reduction, wants, smoothing};
    char* space = static_cast<char*>(workspace);
    const hipStream_t s = as_stream(stream);
    const bool wide = wants != 0 && grad_dtype == F32;
    if (dtype == F32) return run<F32, F32>(who, c, plan, space, s);
    if (dtype == BF16) return wide ? run<BF16, F32>(who, c, plan, space, s) : run<BF16, BF16>(who, c, plan, space, s);
    return wide ? run<F16, F32>(who, c, plan, space, s) : run<F16, F16>(who, c, plan, space, s);
}

int32_t hbt_scale_round(const void* const* srcs, void* const* dsts, const int64_t* numels, int32_t count,
                        int32_t src_dtype, int32_t dst_dtype, const float* factor, void* stream) {
    clear_error();
    const char* who = "hbt_scale_round";
    if (count < 0 || count > HBT_MAX_SCALED) {
        set_error("%s: count must lie in [0, %d], got %d", who, HBT_MAX_SCALED, count);
        return HBT_ERR_INVALID_ARGUMENT;
    }
    const bool pair = (src_dtype == F32 && (dst_dtype == F32 || dst_dtype == BF16 || dst_dtype == F16)) ||
                      (src_dtype == BF16 && dst_dtype == BF16) || (src_dtype == F16 && dst_dtype == F16);
    if (!pair) {
        set_error("%s: dtypes (%d, %d) are not of F32 to any, or of one 2-byte dtype", who, src_dtype, dst_dtype);
        return HBT_ERR_INVALID_ARGUMENT;
    }
    if (count > 0 && (srcs == nullptr || dsts == nullptr || numels == nullptr || factor == nullptr))
        return refuse(who, "a table or the factor is null");
    ScaleArgs p{};
    p.factor = factor;
    int64_t longest = 0;
    bool in_place = true;
    for (int i = 0; i < count; ++i) {
        if (numels[i] < 0) return refuse(who, "numel is negative");
        if (numels[i] == 0) continue;
        if (srcs[i] == nullptr || dsts[i] == nullptr) return refuse(who, "a data pointer is null");
        if (srcs[i] == dsts[i] && src_dtype != dst_dtype) return refuse(who, "in place, both dtypes must be the same");
        in_place = in_place && srcs[i] == dsts[i];
        p.src[p.count] = srcs[i], p.dst[p.count] = dsts[i], p.n[p.count++] = numels[i];
        longest = std::max(longest, numels[i]);
    }
    if (p.count == 0) return HBT_OK;
    for (int i = 0; i < p.count; ++i)
        if (!in_place && p.src[i] == p.dst[i]) return refuse(who, "either every tensor is scaled in place or none");
    const dim3 grid(static_cast<unsigned>(std::min<int64_t>((longest + 2047) / 2048, 4096)));
    const hipStream_t s = as_stream(stream);
    if (src_dtype == F32 && dst_dtype == F32) scale_round_kernel<F32, F32><<<grid, 256, 0, s>>>(p);
    else if (src_dtype == F32 && dst_dtype == BF16) scale_round_kernel<F32, BF16><<<grid, 256, 0, s>>>(p);
    else if (src_dtype == F32) scale_round_kernel<F32, F16><<<grid, 256, 0, s>>>(p);
    else if (src_dtype == BF16) scale_round_kernel<BF16, BF16><<<grid, 256, 0, s>>>(p);
    else scale_round_kernel<F16, F16><<<grid, 256, 0, s>>>(p);
    return check_launch(who);
}

}  // extern "C"
