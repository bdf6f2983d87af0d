// AdamW with both moments held in 8 bits.
//
//   m' = m + (1 - beta1) (g - m);  v' = beta2 v + (1 - beta2) g^2;  r = sqrt(v')
//   p' = decay p - step m' / (r / sqrt(1 - beta2^t) + eps)
//
// Every 256 consecutive elements of a tensor (a block) share two fp32 scales, M = max |m'| and
// R = max r.  m' is held as the e4m3 value nearest to 256 m' / M: 4 significant bits over 14
// octaves, so that an element keeps its relative precision beside one ten thousand times as large.
// v' is held by its root, which spans half the octaves: r / R in 4 exponent and 4 mantissa bits (5
// significant bits over 14 octaves).  A positive root never rounds to zero: the next step would
// divide by eps alone.  The update reads this step's moments before they are rounded.
//
// Nearest codes lose what a step changes by less than half a code, and every later step with it.  A root
// shrinks by at most (1 - beta2) / 2 of itself a step, 0.05% at beta2 = 0.999 where half a code is 1.6 to 3.1%, so it
// stands still beside its block's largest: with half of a block's gradients 20 times smaller from a step on, their
// roots are 10.8 times too large over the steps 2000 to 6000 after it, the others' 1.34 times.  And a first moment's
// smallest codes round back to themselves: an element whose gradients have become zero goes on moving, at betas (0.9,
// 0.95) by a third of a learning rate a step.  So from step 17 on
//   values under 2^-14 of their block's largest, where codes are evenly spaced,
//   all first moments where 1 - beta1 < 1/16, half a code at most, and all roots where 1 - beta2 < 0.04
// go to one of the two codes around them, the upper one with the probability that leaves no bias, by random
// numbers of the step and the element's place: equal inputs give equal bits.  Roots are then within 1% on average
// and 10% each (26% while they fall 20 times).  What else there is is rounded to nearest, which holds each value closer and
// where steps are as large as codes loses nothing: roots at beta2 = 0.95 0.7% off on average and 4.5% each (without
// bias 0.1 and 6.4), at 0.97 2.0 and 5.6 (0.2 and 7.6), at 0.98 6.4 and 9.2 (0.4 and 8.6).  The first 16 steps, in which
// a running sum grows by 1/(2t) a step, half a root's code or more, round to nearest too.  (Up to beta2 = 0.96 a
// root falls past its block's largest because that one, the scale, changes a little with every step, as gradients of
// batches make it; beside one that never changes it could stop at a code of the octave where it began.)
//
// A block's largest element is held exactly (256 M / 256, 1 R), so a decay that all elements share
// is carried by the scales without rounding, and encoding what was decoded gives the same codes.
//
// A wavefront takes a block at a time, four elements a lane, so the maxima are two butterflies in
// registers.  Bound by memory: 16 bytes an element in fp32 (p, g in, p out, two codes in and out)
// and 1/16 byte of scales, where the step with fp32 moments moves 28.
#include "hbt_matmul.hpp"

namespace hbt {
namespace {

using mm::f32x4;
using mm::load_row;
using mm::store_row;
using mm::u32x4;

constexpr int kBlock = 256;  // elements that share scales: one wavefront's four a lane
// Encoding and decoding: four wavefronts, each with two blocks in flight (decoding 1,003,782,656
// elements to bf16: 949 us; single wavefronts 983, four blocks a wavefront 1051).  The step: single
// wavefronts with a block each (fp32: 2683 us; four wavefronts 2822, two blocks a wavefront 3015).
constexpr int kWaves = 4, kUnroll = 2;
constexpr int64_t kTile = int64_t(kBlock) * kWaves * kUnroll;
constexpr int kMaxTensors = HBT_MAX_ADAMW8_TENSORS;
// First moments this far under 1 would overflow the scale's reciprocal; such a block is held as zeros.
constexpr float kLeastScale = 7.8886090522101181e-31f;  // 2^-100

// Codes of four consecutive elements stand together, those of their first moments and then those of
// their roots, so a lane moves them by one 8-byte access; a block's are 512 consecutive bytes.
struct Table {
    void* p[kMaxTensors];
    void* g[kMaxTensors];
    uint2* codes[kMaxTensors];
    float2* scales[kMaxTensors];  // a block's M and R
    int64_t n[kMaxTensors];
    int64_t first[kMaxTensors];  // the tensor's first tile
    int32_t count;
};

struct Scalars {
    float unscale, decay, lerp, beta2, one_minus_beta2, inverse_root, eps, neg_step;
};
// A step's scalars in device memory, for a step recorded into a graph; `step` where the call has one.
struct Slot {
    Scalars scalars;
    uint32_t step;
};

// How a step's moments are rounded: to nearest (step 0), or without bias where codes are evenly spaced, and
// at every size where `firsts` or `roots`.
struct Rounding {
    uint32_t step;
    bool firsts, roots;
};
constexpr uint32_t kNearestSteps = 16;
constexpr float kSlowFirst = 0.0625f, kSlowRoot = 0.04f;
__device__ __forceinline__ Rounding rounding_of(uint32_t step, const Scalars& s) {
    return {step > kNearestSteps ? step : 0u, fabsf(s.lerp) < kSlowFirst, s.one_minus_beta2 < kSlowRoot};
}

// The tensor that owns a tile: the last one whose first tile is not past it.
__device__ __forceinline__ int owner(const Table& tab, int64_t tile) {
    int low = 0, high = tab.count;
    while (high - low > 1) {
        const int mid = (low + high) >> 1;
        if (tab.first[mid] <= tile) low = mid;
        else high = mid;
    }
    return low;
}

// Magnitudes are compared as the whole numbers that their bits are, which orders non-negative floats.
constexpr uint32_t kInfinity = 0x7F800000u;
// The bits of |x|, or of 0 for what is not finite.
__device__ __forceinline__ uint32_t magnitude(float x) {
    const uint32_t bits = __float_as_uint(x) & 0x7FFFFFFFu;
    return bits < kInfinity ? bits : 0u;
}
template <int kCtrl>
__device__ __forceinline__ uint32_t row_move(uint32_t x) {
    return static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(x), kCtrl, 0xF, 0xF, false));
}
// The largest over the wavefront, in every lane.
__device__ __forceinline__ uint32_t wave_max(uint32_t x) {
    const auto half = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    x = max(half[0], half[1]);
    const auto row = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    x = max(row[0], row[1]);
    x = max(x, row_move<0x128>(x));  // row_ror:8
    x = max(x, row_move<0x124>(x));  // row_ror:4
    x = max(x, row_move<0x4E>(x));   // quad_perm [2, 3, 0, 1]
    return max(x, row_move<0xB1>(x));  // quad_perm [1, 0, 3, 2]
}

// ---- the codes -------------------------------------------------------------------------
// Four first moments as e4m3 codes of `inverse`, 256 / scale, times m.  What is not finite becomes NaN (the format
// has no infinity, and 0 times one is NaN where the scale is 0), there and nowhere else in its block.
__device__ __forceinline__ uint32_t encode_first(f32x4 m, float inverse) {
    const int code = __builtin_amdgcn_cvt_pk_fp8_f32(m[0] * inverse, m[1] * inverse, 0, false);
    return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(m[2] * inverse, m[3] * inverse, code, true));
}
__device__ __forceinline__ f32x4 decode_first(uint32_t code, float scale) {
    const auto low = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(code), false);
    const auto high = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(code), true);
    const float unit = scale * 0.00390625f;
    return f32x4{low[0] * unit, low[1] * unit, high[0] * unit, high[1] * unit};
}

// Roots over their scale, in [0, 1]: exponent e (0..15) and mantissa f of a code c = 16 e + f stand
// for (16 + f) 2^(e - 19), or f 2^-18 where e is 0.  Those are the leading bits of the fp32 number
// 2^-112 times as large, so a code is that number rounded at its 19th bit; 1 is code 240, and 255
// stands for NaN.
constexpr float kDown = 1.92592994438723585e-34f, kUp = 5.19229685853482763e33f;  // 2^-112, 2^112
constexpr uint32_t kNanCode = 255;
__device__ __forceinline__ uint32_t encode_root(float r, float inverse) {
    const uint32_t bits = __float_as_uint(r * inverse * kDown);
    const uint32_t code = (bits + 0x3FFFFu + ((bits >> 19) & 1u)) >> 19;
    // At least 1 for a positive root, at most the code of NaN, which the bits of infinity and NaN pass.
    return max(min(code, kNanCode), min(__float_as_uint(r), 1u));
}
__device__ __forceinline__ uint32_t encode_roots(f32x4 r, float inverse) {
    return encode_root(r[0], inverse) | encode_root(r[1], inverse) << 8 | encode_root(r[2], inverse) << 16 |
           encode_root(r[3], inverse) << 24;
}
__device__ __forceinline__ f32x4 decode_roots(uint32_t code, float scale) {
    f32x4 r;
#pragma unroll
    for (int e = 0; e < 4; ++e) r[e] = __uint_as_float(((code >> (8 * e)) & 255u) << 19) * kUp * scale;
    // Whether a byte is 255: a zero byte of the complement.
    if (((~code - 0x01010101u) & code & 0x80808080u) != 0) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (((code >> (8 * e)) & 255u) == kNanCode) r[e] = NAN;
    }
    return r;
}

// ---- rounding without bias -----------------------------------------------------------------
// Random numbers of a step for a lane's four elements of a block.  The block's are 128 bits of the
// counter-based generator Philox4x32 (Salmon, Moraes, Dror and Shaw, Parallel random numbers: as easy as 1, 2, 3,
// 2011) in 7 rounds with key 0, the same for every lane and so the scalar unit's work; from them the lanes stand
// a golden section apart.  So an element's numbers are uniform and independent from step to step, which is what
// keeps it without bias, and its neighbours' are spread evenly.  1 << 29 elements in fp32 at betas (0.9, 0.999):
// 1618 us, 1675 with each lane's own generator, 1444 to nearest.
__device__ __forceinline__ u32x4 random_words(int64_t block, uint32_t step, int lane) {
    uint32_t a = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(block)), d = 0, k0 = 0, k1 = 0;
    uint32_t b = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(block >> 32));
    uint32_t c = __builtin_amdgcn_readfirstlane(step);
#pragma unroll
    for (int i = 0; i < 7; ++i) {
        const uint64_t x = uint64_t(0xD2511F53u) * a, y = uint64_t(0xCD9E8D57u) * c;
        a = static_cast<uint32_t>(y >> 32) ^ b ^ k0, b = static_cast<uint32_t>(y);
        c = static_cast<uint32_t>(x >> 32) ^ d ^ k1, d = static_cast<uint32_t>(x);
        k0 += 0x9E3779B9u, k1 += 0xBB67AE85u;
    }
    return u32x4{a, b, c, d} + lane * 0x9E3779B9u;
}

// e4m3 codes are the leading bits of an fp32 number 2^-120 times as large, as roots' are of one 2^-112 times:
// of `bits`, the last kLow are rounded off, with 16 random ones added where that is to leave no bias.  Under
// kNormal, kEven of the scale, codes are evenly spaced.
constexpr float kDownFirst = 7.52316384526264005e-37f;  // 2^-120
constexpr float kEven = 6.103515625e-05f;               // 2^-14
constexpr uint32_t kNormal = 0x00800000u;
__device__ __forceinline__ uint32_t first_bits(float m, float inverse) {
    return __float_as_uint(m * inverse * kDownFirst) & 0x7FFFFFFFu;
}
__device__ __forceinline__ uint32_t root_bits(float r, float inverse) { return __float_as_uint(r * inverse * kDown); }
template <int kLow>
__device__ __forceinline__ uint32_t round_bits(uint32_t bits, uint32_t random, bool free) {
    const uint32_t nearest = (1u << (kLow - 1)) - 1 + ((bits >> kLow) & 1u);
    const uint32_t any = (random << (kLow - 16)) | (1u << (kLow - 17));
    return (bits + (free || bits < kNormal ? any : nearest)) >> kLow;
}
// The same codes as encode_first's and encode_roots' but for what is rounded without bias.
__device__ __forceinline__ uint2 encode_free(f32x4 m, f32x4 r, float inverse_m, float inverse_r, u32x4 random,
                                             const Rounding& how) {
    uint2 codes = make_uint2(0, 0);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const uint32_t first = min(round_bits<20>(first_bits(m[e], inverse_m), random[e] & 0xFFFFu, how.firsts), 0x7Fu);
        const uint32_t root = min(round_bits<19>(root_bits(r[e], inverse_r), random[e] >> 16, how.roots), kNanCode);
        codes.x |= (first | (__float_as_uint(m[e]) >> 24 & 0x80u)) << (8 * e);
        codes.y |= max(root, min(__float_as_uint(r[e]), 1u)) << (8 * e);
    }
    return codes;
}

// Codes and scales of a block, of which the lane holds four moments and roots.
__device__ __forceinline__ void store_block(const Table& tab, int t, int64_t block, int lane, f32x4 m, f32x4 r,
                                            const Rounding& how) {
    uint32_t m_bits = 0, r_bits = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) m_bits = max(m_bits, magnitude(m[e])), r_bits = max(r_bits, magnitude(r[e]));
    float top_m = __uint_as_float(wave_max(m_bits));
    const float top_r = __uint_as_float(wave_max(r_bits));
    if (top_m < kLeastScale) top_m = 0.0f;
    const float inverse_m = top_m > 0.0f ? 256.0f / top_m : 0.0f, inverse_r = top_r > 0.0f ? 1.0f / top_r : 0.0f;
    bool free = false;  // whether a value of the block is rounded without bias
    if (how.step != 0) {
        const uint32_t low_m = __float_as_uint(top_m * kEven) - 1, low_r = __float_as_uint(top_r * kEven) - 1;
        free = how.firsts || how.roots;
#pragma unroll
        for (int e = 0; e < 4; ++e) free = free || magnitude(m[e]) - 1 < low_m || magnitude(r[e]) - 1 < low_r;
        free = __any(free);
    }
    tab.codes[t][block * 64 + lane] =
        free ? encode_free(m, r, inverse_m, inverse_r, random_words(block, how.step, lane), how)
             : make_uint2(encode_first(m, inverse_m), encode_roots(r, inverse_r));
    if (lane == 0) tab.scales[t][block] = make_float2(top_m, top_r);
}

// ---- kernels -----------------------------------------------------------------------------
// Waits for the global loads issued so far, and keeps the next ones behind.
__device__ __forceinline__ void wait_for_loads() {
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
    __builtin_amdgcn_sched_barrier(0);
}

// A wavefront a block; 1,003,782,656 elements in fp32 at betas (0.9, 0.95) take 2731 us (5.9 TB/s).  With fp32
// gradients each stream is waited for before the next one is asked for (all to nearest: 2647 us, 2790 with all loads
// in flight together).
// 2-byte gradients leave less to move for the same arithmetic (a correctly rounded root and division an
// element), which the loads then have to hide behind (all to nearest: 2335 us together and the gradient last, 2475 one
// after another; fp32 masters and bf16 gradients, 2^29 elements, now 1339 us, 5.6 TB/s).
template <int PD, int GD, bool kWriteBack>
__global__ __launch_bounds__(64) void adamw8_kernel(Table tab, Scalars s, uint32_t step, const Slot* __restrict__ slot,
                                                    bool numbered, const float* __restrict__ grad_mul, int64_t tile_base) {
    if (slot != nullptr) {
        s = slot->scalars;
        if (numbered) step = slot->step;
    }
    const int64_t tile = tile_base + blockIdx.x;
    const int t = owner(tab, tile), lane = threadIdx.x;
    const int64_t n = tab.n[t], block = tile - tab.first[t], e = block * kBlock + lane * 4;
    const int have = static_cast<int>(min<int64_t>(n - e, 4));
    const float mul = grad_mul != nullptr ? *grad_mul : 1.0f;
    f32x4 g;
    if constexpr (GD == HBT_DTYPE_F32) {
        g = load_row<GD>(tab.g[t], e, have);
        wait_for_loads();
    }
    const uint2 codes = tab.codes[t][block * 64 + lane];
    const float2 scales = tab.scales[t][block];
    if constexpr (GD == HBT_DTYPE_F32) wait_for_loads();
    f32x4 p = load_row<PD>(tab.p[t], e, have);
    if constexpr (GD == HBT_DTYPE_F32) wait_for_loads();
    else g = load_row<GD>(tab.g[t], e, have);
    if (mul != 1.0f || s.unscale != 1.0f) {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            if (s.unscale != 1.0f) g[c] = round_to<GD>(g[c] * s.unscale);
            g[c] = round_to<GD>(g[c] * mul);
        }
        if constexpr (kWriteBack) store_row<GD>(tab.g[t], e, have, g);
    }
    f32x4 m = decode_first(codes.x, scales.x), r = decode_roots(codes.y, scales.y);
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        m[c] = m[c] + s.lerp * (g[c] - m[c]);
        r[c] = __builtin_sqrtf(r[c] * r[c] * s.beta2 + (s.one_minus_beta2 * g[c]) * g[c]);
        p[c] = p[c] * s.decay + (s.neg_step * m[c]) / (r[c] * s.inverse_root + s.eps);
        if (c >= have) m[c] = r[c] = 0.0f;  // past the tensor's end: nothing that a scale could come from
    }
    store_row<PD>(tab.p[t], e, have, p);
    store_block(tab, t, block, lane, m, r, rounding_of(step, s));
}

// Moments in fp32 (tab.p, tab.g: first and second) to codes.
__global__ __launch_bounds__(64 * kWaves) void encode_kernel(Table tab, int64_t tile_base) {
    const int64_t tile = tile_base + blockIdx.x;
    const int t = owner(tab, tile), lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t n = tab.n[t], first = (tile - tab.first[t]) * (kWaves * kUnroll) + wave;
    for (int u = 0; u < kUnroll; ++u) {
        const int64_t block = first + u * kWaves, e = block * kBlock + lane * 4;
        if (block * kBlock >= n) break;
        const int have = static_cast<int>(min<int64_t>(n - e, 4));
        const f32x4 m = load_row<HBT_DTYPE_F32>(tab.p[t], e, have), v = load_row<HBT_DTYPE_F32>(tab.g[t], e, have);
        store_block(tab, t, block, lane, m,
                    f32x4{__builtin_sqrtf(v[0]), __builtin_sqrtf(v[1]), __builtin_sqrtf(v[2]), __builtin_sqrtf(v[3])},
                    Rounding{0, false, false});
    }
}

// Codes to moments in OD (tab.p, tab.g: first and second).
template <int OD>
__global__ __launch_bounds__(64 * kWaves) void decode_kernel(Table tab, int64_t tile_base) {
    const int64_t tile = tile_base + blockIdx.x;
    const int t = owner(tab, tile), lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t n = tab.n[t], first = (tile - tab.first[t]) * (kWaves * kUnroll) + wave;
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
        const int64_t block = first + u * kWaves, e = block * kBlock + lane * 4;
        if (block * kBlock >= n) break;
        const int have = static_cast<int>(min<int64_t>(n - e, 4));
        const uint2 codes = tab.codes[t][block * 64 + lane];
        const float2 scales = tab.scales[t][block];
        const f32x4 r = decode_roots(codes.y, scales.y);
        store_row<OD>(tab.p[t], e, have, decode_first(codes.x, scales.x));
        store_row<OD>(tab.g[t], e, have, f32x4{r[0] * r[0], r[1] * r[1], r[2] * r[2], r[3] * r[3]});
    }
}

// ---- host ----------------------------------------------------------------------------
// Fills the table and counts its tiles, or refuses it.
int32_t fill(const char* who, Table& tab, int64_t& tiles, const void* const* p, const void* const* g,
             void* const* codes, void* const* scales, const int64_t* numels, int32_t count, int64_t tile) {
    if (count < 0 || count > kMaxTensors) {
        set_error("%s: count must lie in [0, %d], got %d", who, kMaxTensors, count);
        return HBT_ERR_INVALID_ARGUMENT;
    }
    if (count > 0 && (p == nullptr || g == nullptr || codes == nullptr || scales == nullptr || numels == nullptr)) {
        set_error("%s: null table pointer", who);
        return HBT_ERR_INVALID_ARGUMENT;
    }
    tiles = 0;
    tab.count = 0;
    for (int i = 0; i < count; ++i) {
        if (numels[i] < 0) {
            set_error("%s: tensor %d has negative numel %lld", who, i, static_cast<long long>(numels[i]));
            return HBT_ERR_INVALID_ARGUMENT;
        }
        if (numels[i] == 0) continue;
        if (p[i] == nullptr || g[i] == nullptr || codes[i] == nullptr || scales[i] == nullptr) {
            set_error("%s: tensor %d has a null data pointer", who, i);
            return HBT_ERR_INVALID_ARGUMENT;
        }
        if ((reinterpret_cast<uintptr_t>(codes[i]) | reinterpret_cast<uintptr_t>(scales[i])) % 8 != 0) {
            set_error("%s: tensor %d has codes or scales off 8 bytes", who, i);
            return HBT_ERR_INVALID_ARGUMENT;
        }
        const int at = tab.count++;
        tab.p[at] = const_cast<void*>(p[i]);
        tab.g[at] = const_cast<void*>(g[i]);
        tab.codes[at] = static_cast<uint2*>(codes[i]);
        tab.scales[at] = static_cast<float2*>(scales[i]);
        tab.n[at] = numels[i];
        tab.first[at] = tiles;
        tiles += (numels[i] + tile - 1) / tile;
    }
    return HBT_OK;
}

// Either entry point; `numbered`: whether the call has a step, and its slot one.
int32_t adamw8_step(const char* who, void* const* params, void* const* grads, void* const* codes, void* const* scales,
                    const int64_t* numels, int32_t count, int32_t param_dtype, int32_t grad_dtype, const Scalars& s,
                    const float* grad_mul, uint32_t step, bool numbered, const float* slot, int32_t flags, void* stream) {
    clear_error();
    constexpr int F32 = HBT_DTYPE_F32, BF16 = HBT_DTYPE_BF16, F16 = HBT_DTYPE_F16;
    const bool pair = (param_dtype == F32 && (grad_dtype == F32 || grad_dtype == BF16)) ||
                      (param_dtype == BF16 && grad_dtype == BF16) || (param_dtype == F16 && grad_dtype == F16);
    if (!pair) {
        set_error("%s: (parameter, gradient) dtypes (%d, %d) are not (F32, F32), (F32, BF16), (BF16, BF16) or "
                  "(F16, F16)", who, param_dtype, grad_dtype);
        return HBT_ERR_INVALID_ARGUMENT;
    }
    if ((flags & ~HBT_STEP_WRITE_GRAD) != 0) {
        set_error("%s: unknown flags 0x%x", who, static_cast<unsigned>(flags));
        return HBT_ERR_INVALID_ARGUMENT;
    }
    if (reinterpret_cast<uintptr_t>(slot) % 4 != 0) {
        set_error("%s: the slot is not 4-byte aligned", who);
        return HBT_ERR_INVALID_ARGUMENT;
    }
    Table tab{};
    int64_t tiles = 0;
    const int32_t status = fill(who, tab, tiles, params, grads, codes, scales, numels, count, kBlock);
    if (status != HBT_OK) return status;
    const Slot* from = reinterpret_cast<const Slot*>(slot);
    const bool write_back = (flags & HBT_STEP_WRITE_GRAD) != 0;
    const hipStream_t st = as_stream(stream);
    return launch_sliced(who, tiles, 64, [&](int64_t first, dim3 grid) {
        const auto launch = [&](auto pd, auto gd) {
            constexpr int PD = decltype(pd)::value, GD = decltype(gd)::value;
            if (write_back) adamw8_kernel<PD, GD, true><<<grid, 64, 0, st>>>(tab, s, step, from, numbered, grad_mul, first);
            else adamw8_kernel<PD, GD, false><<<grid, 64, 0, st>>>(tab, s, step, from, numbered, grad_mul, first);
        };
        const std::integral_constant<int, F32> f32{};
        const std::integral_constant<int, BF16> bf16{};
        const std::integral_constant<int, F16> f16{};
        if (param_dtype == F32 && grad_dtype == F32) launch(f32, f32);
        else if (param_dtype == F32) launch(f32, bf16);
        else if (param_dtype == BF16) launch(bf16, bf16);
        else launch(f16, f16);
    });
}

}  // namespace
}  // namespace hbt

using namespace hbt;

extern "C" {

int32_t hbt_adamw8_step(void* const* params, void* const* grads, void* const* codes, void* const* scales,
                        const int64_t* numels, int32_t count, int32_t param_dtype, int32_t grad_dtype, float unscale,
                        const float* grad_mul, float decay, float lerp_weight, float beta2, float one_minus_beta2,
                        float inverse_bias_correction2_sqrt, float eps, float neg_step_size, const float* slot,
                        int32_t flags, void* stream) {
    return adamw8_step("hbt_adamw8_step", params, grads, codes, scales, numels, count, param_dtype, grad_dtype,
                       {unscale, decay, lerp_weight, beta2, one_minus_beta2, inverse_bias_correction2_sqrt, eps, neg_step_size},
                       grad_mul, 0, false, slot, flags, stream);
}

int32_t hbt_adamw8_step_numbered(void* const* params, void* const* grads, void* const* codes, void* const* scales,
                                 const int64_t* numels, int32_t count, int32_t param_dtype, int32_t grad_dtype,
                                 float unscale, const float* grad_mul, float decay, float lerp_weight, float beta2,
                                 float one_minus_beta2, float inverse_bias_correction2_sqrt, float eps,
                                 float neg_step_size, uint32_t step, const float* slot, int32_t flags, void* stream) {
    return adamw8_step("hbt_adamw8_step_numbered", params, grads, codes, scales, numels, count, param_dtype, grad_dtype,
                       {unscale, decay, lerp_weight, beta2, one_minus_beta2, inverse_bias_correction2_sqrt, eps, neg_step_size},
                       grad_mul, step, true, slot, flags, stream);
}

int32_t hbt_moments8_encode(const void* const* firsts, const void* const* seconds, void* const* codes,
                            void* const* scales, const int64_t* numels, int32_t count, void* stream) {
    clear_error();
    const char* who = "hbt_moments8_encode";
    Table tab{};
    int64_t tiles = 0;
    const int32_t status = fill(who, tab, tiles, firsts, seconds, codes, scales, numels, count, kTile);
    if (status != HBT_OK) return status;
    return launch_sliced(who, tiles, 64 * kWaves, [&](int64_t first, dim3 grid) {
        encode_kernel<<<grid, 64 * kWaves, 0, as_stream(stream)>>>(tab, first);
    });
}

int32_t hbt_moments8_decode(void* const* codes, void* const* scales, void* const* firsts, void* const* seconds,
                            const int64_t* numels, int32_t count, int32_t out_dtype, void* stream) {
    clear_error();
    const char* who = "hbt_moments8_decode";
    if (out_dtype != HBT_DTYPE_F32 && out_dtype != HBT_DTYPE_BF16) {
        set_error("%s: out_dtype %d is not F32 or BF16", who, out_dtype);
        return HBT_ERR_INVALID_ARGUMENT;
    }
    Table tab{};
    int64_t tiles = 0;
    const int32_t status = fill(who, tab, tiles, firsts, seconds, codes, scales, numels, count, kTile);
    if (status != HBT_OK) return status;
    return launch_sliced(who, tiles, 64 * kWaves, [&](int64_t first, dim3 grid) {
        if (out_dtype == HBT_DTYPE_F32) decode_kernel<HBT_DTYPE_F32><<<grid, 64 * kWaves, 0, as_stream(stream)>>>(tab, first);
        else decode_kernel<HBT_DTYPE_BF16><<<grid, 64 * kWaves, 0, as_stream(stream)>>>(tab, first);
    });
}

}  // extern "C"
