// Tile products on the matrix cores (gfx950), shared by the linear layer and the
// orthogonalised update.
//
// A workgroup forms one BM x BN tile of C[m][n] = sum_k A(m, k) B(n, k).  Each operand is
// stored either k-major (the k of one row consecutive: x and W of y = x W^T) or
// row-major in the other sense (the rows of one k consecutive: both operands of
// dW = dz^T x), so the three products of a layer and its backward pass, and the Gram and
// iterate products of a Newton-Schulz step, read every matrix where it lies.
//
// Operands whose rows start on 16 bytes go straight from global memory into one of the tile's
// LDS stages (buffer loads with an LDS destination), several k-tiles ahead of the matrix cores,
// with one barrier per k-tile.  Others go through registers into two stages: unaligned 16-byte
// units are loaded as they lie, and a unit that straddles an edge element by element.  A unit
// out of range is read at an offset past the buffer's end, which returns zeros.
#pragma once

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "hbt_common.hpp"

namespace hbt {
namespace mm {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

template <int D>
constexpr int elem_bytes() { return D == HBT_DTYPE_F32 ? 4 : 2; }
// Elements of a 16-byte unit.
template <int D>
constexpr int unit_elems() { return 16 / elem_bytes<D>(); }
// Elements of k per tile: 128 bytes.
template <int D>
constexpr int tile_k() { return 128 / elem_bytes<D>(); }

template <int D>
__device__ __forceinline__ float load_elem(const void* p, int64_t i) {
    if constexpr (D == HBT_DTYPE_F32) return static_cast<const float*>(p)[i];
    else return b16_to_f32<D == HBT_DTYPE_F16>(static_cast<const uint16_t*>(p)[i]);
}
template <int D>
__device__ __forceinline__ void store_elem(void* p, int64_t i, float v) {
    if constexpr (D == HBT_DTYPE_F32) static_cast<float*>(p)[i] = v;
    else static_cast<uint16_t*>(p)[i] = static_cast<uint16_t>(f32_to_b16<D == HBT_DTYPE_F16>(v));
}
// Four consecutive elements from any element boundary.
template <int D>
__device__ __forceinline__ f32x4 load4(const void* p, int64_t i) {
    f32x4 v;
    if constexpr (D == HBT_DTYPE_F32) {
        typedef float u __attribute__((ext_vector_type(4), aligned(4)));
        const u x = *reinterpret_cast<const u*>(static_cast<const float*>(p) + i);
        v = f32x4{x[0], x[1], x[2], x[3]};
    } else {
        typedef uint32_t u __attribute__((ext_vector_type(2), aligned(2)));
        const u x = *reinterpret_cast<const u*>(static_cast<const uint16_t*>(p) + i);
        constexpr bool H = D == HBT_DTYPE_F16;
        v = f32x4{b16_to_f32<H>(x[0] & 0xFFFFu), b16_to_f32<H>(x[0] >> 16), b16_to_f32<H>(x[1] & 0xFFFFu),
                  b16_to_f32<H>(x[1] >> 16)};
    }
    return v;
}
template <int D>
__device__ __forceinline__ void store4(void* p, int64_t i, f32x4 v) {
    if constexpr (D == HBT_DTYPE_F32) {
        typedef float u __attribute__((ext_vector_type(4), aligned(4)));
        *reinterpret_cast<u*>(static_cast<float*>(p) + i) = u{v[0], v[1], v[2], v[3]};
    } else {
        typedef uint32_t u __attribute__((ext_vector_type(2), aligned(2)));
        *reinterpret_cast<u*>(static_cast<uint16_t*>(p) + i) =
            u{pack2_rounded<D>(v[0], v[1]), pack2_rounded<D>(v[2], v[3])};
    }
}

// 16 bytes from any element boundary.
__device__ __forceinline__ u32x4 load16(const char* at) {
    typedef uint32_t u __attribute__((ext_vector_type(4), aligned(2)));
    const u v = *reinterpret_cast<const u*>(at);
    return u32x4{v[0], v[1], v[2], v[3]};
}

// Element e of a 16-byte unit.
template <int D>
__device__ __forceinline__ float element(const u32x4& unit, int e) {
    if constexpr (D == HBT_DTYPE_F32) return __uint_as_float(unit[e]);
    else return b16_to_f32<D == HBT_DTYPE_F16>((unit[e / 2] >> (16 * (e % 2))) & 0xFFFFu);
}

// Elements i .. i + 3, or as many of them as exist.
template <int D>
__device__ __forceinline__ f32x4 load_row(const void* p, int64_t i, int have) {
    if (have >= 4) return load4<D>(p, i);
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int e = 0; e < 3; ++e)
        if (e < have) v[e] = load_elem<D>(p, i + e);
    return v;
}
template <int D>
__device__ __forceinline__ void store_row(void* p, int64_t i, int have, f32x4 v) {
    if (have >= 4) {
        store4<D>(p, i, v);
        return;
    }
#pragma unroll
    for (int e = 0; e < 3; ++e)
        if (e < have) store_elem<D>(p, i + e, v[e]);
}

// The same for data that is read once and does not fit the memory-side cache.
__device__ __forceinline__ u32x4 stream16(const char* at) {
    typedef uint32_t u __attribute__((ext_vector_type(4), aligned(2)));
    const u v = __builtin_nontemporal_load(reinterpret_cast<const u*>(at));
    return u32x4{v[0], v[1], v[2], v[3]};
}

// c += a b over one 16-byte fragment pair: 32 values of k in 2-byte types (one
// instruction), 16 in fp32 (four).  Lane l holds row l % 16 of each operand and the unit of
// k that its quarter l / 16 names; the order of k inside a fragment is the same in both.
// The result has element [4 (l / 16) + r][l % 16] of (first operand's row, second's).
template <int D>
__device__ __forceinline__ f32x4 mma(u32x4 a, u32x4 b, f32x4 c) {
    if constexpr (D == HBT_DTYPE_F16) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c,
                                                      0, 0, 0);
    } else if constexpr (D == HBT_DTYPE_BF16) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b),
                                                       c, 0, 0, 0);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a[j]), __uint_as_float(b[j]), c, 0, 0, 0);
        return c;
    }
}

__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer_at(const void* base) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, 0x7FFFFFFF, 0x00020000);
}
// An offset past every buffer's end: reads zeros.
constexpr uint32_t kNowhere = 0xFFFFFF00u;

// One operand's share of a tile: ROWS rows (m or n) by tile_k of k, moved by THREADS lanes.
// kKMajor: element (row, k) at base[row * ld + k]; else at base[k * ld + row].
// kAsync: rows and base on 16 bytes, and whole units (the rows of an operand that is not
// k-major, or the k of one that is, a multiple of a unit or padded to one, the k with zeros).
template <int D, bool kKMajor, int ROWS, int THREADS, bool kAsync>
struct Operand {
    static constexpr int E = unit_elems<D>(), BK = tile_k<D>(), B = elem_bytes<D>();
    static constexpr int kUnitsPerLine = kKMajor ? BK / E : ROWS / E;  // units per LDS line
    static constexpr int kLineBytes = kUnitsPerLine * 16;
    static constexpr int kUnits = ROWS * BK / E / THREADS;  // units per lane
    static constexpr int kBytes = ROWS * BK * B;
    static constexpr int kReads = kKMajor ? 1 : B;  // LDS reads per fragment: two transposing, or four
    static_assert(ROWS * BK / E % THREADS == 0, "whole units per lane");

    const char* base;      // the tile's first row (k-major) or column at k = 0
    int64_t ld;            // elements between rows (k-major) or between k
    int rows;              // rows of the operand from the tile's first one
    uint32_t offset[kUnits];
    u32x4 held[kUnits];
    bool straddles;        // some lane's unit crosses the last row (not k-major)
    bool shifted;          // ... and is loaded back from that row, to be shifted down

    // LDS position of a unit: lines are XOR-swizzled in units so that the 16 rows of a
    // fragment read (k-major), or the four k of a transposing read, fall on distinct banks.
    static __device__ __forceinline__ int swizzle(int line) {
        if constexpr (kKMajor) return line & 7;
        else if constexpr (B == 2) return (line & 3) << 1;
        else return ((line >> 2) & 3) << 2;
    }

    // The unit of its line that unit u of the lane order is.  An asynchronous load writes lane l's
    // 16 bytes l units after its wave's LDS address, so there the swizzle picks what a lane loads.
    static __device__ __forceinline__ int column(int u) {
        const int line = u / kUnitsPerLine, at = u % kUnitsPerLine;
        return kAsync ? at ^ swizzle(line) : at;
    }

    __device__ __forceinline__ void init(const void* p, int64_t ld_, int64_t row0, int64_t row_count, int tid) {
        ld = ld_;
        rows = static_cast<int>(row_count - row0 < ROWS ? row_count - row0 : ROWS);
        base = static_cast<const char*>(p) + (kKMajor ? row0 * ld_ : row0) * B;
        straddles = !kAsync && !kKMajor && rows < ROWS && rows % E != 0;
        shifted = straddles && row_count >= E;
#pragma unroll
        for (int i = 0; i < kUnits; ++i) {
            const int u = i * THREADS + tid, line = u / kUnitsPerLine, at = column(u);
            const bool in = kKMajor ? line < rows : (at + 1) * E <= rows;
            offset[i] = in ? static_cast<uint32_t>(line * ld * B) + at * 16 : kNowhere;
            if constexpr (!kAsync && !kKMajor) {
                if (shifted && at == rows / E) offset[i] = static_cast<uint32_t>(line * ld * B) + (rows - E) * B;
            }
        }
        if constexpr (!kAsync && !kKMajor) {
            // A tile of fewer rows than a unit's reaches back before its own first one.
            if (shifted && rows < E) {
                base -= E * B;
#pragma unroll
                for (int i = 0; i < kUnits; ++i) offset[i] += offset[i] == kNowhere ? 0 : E * B;
            }
        }
    }

    // v moved down by `bytes`, 2 to 14, zeros following.
    static __device__ __forceinline__ u32x4 shift_down(u32x4 v, int bytes) {
        const int words = bytes >> 2, bits = (bytes & 3) * 8;
        u32x4 r;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            uint32_t low = 0, high = 0;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                if (e + words == w) low = v[w];
                if (e + words + 1 == w) high = v[w];
            }
            r[e] = __builtin_amdgcn_alignbit(high, low, bits);
        }
        return r;
    }

    // The lane's units of the whole k-tile at k0.
    __device__ __forceinline__ void load(int64_t k0, int tid) {
        const char* at_k = base + (kKMajor ? k0 : k0 * ld) * B;
        const auto buffer = buffer_at(at_k);
#pragma unroll
        for (int i = 0; i < kUnits; ++i)
            held[i] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(buffer, offset[i], 0, 0));
        if constexpr (!kAsync && !kKMajor) {
            if (straddles && !shifted) load_edge(at_k, BK, tid);
        }
    }

    // The k-tile at k0 into the LDS stage at byte address `lds`, without waiting: kUnits loads a wave.
    // Of the last k-tile only `left` values of k exist; other calls have kWhole.  The loads are
    // written as assembly because the compiler makes every LDS read wait for all such loads; they
    // have no register results, and wait_loads() below waits for them.
    //
    // The hardware holds no load back for its scalar registers.  The compiler, which may form the
    // descriptor by v_readfirstlane, does not see that a load reads it, so the wait states stand in
    // the assembly: five between a vector instruction's scalar result and a load (the move to m0 and
    // s_nop 3), one between a write of m0 and a load into LDS.  8192 x 8192 x 8192 in bf16 takes
    // 817 us with them and 819 without.
    template <bool kWhole>
    __device__ __forceinline__ void load_async(int64_t k0, int64_t left, uint32_t lds, int tid, int wave) const {
        static_assert(kUnits == 2 || kUnits == 4, "the assembly below");
        const uint64_t at_k = reinterpret_cast<uint64_t>(base + (kKMajor ? k0 : k0 * ld) * B);
        const u32x4 buffer = {static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<uint32_t>(at_k))),
                              static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<uint32_t>(at_k >> 32))),
                              0x7FFFFFFFu, 0x00020000u};
        uint32_t from[kUnits];
#pragma unroll
        for (int i = 0; i < kUnits; ++i) {
            from[i] = offset[i];
            if constexpr (!kWhole) {
                const int u = i * THREADS + tid;
                if (!(kKMajor ? column(u) * E < left : u / kUnitsPerLine < left)) from[i] = kNowhere;
            }
        }
        const uint32_t to = __builtin_amdgcn_readfirstlane(lds + wave * 64 * 16);
        constexpr int kNext = THREADS * 16;  // bytes of LDS between a wave's units
        if constexpr (kUnits == 2) {
            asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\t"
                         "buffer_load_dwordx4 %1, %3, 0 offen lds\n\t"
                         "s_add_u32 m0, m0, %4\n\ts_nop 0\n\t"
                         "buffer_load_dwordx4 %2, %3, 0 offen lds"
                         :: "s"(to), "v"(from[0]), "v"(from[1]), "s"(buffer), "n"(kNext) : "memory", "m0", "scc");
        } else {
            asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\t"
                         "buffer_load_dwordx4 %1, %5, 0 offen lds\n\t"
                         "s_add_u32 m0, m0, %6\n\ts_nop 0\n\t"
                         "buffer_load_dwordx4 %2, %5, 0 offen lds\n\t"
                         "s_add_u32 m0, m0, %6\n\ts_nop 0\n\t"
                         "buffer_load_dwordx4 %3, %5, 0 offen lds\n\t"
                         "s_add_u32 m0, m0, %6\n\ts_nop 0\n\t"
                         "buffer_load_dwordx4 %4, %5, 0 offen lds"
                         :: "s"(to), "v"(from[0]), "v"(from[1]), "v"(from[2]), "v"(from[3]), "s"(buffer), "n"(kNext)
                         : "memory", "m0", "scc");
        }
    }

    // The lane's units of the k-tile at k0, of which only `left` values of k exist.
    __device__ __forceinline__ void load_part(int64_t k0, int left, int tid) {
        const char* at_k = base + (kKMajor ? k0 : k0 * ld) * B;
        const auto buffer = buffer_at(at_k);
#pragma unroll
        for (int i = 0; i < kUnits; ++i) {
            const int u = i * THREADS + tid, line = u / kUnitsPerLine, at = column(u);
            const bool in = kKMajor ? (at + 1) * E <= left : line < left;  // out of the rows: already nowhere
            held[i] = __builtin_bit_cast(
                u32x4, __builtin_amdgcn_raw_buffer_load_b128(buffer, in ? offset[i] : kNowhere, 0, 0));
        }
        if ((straddles && !shifted) || (kKMajor && left % E != 0)) load_edge(at_k, left, tid);
    }

    // Units that cross the last row or the last k, element by element.
    __device__ __forceinline__ void load_edge(const char* at_k, int left, int tid) {
#pragma unroll
        for (int i = 0; i < kUnits; ++i) {
            const int u = i * THREADS + tid, line = u / kUnitsPerLine, at = column(u);
            const int have = (kKMajor ? left : rows) - at * E;  // elements of the unit that exist
            const bool line_in = kKMajor ? line < rows : line < left;
            if (line_in && have > 0 && have < E) {
                u32x4 v = {0, 0, 0, 0};
                const int64_t first = line * ld + at * E;
#pragma unroll
                for (int e = 0; e < E - 1; ++e) {
                    if (e < have) {
                        if constexpr (B == 4) v[e] = reinterpret_cast<const uint32_t*>(at_k)[first + e];
                        else v[e / 2] |= static_cast<uint32_t>(reinterpret_cast<const uint16_t*>(at_k)[first + e])
                                         << (16 * (e % 2));
                    }
                }
                held[i] = v;
            }
        }
    }

    __device__ __forceinline__ void store(char* lds, int tid) {
        if constexpr (!kAsync && !kKMajor) {
            if (shifted) {
#pragma unroll
                for (int i = 0; i < kUnits; ++i)
                    if (column(i * THREADS + tid) == rows / E) held[i] = shift_down(held[i], 16 - rows % E * B);
            }
        }
#pragma unroll
        for (int i = 0; i < kUnits; ++i) {
            const int u = i * THREADS + tid, line = u / kUnitsPerLine, at = column(u) ^ swizzle(line);
            *reinterpret_cast<u32x4*>(lds + line * kLineBytes + (at << 4)) = held[i];
        }
    }

    // The fragment of rows [row, row + 16), k-units 4 * step .. 4 * step + 3 of the tile.
    static __device__ __forceinline__ u32x4 fragment(const char* lds, int row, int step, int lane) {
        const int q = step * 4 + (lane >> 4);
        if constexpr (kKMajor) {
            const int line = row + (lane & 15);
            return *reinterpret_cast<const u32x4*>(lds + line * kLineBytes + ((q ^ swizzle(line)) << 4));
        } else if constexpr (B == 2) {
            // A transposing read takes 4 values of k by 16 rows per quarter wave: lane i of it
            // addresses k = i / 4, rows 4 (i % 4) .. + 3, and receives row i's four values.
            const int i = lane & 15, line = q * 8 + (i >> 2), r = row + (i & 3) * 4;
            const int at = line * kLineBytes + (((r >> 3) ^ swizzle(line)) << 4) + (r & 7) * 2;
            using lds_ptr = __attribute__((address_space(3))) s16x4*;
            // line + 4 has the same swizzle, so the second half is four lines further.
            const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(const_cast<char*>(lds) + at));
            const s16x4 hi =
                __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(const_cast<char*>(lds) + at + 4 * kLineBytes));
            const u32x2 a = __builtin_bit_cast(u32x2, lo), b = __builtin_bit_cast(u32x2, hi);
            return u32x4{a[0], a[1], b[0], b[1]};
        } else {
            const int r = row + (lane & 15), line = q * 4;  // the four lines share a swizzle
            const char* at = lds + line * kLineBytes + (((r >> 2) ^ swizzle(line)) << 4) + (r & 3) * 4;
            u32x4 v;
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = *reinterpret_cast<const uint32_t*>(at + j * kLineBytes);
            return v;
        }
    }
};

// Waits until at most N of the wave's global loads are in flight, and for its LDS reads.
template <int N>
__device__ __forceinline__ void wait_loads() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" :: "n"(N) : "memory");
}

// A workgroup's tile: BM x BN by WM x WN waves, with kStages_ LDS stages for asynchronous loads.
template <int BM_, int BN_, int WM_, int WN_, int kStages_>
struct Tile {
    static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, kThreads = 64 * WM * WN, kStages = kStages_;
    static constexpr int TM = BM / WM / 16, TN = BN / WN / 16;  // 16 x 16 results per wave
    static constexpr int kStageBytes = (BM + BN) * 128;
};

template <class T, bool kAsync>
constexpr int lds_bytes() { return (kAsync ? T::kStages : 2) * T::kStageBytes; }

// N fragments of consecutive sixteens of rows.
template <class Op, int N>
__device__ __forceinline__ void read(u32x4 (&f)[N], const char* lds, int row, int step, int lane) {
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = Op::fragment(lds, row + 16 * i, step, lane);
}
template <int D, class T, int kFirst, int N>
__device__ __forceinline__ void multiply(const u32x4 (&a)[N], const u32x4 (&b)[T::TN], f32x4 (&acc)[T::TM][T::TN]) {
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int j = 0; j < T::TN; ++j) acc[kFirst + i][j] = mma<D>(b[j], a[i], acc[kFirst + i][j]);
}
// Asks the scheduler to spread LDS reads among matrix instructions.
template <int kReads, int kMmas>
__device__ __forceinline__ void interleave() {
#pragma unroll
    for (int i = 0; i < kReads; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);  // an LDS read
        __builtin_amdgcn_sched_group_barrier(0x008, kMmas / kReads > 0 ? kMmas / kReads : 1, 0);
    }
}

// Forms the tile at rows m0 of A and n0 of B over k in [k0, k1) into acc: acc[i][j] holds, in
// lane l, element m = 16 i + l % 16, n = 16 j + 4 (l / 16) + r (r = 0..3) of the wave's part.
// A partial k-tile comes last among asynchronous loads, so that the others start on whole units,
// and first among those through registers, whose loop then moves whole ones.
template <int D, bool kA, bool kB, class T, bool kAsync>
__device__ __forceinline__ void tile_product(const void* a, int64_t lda, int64_t m0, int64_t m_count, const void* b,
                                             int64_t ldb, int64_t n0, int64_t n_count, int64_t k0, int64_t k1,
                                             char* lds, f32x4 (&acc)[T::TM][T::TN]) {
    constexpr int BK = tile_k<D>(), B = elem_bytes<D>(), kThreads = T::kThreads;
    using OpA = Operand<D, kA, T::BM, kThreads, kAsync>;
    using OpB = Operand<D, kB, T::BN, kThreads, kAsync>;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int wm = (wave / T::WN) * (T::BM / T::WM), wn = (wave % T::WN) * (T::BN / T::WN);
#pragma unroll
    for (int i = 0; i < T::TM; ++i)
#pragma unroll
        for (int j = 0; j < T::TN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (k0 >= k1) return;
    OpA oa;
    OpB ob;
    oa.init(a, lda, m0, m_count, tid);
    ob.init(b, ldb, n0, n_count, tid);
    const int tiles = static_cast<int>((k1 - k0 + BK - 1) / BK);
    int64_t k = k0;  // the next k-tile to load
    constexpr int kStages = kAsync ? T::kStages : 2, kLoads = OpA::kUnits + OpB::kUnits, kAhead = kStages - 1;
    const uint32_t at = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char*)lds));
    const auto issue = [&](int stage) {  // asynchronous
        const uint32_t to_a = at + stage * T::kStageBytes, to_b = to_a + OpA::kBytes;
        if (k1 - k >= BK) {
            oa.template load_async<true>(k, BK, to_a, tid, wave);
            ob.template load_async<true>(k, BK, to_b, tid, wave);
        } else {
            oa.template load_async<false>(k, k1 - k, to_a, tid, wave);
            ob.template load_async<false>(k, k1 - k, to_b, tid, wave);
        }
        k += BK;
    };
    const auto load = [&]() {  // into registers
        oa.load(k, tid);
        ob.load(k, tid);
        k += BK;
    };
    const auto store = [&](int stage) {
        oa.store(lds + stage * T::kStageBytes, tid);
        ob.store(lds + stage * T::kStageBytes + OpA::kBytes, tid);
    };
    if constexpr (kAsync) {
        issue(0);
#pragma unroll
        for (int s = 1; s <= kAhead; ++s)
            if (s < tiles) issue(s);
        if (kAhead < tiles) wait_loads<kLoads * kAhead>();
        else wait_loads<0>();
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    } else {
        const int part = static_cast<int>((k1 - k0) % BK);
        if (part != 0) {
            oa.load_part(k, part, tid);
            ob.load_part(k, part, tid);
            k += part;
        } else {
            load();
        }
        store(0);
        if (tiles > 1) load();
        __syncthreads();
    }
    // Each k-tile is two steps of two halves of the wave's rows.  While one half's matrix
    // instructions run, the fragments of the next are read: two sets of each operand's are held.
    constexpr int kHalf = T::TM / 2, kReadsA = OpA::kReads * kHalf, kReadsB = OpB::kReads * T::TN;
    constexpr int kMmas = kHalf * T::TN * (B == 4 ? 4 : 1);
    u32x4 a0[kHalf], a1[kHalf], b0[T::TN], b1[T::TN];
    read<OpB>(b0, lds + OpA::kBytes, wn, 0, lane);
    read<OpA>(a0, lds, wm, 0, lane);
    int stage = 0;
    for (int t = 0; t < tiles; ++t) {
        const char* now = lds + stage * T::kStageBytes;
        read<OpA>(a1, now, wm + 16 * kHalf, 0, lane);
        multiply<D, T, 0>(a0, b0, acc);
        interleave<kReadsA, kMmas>();
        if constexpr (!kAsync) {
            // Every wave has passed the barrier that ended the reads of the other stage.
            if (t + 1 < tiles) {
                store(stage ^ 1);
                if (t + 2 < tiles) load();
            }
        }
        read<OpB>(b1, now + OpA::kBytes, wn, 1, lane);
        read<OpA>(a0, now, wm, 1, lane);
        multiply<D, T, kHalf>(a1, b0, acc);
        interleave<kReadsA + kReadsB, kMmas>();
        read<OpA>(a1, now, wm + 16 * kHalf, 1, lane);
        multiply<D, T, 0>(a0, b1, acc);
        interleave<kReadsA, kMmas>();
        if (t + 1 < tiles) {
            if constexpr (kAsync) {
                // At most the kAhead - 1 tiles after t + 1 are in flight, so it has landed; past the
                // barrier it has for every wave, and every wave holds the last of tile t, whose
                // stage the next load takes.
                if (t + 1 + kAhead <= tiles) wait_loads<kLoads * (kAhead - 1)>();
                else wait_loads<0>();
                __builtin_amdgcn_s_barrier();
                asm volatile("" ::: "memory");
                if (t + 1 + kAhead < tiles) issue(stage);
            } else {
                __syncthreads();
            }
            stage = stage + 1 == kStages ? 0 : stage + 1;
            const char* next = lds + stage * T::kStageBytes;
            read<OpB>(b0, next + OpA::kBytes, wn, 0, lane);
            read<OpA>(a0, next, wm, 0, lane);
        }
        multiply<D, T, kHalf>(a1, b1, acc);
        interleave<kReadsA + kReadsB, kMmas>();
    }
    __syncthreads();  // the LDS is free
}

// Finishes the tile, four consecutive n of a row at a time: `load(m, n)` fetches what the result
// is combined with, `store(m, n, v, loaded)` stores it and returns the value kept.  The
// accumulators pass through LDS (free by now), so that this code stands once and a wave's loads
// and stores cover whole rows; a lane issues the loads of up to kMostBatch units before it uses the first.
//
// `mirror(n, m, v)`, unless it is NoMirror or `mirrored` is false, then gets the kept values
// transposed, four consecutive m at a time: a wave takes sixteen n by four units of m, so its
// LDS reads fall on distinct banks and its stores cover 32 bytes of a row.
struct NoMirror {};
template <class T, bool kAsync, int kMostBatch, class Load, class Store, class Mirror = NoMirror>
__device__ __forceinline__ void finish_tile(char* lds, const f32x4 (&acc)[T::TM][T::TN], Load&& load, Store&& store,
                                            bool mirrored = false, Mirror&& mirror = Mirror{}) {
    constexpr bool kMirror = !std::is_same_v<std::decay_t<Mirror>, NoMirror>;
    constexpr int kRowUnits = T::BN / 4, kPhases = T::BM * T::BN * 4 > lds_bytes<T, kAsync>() ? T::WM : 1;
    constexpr int kRows = T::BM / kPhases, kUnits = kRows * kRowUnits / T::kThreads, kBatch = kUnits < kMostBatch ? kUnits : kMostBatch;
    static_assert(kRows * T::BN * 4 <= lds_bytes<T, kAsync>(), "a phase fits the tile's LDS");
    static_assert(kRows * kRowUnits % (T::kThreads * kBatch) == 0, "whole batches");
    using Loaded = decltype(load(0, 0));
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int wm = (wave / T::WN) * (T::BM / T::WM), wn = (wave % T::WN) * (T::BN / T::WN);
    f32x4* out = reinterpret_cast<f32x4*>(lds);
#pragma unroll
    for (int phase = 0; phase < kPhases; ++phase) {
        if (phase > 0) __syncthreads();
        if (kPhases == 1 || wave / T::WN == phase) {
#pragma unroll
            for (int i = 0; i < T::TM; ++i)
#pragma unroll
                for (int j = 0; j < T::TN; ++j) {
                    const int m = wm - phase * kRows + 16 * i + (lane & 15), unit = wn / 4 + 4 * j + (lane >> 4);
                    out[m * kRowUnits + (unit ^ (m & 15))] = acc[i][j];
                }
        }
        __syncthreads();
#pragma unroll 1
        for (int first = tid; first < kRows * kRowUnits; first += kBatch * T::kThreads) {
            Loaded loaded[kBatch];
#pragma unroll
            for (int b = 0; b < kBatch; ++b) {
                const int u = first + b * T::kThreads;
                loaded[b] = load(phase * kRows + u / kRowUnits, u % kRowUnits * 4);
            }
#pragma unroll
            for (int b = 0; b < kBatch; ++b) {
                const int u = first + b * T::kThreads, m = u / kRowUnits, unit = u % kRowUnits;
                f32x4& at = out[m * kRowUnits + (unit ^ (m & 15))];
                const f32x4 kept = store(phase * kRows + m, unit * 4, at, loaded[b]);
                if constexpr (kMirror) {
                    if (mirrored) at = kept;
                }
            }
        }
        if constexpr (kMirror) {
            if (mirrored) {
                __syncthreads();
                const float* flat = reinterpret_cast<const float*>(lds);
#pragma unroll 4
                for (int u = tid; u < T::BN * kRows / 4; u += T::kThreads) {
                    const int block = u >> 6, n = block % (T::BN / 16) * 16 + (u & 15);
                    const int m = (block / (T::BN / 16) * 4 + ((u >> 4) & 3)) * 4;
                    f32x4 v;
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        v[e] = flat[((m + e) * kRowUnits + ((n >> 2) ^ ((m + e) & 15))) * 4 + (n & 3)];
                    mirror(n, phase * kRows + m, v);
                }
            }
        }
    }
}

// ---- the order of tiles --------------------------------------------------------------
// Workgroup b of `count` as a tile index such that each XCD (workgroups b mod 8) takes one
// run of consecutive tiles: neighbours share their operands in that XCD's L2.
__device__ __forceinline__ int xcd_tile(int b, int count) {
    const int xcd = b & 7, q = count >> 3, r = count & 7;
    return xcd * q + min(xcd, r) + (b >> 3);
}
// Tile t of a tiles_m x tiles_n grid, in bands of kBand tile rows walked column by column.
template <int kBand>
__device__ __forceinline__ void band_order(int t, int tiles_m, int tiles_n, int& m, int& n) {
    const int width = kBand * tiles_n, band = t / width, first = band * kBand;
    const int height = min(tiles_m - first, kBand), within = t - band * width;
    m = first + within % height;
    n = within / height;
}

// ---- launches ------------------------------------------------------------------------
// Lets `kernel` use `bytes` of dynamic LDS on the current device, once for each device (`done`, a
// bit a device, belongs to the kernel).
inline int32_t allow_lds(const char* who, const void* kernel, int bytes, std::atomic<uint64_t>& done) {
    int device = 0;
    const int32_t status = check_hip(hipGetDevice(&device), who);
    if (status != HBT_OK) return status;
    const uint64_t bit = uint64_t(1) << (device & 63);
    if (device < 64 && (done.load(std::memory_order_acquire) & bit) != 0) return HBT_OK;
    const int32_t set = check_hip(hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes), who);
    if (set == HBT_OK) done.fetch_or(bit, std::memory_order_release);
    return set;
}

// ---- the choice of a tile ---------------------------------------------------------------
using Tile256 = Tile<256, 256, 2, 4, 2>;
using Tile128 = Tile<128, 128, 2, 2, 2>;
using Tile64 = Tile<64, 64, 2, 2, 4>;

// An estimate, in microseconds, of `tiles` workgroups of `size` x `size` results with `steps`
// k-tiles each: rounds of the device times a round's length.  Larger tiles read less per product
// (bf16, 4096^3: 108 us in tiles of 256, 124 of 128, 206 of 64); smaller ones fill the device
// with less, and a CU's two workgroups of 128 or 64 hide each other's first loads and stores
// (2048 x 768 by 768: 27, 14 and 9 us).  `fixed`: what a round costs beside its k-tiles.
// Round lengths are fitted to such measurements over 17 shapes (256 CUs, one workgroup of 256 or
// two of the others a CU), within about a fifth.
inline double round_cost(int size, int64_t tiles, double steps, bool f32, double fixed) {
    constexpr int64_t kCus = 256;
    if (size == 256) return static_cast<double>((tiles + kCus - 1) / kCus) * (steps * 1.5 + fixed);
    const bool alone = tiles <= kCus;  // one workgroup a CU has the matrix cores for itself
    if (f32) {  // the matrix cores are the bound: workgroups of a CU take turns
        const double step = size == 128 ? (alone ? 2.25 : 1.87) : (alone ? 0.7 : 0.52);
        return static_cast<double>((tiles + kCus - 1) / kCus) * steps * step + fixed;
    }
    const double step = size == 128 ? (alone ? 0.7 : 0.98) : 0.41;
    return static_cast<double>((tiles + 2 * kCus - 1) / (2 * kCus)) * (steps * step + fixed);
}

}  // namespace mm
}  // namespace hbt
