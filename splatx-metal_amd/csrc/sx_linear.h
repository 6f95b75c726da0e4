// sx_linear.h — linear layers over rows, forward and backward, all rows with one weight or groups of rows with their own
// (include/splatx_hip.h has the formulas): the kernels and their launches for one type of elements, each type a file of its own
// (k_linear_f32.hip, k_linear_bf16.hip, k_linear_f16.hip), which build side by side.
#pragma once

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>
#include <stdexcept>
#include <type_traits>

#include "sx_linear_plan.h"
#include "sx_mma.h"

namespace sxk {
using namespace sxd;
namespace {

// A barrier for what lies in LDS: unlike __syncthreads it does not wait for the wave's loads and stores of memory.
__device__ inline void lds_barrier() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}
// Until of the wave's loads and stores of memory only the last N (63: any) are on their way, and none of LDS.
template <int N>
__device__ inline void wait_for() {
    static_assert(N < 64);
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt((N & 15) | (N >> 4) << 14 | 7 << 4);
    asm volatile("" ::: "memory");
}
// What has been loaded is there from here on. Loads and stores of memory are counted together, so that a wait for loads that
// comes after stores waits for these as well: the wait comes before them.
template <class T, int N>
__device__ inline void arrived(Vec<T, kPer<T>> (&v)[N]) {
    using Words = uint32_t __attribute__((ext_vector_type(4)));
#pragma unroll
    for (int i = 0; i < N; i++) {
        Words w = __builtin_bit_cast(Words, v[i]);
        asm volatile("" : "+v"(w));
        v[i] = __builtin_bit_cast(Frag<T>, w);
    }
}

// The wave's number in its workgroup, known to be one for all its lanes.
__device__ inline int wave_of() { return __builtin_amdgcn_readfirstlane(threadIdx.x / 64); }

// ---- tiles ------------------------------------------------------------------------------------------------
//
// out[r][c] = sum over d of row(r, d) col(c, d): x W^T, dz W and dz^T x, each operand either with its sums' elements side by
// side in memory (plain) or with its rows side by side (Across: W's columns, dz's and x's).

// What follows the sums, of rows of `cols` columns.
struct Finish {
    void* out;
    int64_t out_stride, cols;
    const void* residual;
    int64_t residual_stride;
    void* pre;
    int64_t pre_stride;
    int act;
    bool clear;  // rows behind the last group become zero
};

struct TileArgs {
    const void *row, *col;
    int64_t row_stride, col_stride;  // elements between the rows in memory
    int64_t col_group;               // elements between the groups' col operands
    int64_t row_width, col_width;    // of an Across operand's rows in memory, whole fragments
    Finish to;                       // (its cols are the outputs')
    int64_t out_group;
    int64_t rows, depth;             // rows (of the products over rows), depth (of those over groups' rows): all groups'
    Groups groups;
    int shift;                       // the parts' rows, log2
    int64_t slots;
    float* partial;                  // [slabs][rows][cols] in place of out, or null
    int64_t split;                   // depth of a slab
    int splits;
    const void* bias;
    int64_t bias_group;
};

// Where the 16 bytes (row r, chunk c) of a plain operand's tile lie: 128 bytes a row, one chunk of sixteen rows in sixteen places of
// 256 bytes, so that lanes that read one chunk of several rows read different banks.
__device__ inline int plain_at(int r, int c) { return r * 128 + (c ^ (r >> 1 & 7)) * 16; }
// Of an Across operand's tile: `row_bytes` (128 or a multiple of 256) a row of the sums' dimension; the 64 bytes that thirty-two
// lanes read of each of four rows in different places of 256 bytes.
template <class T>
__device__ inline int across_at(int m, int byte, int row_bytes) {
    return m * row_bytes + (sizeof(T) == 4 ? byte : row_bytes == 128 ? byte ^ ((m >> 1 & 1) << 6) : byte ^ ((m & 3) << 6));
}

// A thread's part of an operand's tile, R rows by 128 bytes of the sums' dimension, on its way from memory to LDS.
template <class T, int R, bool Across, int Threads>
struct Stage {
    static constexpr int V = kPer<T>, kDepth = 128 / static_cast<int>(sizeof(T));
    static constexpr int kPerLine = Across ? R / V : 8;  // chunks of a line in memory
    static constexpr int kLines = Threads / kPerLine, N = R * 8 / Threads;
    static_assert(Threads % kPerLine == 0 && R * 8 % Threads == 0);
    Frag<T> v[N];
    const T* base;
    int64_t stride, first, limit;
    int chunk, line;

    // Rows [first, limit) (clamped, of a plain operand; columns of the memory's rows else)
    __device__ Stage(const T* b, int64_t s, int64_t f, int64_t l) : base(b), stride(s), first(f), limit(l) {
        chunk = threadIdx.x % kPerLine;
        line = threadIdx.x / kPerLine;
    }
    // Of the sums' dimension [d, d + kDepth), zeros from `end` on. (In a tile that ends inside its operand all loads go out
    // together; a branch for each would wait for each.)
    __device__ void load(int64_t d, int64_t end) {
        const int64_t width = Across ? limit : end;
        const bool inside = d + kDepth <= end && (!Across || first + R <= limit);
#pragma unroll
        for (int i = 0; i < N; i++) {
            const int l = line + i * kLines;
            if constexpr (Across) {
                const T* const p = base + min(d + l, end - 1) * stride;
                if (inside) v[i] = load_raw<V>(p + first + chunk * V);
                else if (width >= V) v[i] = load_clamped(p, first + chunk * V, limit);
                else v[i] = load_within(p, first + chunk * V, limit);
                if (!inside && d + l >= end) v[i] = Frag<T>(0);
            } else {
                const T* const p = base + min(first + l, limit - 1) * stride;
                if (inside) v[i] = load_raw<V>(p + d + chunk * V);
                else if (width >= V) v[i] = load_clamped(p, d + chunk * V, end);
                else v[i] = load_within(p, d + chunk * V, end);
            }
        }
    }
    __device__ void store(char* lds) const {
#pragma unroll
        for (int i = 0; i < N; i++) {
            const int l = line + i * kLines;
            const int at = Across ? across_at<T>(l, chunk * 16, R * static_cast<int>(sizeof(T))) : plain_at(l, chunk);
            *reinterpret_cast<Frag<T>*>(lds + at) = v[i];
        }
    }
};

// The same straight from memory into LDS, of whole tiles whose lines begin on 16 bytes: a wave's load fills 1 KiB of LDS in the
// order of the lanes, so that it is the lane's place in memory that goes by where the chunk lies. A plain operand's eight lines
// of a load have a beginning of their own: those of the whole tile may be further apart than 32 bits reach.
template <class T, int R, bool Across, int Threads>
struct DirectStage {
    static constexpr int V = kPer<T>, kDepth = kTileDepthBytes / static_cast<int>(sizeof(T)), N = R * 8 / Threads;
    static_assert(kTileDepthBytes * kLoadLines == 64 * 16);
    const char* base[Across ? 1 : N];
    int64_t step;        // bytes to the next tile
    uint32_t offset[N];  // of the lane's chunks
    // As Stage's; `d` the sums' first element
    __device__ DirectStage(const T* b, int64_t s, int64_t f, int64_t l, int64_t d) {
        const int64_t line = s * static_cast<int64_t>(sizeof(T));
        const char* const from = reinterpret_cast<const char*>(b);
        step = Across ? kDepth * line : kTileDepthBytes;
        if constexpr (Across) base[0] = from + d * line;
#pragma unroll
        for (int i = 0; i < N; i++) {
            if constexpr (Across) {
                constexpr int kLine = R * static_cast<int>(sizeof(T));
                const int at = (i * Threads + static_cast<int>(threadIdx.x)) * 16;  // in the tile
                const int m = at / kLine, byte = across_at<T>(m, at % kLine, kLine) - m * kLine;
                offset[i] = static_cast<uint32_t>(
                    across_offset(m, line, min(f * static_cast<int64_t>(sizeof(T)) + byte, (l - V) * static_cast<int64_t>(sizeof(T)))));
            } else {
                const int first = i * Threads / 8 + wave_of() * kLoadLines, r = first + static_cast<int>(threadIdx.x) % 64 / 8;
                const int64_t last = l - 1 - f, start = min(int64_t{first}, last);
                base[i] = from + (f + start) * line + d * static_cast<int64_t>(sizeof(T));
                offset[i] = static_cast<uint32_t>(plain_offset(min(int64_t{r}, last) - start, line, static_cast<int>(threadIdx.x) % 8 ^ (r >> 1 & 7)));
            }
        }
    }
    __device__ void load(char* lds) {
        using Global = __attribute__((address_space(1))) const void*;
        using Lds = __attribute__((address_space(3))) void*;
#pragma unroll
        for (int i = 0; i < N; i++) {
            const char* const p = base[Across ? 0 : i];
            __builtin_amdgcn_global_load_lds((Global)(p + offset[i]), (Lds)(lds + (i * Threads + wave_of() * 64) * 16), 16, 0, 0);
            if constexpr (!Across) base[i] += step;
        }
        if constexpr (Across) base[0] += step;
    }
};

// The lane's fragment of rows [r, r + 32), step s of the tile's four.
template <class T, int R, bool Across>
__device__ inline Frag<T> fragment(const char* lds, int r, int s) {
    const int lane = threadIdx.x % 64, half = lane / 32;
    if constexpr (!Across) {
        return *reinterpret_cast<const Frag<T>*>(lds + plain_at(r + lane % 32, 2 * s + half));
    } else if constexpr (sizeof(T) == 4) {
        Frag<T> f;
#pragma unroll
        for (int i = 0; i < 4; i++) f[i] = *reinterpret_cast<const float*>(lds + across_at<T>(s * 8 + half * 4 + i, (r + lane % 32) * 4, R * 4));
        return f;
    } else {
        // sixteen lanes read four lines of sixteen columns and get a column each
        using Four = short __attribute__((ext_vector_type(4)));
        using Lds = __attribute__((address_space(3))) Four*;
        const int group = lane % 16, column = r + (lane % 32) / 16 * 16 + group % 4 * 4;
        Four part[2];
#pragma unroll
        for (int j = 0; j < 2; j++)
            part[j] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (Lds)(lds + across_at<T>(s * 16 + half * 8 + j * 4 + group / 4, column * 2, R * 2)));
        return __builtin_bit_cast(Frag<T>, __builtin_shufflevector(part[0], part[1], 0, 1, 2, 3, 4, 5, 6, 7));
    }
}

template <class T, int V>
__device__ inline Floats<V> load_some(const T* p, int n) {
    if (n >= V) return floats<T, V>(load_raw<V>(p));
    Floats<V> v(0.0f);
#pragma unroll
    for (int e = 0; e < V; e++)
        if (e < n) v[e] = static_cast<float>(p[e]);
    return v;
}
template <class T, int V>
__device__ inline void store_some(T* p, Floats<V> v, int n) {
    if (n >= V) {
        store_raw<V>(p, raw<T, V>(v));
        return;
    }
#pragma unroll
    for (int e = 0; e < V; e++)
        if (e < n) p[e] = static_cast<T>(v[e]);
}

// Four columns from c on of row r, bias included.
template <class T>
__device__ inline void finish4(const Finish& a, int64_t r, int64_t c, Floats<4> v) {
    const int n = static_cast<int>(min(a.cols - c, int64_t{4}));
    if (n <= 0) return;
    if (a.pre) store_some<T, 4>(static_cast<T*>(a.pre) + r * a.pre_stride + c, v, n);
    activate<T, 4>(v, a.act);
    if (a.residual) v += load_some<T, 4>(static_cast<const T*>(a.residual) + r * a.residual_stride + c, n);
    store_some<T, 4>(static_cast<T*>(a.out) + r * a.out_stride + c, v, n);
}
// The same of a row behind the last group.
template <class T>
__device__ inline void clear4(const Finish& a, int64_t r, int64_t c) {
    const int n = static_cast<int>(min(a.cols - c, int64_t{4}));
    if (n <= 0 || !a.clear) return;
    store_some<T, 4>(static_cast<T*>(a.out) + r * a.out_stride + c, Floats<4>(0.0f), n);
    if (a.pre) store_some<T, 4>(static_cast<T*>(a.pre) + r * a.pre_stride + c, Floats<4>(0.0f), n);
}

// A wave's outputs go through LDS of its own as floats, so that a store has whole lines of eight rows: from the sums' layout (a
// lane has four columns of its row in each place) to memory's, 32 rows of 128 bytes of the type, of which a lane takes 16 at a
// time through what follows the sums. (Stores of 16 bytes a row from the registers, the rows' lines in four parts: a layer of
// 64 outputs took twice as long.)
template <class T>
constexpr int kUnitTiles = unit_tiles(sizeof(T));
template <class T>
constexpr int kUnitLine = unit_line(sizeof(T));
template <class T>
constexpr int kUnitBytes = unit_bytes(sizeof(T));

// What lanes of the wave have written to LDS is there for the others.
__device__ inline void wave_sees() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

template <class T>
__device__ inline void store_chunk(T* p, Floats<kPer<T>> f, int n) {
    const Frag<T> v = raw<T, kPer<T>>(f);
    if (n == kPer<T>) {
        store_raw<kPer<T>>(p, v);
        return;
    }
#pragma unroll
    for (int e = 0; e < kPer<T> - 1; e++)
        if (e < n) p[e] = v[e];
}

// 32 rows from r on (those before `stop`) and the columns [c, c + 128 bytes). Every lane takes part.
template <class T>
struct Unit {
    static constexpr int V = kPer<T>;
    const Finish* f;
    int64_t r, c;
    int column, row, n, rows;
    Frag<T> residual[4];

    __device__ Unit(const Finish& a, int64_t first, int64_t stop, int64_t col) : f(&a), r(first), c(col) {
        column = threadIdx.x % 8 * V;
        row = threadIdx.x % 64 / 8;
        n = static_cast<int>(max(int64_t{0}, min(a.cols - c - column, int64_t{V})));
        rows = static_cast<int>(min(stop - r, int64_t{32}));
        if (a.residual && rows > 0 && a.cols > c)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const T* const p = static_cast<const T*>(a.residual) + (r * a.residual_stride + c) + min(row + 8 * i, rows - 1) * a.residual_stride;
                residual[i] = a.cols - c >= 8 * V ? load_raw<V>(p + column) : a.cols - c >= V ? load_clamped(p, column, a.cols - c) : load_within(p, column, a.cols - c);
            }
    }
    // (what all lanes share is added apart from what a lane has of its own, which stays over the units)
    template <class P>
    __device__ P* at(P* p, int64_t stride) const { return p + (r * stride + c) + (row * stride + column); }

    // The sums, bias included, through the wave's LDS.
    __device__ void finish(const Sums (&sums)[kUnitTiles<T>], char* lds) const {
        const Finish& a = *f;
        const int lane = threadIdx.x % 64;
        wave_sees();  // (what was there has been read)
#pragma unroll
        for (int u = 0; u < kUnitTiles<T>; u++)
#pragma unroll
            for (int q = 0; q < 4; q++)
                *reinterpret_cast<Floats<4>*>(lds + lane % 32 * kUnitLine<T> + lane / 32 * 16 + u * 128 + q * 32) =
                    Floats<4>{sums[u][4 * q], sums[u][4 * q + 1], sums[u][4 * q + 2], sums[u][4 * q + 3]};
        wave_sees();
        T* out = at(static_cast<T*>(a.out), a.out_stride);
        T* pre = a.pre ? at(static_cast<T*>(a.pre), a.pre_stride) : nullptr;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            Floats<V> v;
#pragma unroll
            for (int e = 0; e < V; e += 4) {
                const Floats<4> f = *reinterpret_cast<const Floats<4>*>(lds + (row + 8 * i) * kUnitLine<T> + column * 4 + e * 4);
                v[e] = f[0]; v[e + 1] = f[1]; v[e + 2] = f[2]; v[e + 3] = f[3];
            }
            if (a.pre) {
                if (row + 8 * i < rows) store_chunk(pre, v, n);
                pre += 8 * a.pre_stride;
            }
            activate<T, V>(v, a.act);
            if (a.residual) v += floats<T, V>(residual[i]);
            if (row + 8 * i < rows) store_chunk(out, v, n);
            out += 8 * a.out_stride;
            __builtin_amdgcn_sched_barrier(0);  // (one after another: their registers together would cost waves)
        }
    }
};

// The same of sums that are the outputs, through half the LDS.
template <class T>
__device__ inline void store_unit(const Finish& a, int64_t r, int64_t stop, int64_t c, const Sums (&sums)[kUnitTiles<T>], char* lds) {
    constexpr int V = kPer<T>;
    const int lane = threadIdx.x % 64;
    wave_sees();
#pragma unroll
    for (int u = 0; u < kUnitTiles<T>; u++)
#pragma unroll
        for (int q = 0; q < 4; q++)
            *reinterpret_cast<Vec<T, 4>*>(lds + lane % 32 * kBareLine + (u * 32 + 8 * q + lane / 32 * 4) * static_cast<int>(sizeof(T))) =
                raw<T, 4>(Floats<4>{sums[u][4 * q], sums[u][4 * q + 1], sums[u][4 * q + 2], sums[u][4 * q + 3]});
    wave_sees();
    const int column = lane % 8 * V, row = lane / 8;
    const int n = static_cast<int>(max(int64_t{0}, min(a.cols - c - column, int64_t{V})));
    const int rows = static_cast<int>(min(stop - r, int64_t{32}));
    T* p = static_cast<T*>(a.out) + (r * a.out_stride + c) + (row * a.out_stride + column);
#pragma unroll
    for (int i = 0; i < 32; i += 8, p += 8 * a.out_stride) {
        const Frag<T> v = *reinterpret_cast<const Frag<T>*>(lds + (row + i) * kBareLine + lane % 8 * 16);
        if (row + i >= rows) continue;
        if (n == V) store_raw<V>(p, v);
        else
#pragma unroll
            for (int e = 0; e < V - 1; e++)
                if (e < n) p[e] = v[e];
    }
}

// BR x BC outputs a workgroup, WR x WC a wave. OverRows: the sums go over a group's rows (dW), else the outputs' rows are the
// groups' rows. Bound by the matrix cores, and of long sums by the power they take (1.6 GHz, 64 % of the cycles a product on its
// way): 16,383 rows, 8192 to 2048 half with a residual 505 us, 1.09 PFLOP/s (the library's bare product 457); of 2048 to 4096 dx
// 290 us and dweight 291 (the library 272 and 330); 20,001 rows in 16 groups, 1024 to 1408, bfloat16 90 us. Floats of 4096 cubed
// 978 us, 140 TFLOP/s (the library 910).
// Staged: the operands lie anywhere and go through registers.
template <class T, int BR, int BC, int WR, int WC, bool RowAcross, bool ColAcross, bool Staged>
__global__ void __launch_bounds__(BR / WR * (BC / WC) * 64) k_tile(TileArgs a) {
    constexpr bool OverRows = RowAcross;
    constexpr int kWaves = BR / WR * (BC / WC), kThreads = kWaves * 64, kDepth = 128 / static_cast<int>(sizeof(T));
    constexpr int kBuffer = (BR + BC) * 128, I = WR / 32, J = WC / 32;
    // (two arrays, so that a load into one is seen to be no store into the other)
    __shared__ __attribute__((aligned(128))) char lds[kBuffer], lds1[kBuffer];
    // Which tile: workgroups go round the eight dies, and each die takes tiles side by side, eight rows of tiles at a time. A slab
    // begins with a die of its own: where it has fewer than eight tiles the others would have no work. (Floats, 919,424 rows of 32
    // in 4 groups, gradients of 144 outputs: 1,900 us without, 1,527 so.)
    const int64_t across = (a.to.cols + BC - 1) / BC, down = OverRows ? (a.rows + BR - 1) / BR : a.slots, tiles = across * down;
    const int64_t each = (tiles + 7) / 8, tile = (blockIdx.x + blockIdx.y) % 8 * each + blockIdx.x / 8;
    if (blockIdx.x / 8 >= each || tile >= tiles) return;
    const int64_t band = tile / (8 * across), height = min(down - band * 8, int64_t{8});
    const int64_t tr = band * 8 + (tile - band * 8 * across) % height, tc = (tile - band * 8 * across) / height;

    const Part part = part_of(a.groups, OverRows ? blockIdx.y : tr, a.shift);
    int64_t r0, r1, d0, d1;
    const int64_t c0 = tc * BC;
    if constexpr (OverRows) {
        r0 = tr * BR;
        r1 = a.rows;
        d0 = part.begin;
        d1 = part.end;
        if (part.group >= a.groups.groups || (a.partial && d0 >= d1)) return;
    } else {
        r0 = part.begin;
        r1 = part.end;
        d0 = blockIdx.y * a.split;
        d1 = min(a.depth, d0 + a.split);
        if (r0 >= r1) return;
    }
    const int wave = wave_of(), lane = threadIdx.x % 64;
    const int wr = wave / (BC / WC) * WR, wc = wave % (BC / WC) * WC;
    if (!OverRows && part.group >= a.groups.groups) {
        if (a.partial) return;
        for (int64_t r = r0 + threadIdx.x / 32; r < r1; r += kThreads / 32)
            for (int c = threadIdx.x % 32 * 4; c < BC; c += 128) clear4<T>(a.to, r, c0 + c);
        return;
    }
    // (the bias of the tile's columns, a thread's one, goes to LDS in the end)
    float own_bias = 0.0f;
    if (a.bias && threadIdx.x < BC && c0 + threadIdx.x < a.to.cols)
        own_bias = static_cast<float>(static_cast<const T*>(a.bias)[part.group * a.bias_group + c0 + threadIdx.x]);
    Sums sums[I][J];
#pragma unroll
    for (int i = 0; i < I; i++)
#pragma unroll
        for (int j = 0; j < J; j++) sums[i][j] = Sums(0.0f);
    const T *const rows_from = static_cast<const T*>(a.row), *const cols_from = static_cast<const T*>(a.col) + part.group * a.col_group;
    const int64_t row_end = RowAcross ? a.row_width : r1, col_end = ColAcross ? a.col_width : a.to.cols;
    {
        // The fragments of a step are read while the products of the step before it run, also over the end of a tile: when the
        // last step's are there the tile's place in LDS is free, and the next tile's loads, as long on their way as a tile's
        // products take, have landed.
        Frag<T> fr[2][I], fc[2][J];
        const auto read = [&](int to, const char* buffer, int s) {
#pragma unroll
            for (int i = 0; i < I; i++) fr[to][i] = fragment<T, BR, RowAcross>(buffer, wr + i * 32, s);
#pragma unroll
            for (int j = 0; j < J; j++) fc[to][j] = fragment<T, BC, ColAcross>(buffer + BR * 128, wc + j * 32, s);
        };
        const auto product = [&](int of) {
#pragma unroll
            for (int i = 0; i < I; i++)
#pragma unroll
                for (int j = 0; j < J; j++) mma(sums[i][j], fc[of][j], fr[of][i]);
        };
        if constexpr (Staged) {
            // A tile's chunks are on their way while the products of the tile before it run; one barrier a tile, for the place that is
            // written was read before the last one.
            Stage<T, BR, RowAcross, kThreads> rows(rows_from, a.row_stride, r0, row_end);
            Stage<T, BC, ColAcross, kThreads> cols(cols_from, a.col_stride, c0, col_end);
            const auto load = [&](int64_t d) {
                rows.load(d, d1);
                cols.load(d, d1);
            };
            const auto step = [&](int64_t d, char* now) {
                rows.store(now);
                cols.store(now + BR * 128);
                lds_barrier();
                if (d + kDepth < d1) load(d + kDepth);
                read(0, now, 0);
#pragma unroll
                for (int s = 0; s < 4; s++) {
                    if (s < 3) read((s + 1) % 2, now, s + 1);
                    product(s % 2);
                }
            };
            if (d0 < d1) load(d0);
            for (int64_t d = d0; d < d1;) {
                step(d, lds);
                if ((d += kDepth) >= d1) break;
                step(d, lds1);
                d += kDepth;
            }
        } else {
            DirectStage<T, BR, RowAcross, kThreads> rows(rows_from, a.row_stride, r0, row_end, d0);
            DirectStage<T, BC, ColAcross, kThreads> cols(cols_from, a.col_stride, c0, col_end, d0);
            const int64_t whole = (d1 - d0) / kDepth;
            const auto load = [&](char* to) {
                rows.load(to);
                cols.load(to + BR * 128);
            };
            constexpr int kAcrossReads = sizeof(T) == 4 ? 4 : 2, kReads = I * (RowAcross ? kAcrossReads : 1) + J * (ColAcross ? kAcrossReads : 1);
            constexpr int kProducts = I * J * (sizeof(T) == 4 ? 4 : 1), kEach = (kReads + kProducts - 1) / kProducts;
            const auto alternate = [&] {
#pragma unroll
                for (int k = 0; k < kProducts; k++) {
                    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                    __builtin_amdgcn_sched_group_barrier(0x100, kEach, 0);
                }
            };
            const auto step = [&](int64_t t, char* now, const char* next) {
#pragma unroll
                for (int s = 0; s < 3; s++) {
                    read((s + 1) % 2, now, s + 1);
                    product(s % 2);
                    alternate();
                }
                asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
                __syncthreads();
                if (t + 2 < whole) load(now);
                read(0, next, 0);  // (after the last tile of what is there, for nothing)
                product(1);
                alternate();
            };
            if (whole) {
                load(lds);
                asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
                __syncthreads();
                if (whole > 1) load(lds1);
                read(0, lds, 0);
                for (int64_t t = 0;;) {
                    step(t, lds, lds1);
                    if (++t == whole) break;
                    step(t, lds1, lds);
                    if (++t == whole) break;
                }
            }
            if (d0 + whole * kDepth < d1) {
                Stage<T, BR, RowAcross, kThreads> row(rows_from, a.row_stride, r0, row_end);
                Stage<T, BC, ColAcross, kThreads> col(cols_from, a.col_stride, c0, col_end);
                row.load(d0 + whole * kDepth, d1);
                col.load(d0 + whole * kDepth, d1);
                __syncthreads();
                row.store(lds);
                col.store(lds + BR * 128);
                __syncthreads();
                read(0, lds, 0);
#pragma unroll
                for (int s = 0; s < 4; s++) {
                    if (s < 3) read((s + 1) % 2, lds, s + 1);
                    product(s % 2);
                }
            }
        }
        __syncthreads();
    }
    float* const bias = reinterpret_cast<float*>(lds + kBuffer - BC * 4);
    if (a.bias) {
        if (threadIdx.x < BC) bias[threadIdx.x] = own_bias;
        __syncthreads();
    }
    static_assert((kWaves + 1) / 2 * kUnitBytes<T> + BC * 4 <= kBuffer && BC <= kThreads);
    char* const mine = (wave % 2 ? lds1 : lds) + wave / 2 * kUnitBytes<T>;
    Finish to = a.to;
    to.out = static_cast<T*>(to.out) + part.group * a.out_group;
    // (a unit's residual is on its way while the one before it is finished, where the sums leave registers for that)
    constexpr int kAcross = J / kUnitTiles<T>;
    constexpr bool kAhead = I * J <= 4;
    const auto unit_of = [&](int n) { return Unit<T>(to, r0 + wr + n / kAcross * 32, r1, c0 + wc + n % kAcross * kUnitTiles<T> * 32); };
    Unit<T> next = unit_of(0);
#pragma unroll
    for (int n = 0; n < I * kAcross; n++) {
        const Unit<T> now = kAhead || n == 0 ? next : unit_of(n);
        if (kAhead && n + 1 < I * kAcross) next = unit_of(n + 1);
        if (now.rows <= 0 || now.c >= a.to.cols) continue;
        Sums unit[kUnitTiles<T>];
#pragma unroll
        for (int u = 0; u < kUnitTiles<T>; u++) {
            unit[u] = sums[n / kAcross][n % kAcross * kUnitTiles<T> + u];
#pragma unroll
            for (int q = 0; q < 4; q++) {
                const int place = u * 32 + 8 * q + lane / 32 * 4;
                if (a.partial) {
                    const int64_t r = now.r + lane % 32, at = now.c + place;
                    const Floats<4> v = {unit[u][4 * q], unit[u][4 * q + 1], unit[u][4 * q + 2], unit[u][4 * q + 3]};
                    store_some<float, 4>(a.partial + (int64_t{blockIdx.y} * a.rows + r) * a.to.cols + at, v,
                                         r < r1 ? static_cast<int>(max(int64_t{0}, min(a.to.cols - at, int64_t{4}))) : 0);
                } else if (a.bias) {
                    const Floats<4> v = *reinterpret_cast<const Floats<4>*>(bias + static_cast<int>(now.c - c0) + place);
#pragma unroll
                    for (int e = 0; e < 4; e++) unit[u][4 * q + e] += v[e];
                }
            }
        }
        if (a.partial) continue;
        if constexpr (ColAcross) store_unit<T>(to, now.r, r1, now.c, unit, mine);
        else now.finish(unit, mine);
    }
}

// The splits' slabs, added in an order of their own: `turns` threads (a power of two) share four elements.
template <class T>
__global__ void __launch_bounds__(256) k_split_join(TileArgs a, int turns) {
    __shared__ Floats<4> part[256];
    const int each = 256 / turns, lane = threadIdx.x % each, turn = threadIdx.x / each;
    const int64_t quads = (a.to.cols + 3) / 4, all = a.rows * quads;
    for (int64_t first = int64_t{blockIdx.x} * each; first < all; first += int64_t{gridDim.x} * each) {
        const int64_t i = min(first + lane, all - 1), r = i / quads, c = i % quads * 4;
        const int n = static_cast<int>(min(a.to.cols - c, int64_t{4}));
        Floats<4> sum(0.0f);
#pragma unroll 4
        for (int s = turn; s < a.splits; s += turns) sum += load_some<float, 4>(a.partial + (s * a.rows + r) * a.to.cols + c, n);
        if (turns > 1) {
            __syncthreads();
            part[threadIdx.x] = sum;
            __syncthreads();
            for (int w = turns / 2; w; w /= 2) {
                if (turn < w) part[threadIdx.x] += part[threadIdx.x + w * each];
                __syncthreads();
            }
            sum = part[lane];
        }
        if (turn || first + lane >= all) continue;
        int group = 0;
        if (a.groups.ends) {
            int hi = a.groups.groups;  // the first group that ends behind the row
            while (group < hi) {
                const int mid = (group + hi) / 2;
                if (a.groups.end(mid) <= r) group = mid + 1;
                else hi = mid;
            }
            if (group >= a.groups.groups) {
                clear4<T>(a.to, r, c);
                continue;
            }
        }
        if (a.bias) sum += load_some<T, 4>(static_cast<const T*>(a.bias) + group * a.bias_group + c, n);
        finish4<T>(a.to, r, c, sum);
    }
}

// Gradients of a group's weights from the slabs of its parts of the rows: [out * in] of dweight, then, where dbias is wanted,
// [out] of it. A group's first slab is g + its first row / step; each has `step` rows, counted from the group's first row
// (`from_begin`) or from the first of all. `turns` threads (a power of two) share four elements.
struct JoinArgs {
    const float* partial;
    void *dweight, *dbias;
    int64_t weights, wanted, size;  // elements of a group's dweight, of what is joined, of a slab
    Groups groups;
    int64_t step;
    bool from_begin;
    int64_t slabs;  // without groups; else 0
    int turns;
};
template <class T>
__global__ void __launch_bounds__(256) k_weights_join(JoinArgs a) {
    __shared__ Floats<4> part[256];
    const int each = 256 / a.turns, lane = threadIdx.x % each, turn = threadIdx.x / each, group = blockIdx.y;
    const int64_t begin = a.groups.begin(group), end = a.groups.end(group), first = group + begin / a.step;
    const int64_t slabs = a.slabs ? a.slabs : end > begin ? (end - 1 - (a.from_begin ? begin : 0)) / a.step - (a.from_begin ? 0 : begin / a.step) + 1 : 0;
    for (int64_t at = int64_t{blockIdx.x} * each; at * 4 < a.wanted; at += int64_t{gridDim.x} * each) {
        const int64_t i = (at + lane) * 4;
        const int n = static_cast<int>(max(int64_t{0}, min(a.wanted - i, int64_t{4})));
        Floats<4> sum(0.0f);
        if (n > 0)
#pragma unroll 4
            for (int64_t s = turn; s < slabs; s += a.turns) sum += load_some<float, 4>(a.partial + (first + s) * a.size + i, n);
        if (a.turns > 1) {
            __syncthreads();
            part[threadIdx.x] = sum;
            __syncthreads();
            for (int w = a.turns / 2; w; w /= 2) {
                if (turn < w) part[threadIdx.x] += part[threadIdx.x + w * each];
                __syncthreads();
            }
            if (turn) continue;
            sum = part[threadIdx.x];
        }
        T* const dweight = static_cast<T*>(a.dweight) + group * a.weights;
        if (a.dweight && i + n <= a.weights) {
            store_some<T, 4>(dweight + i, sum, n);
            continue;
        }
        for (int e = 0; e < n; e++) {
            if (i + e >= a.weights) static_cast<T*>(a.dbias)[group * (a.wanted - a.weights) + i + e - a.weights] = static_cast<T>(sum[e]);
            else if (a.dweight) dweight[i + e] = static_cast<T>(sum[e]);
        }
    }
}

// ---- narrow layers ----------------------------------------------------------------------------------------
//
// Where the weight fits the LDS a layer is bound by its rows' bytes: each workgroup holds the weight there, as fragments in the
// order of the lanes, and takes its share of all rows past it, `chunk` rows side by side (a group's end among them changes the
// weight).

// The group that has the row; every lane of the wave takes part.
__device__ inline int group_of(const Groups& g, int64_t row) {
    int k = 0;
    if (g.ends)
        for (int first = 0; first < g.groups; first += 64) {
            const int e = first + static_cast<int>(threadIdx.x % 64);
            k += __builtin_popcountll(__ballot(e < g.groups && g.end(e) <= row));
        }
    return __builtin_amdgcn_readfirstlane(k);
}

struct NarrowArgs {
    const void *x, *weight, *bias;
    int64_t x_stride;
    Finish to;
    int64_t in, out, chunk;
    Groups groups;
};

// Fragments of a row of up to K steps. The load reads nothing outside the row; what it reads in place of elements past the
// row's end is taken out before the products, when it has arrived.
template <class T, int K>
struct RowLoad {
    static constexpr int V = kPer<T>;
    static constexpr int kWhole = K == 6 || K == 8 ? K - 2 : K == 12 || K == 16 ? K - 4 : K - 1;  // steps that any row of so many has whole
    int in, first;
    bool small;  // less than a fragment
    __device__ explicit RowLoad(int64_t n) : in(static_cast<int>(n)), first(static_cast<int>(threadIdx.x) % 64 / 32 * V), small(n < V) {}
    __device__ void operator()(Frag<T> (&f)[K], const T* row) const {
        if (small) {
            f[0] = load_within(row, first, in);
            return;
        }
#pragma unroll
        for (int k = 0; k < K; k++) f[k] = load_raw<V>(row + (k < kWhole ? 2 * k * V + first : min(2 * k * V + first, in - V)));
    }
    __device__ void cut(Frag<T> (&f)[K]) const {
#pragma unroll
        for (int k = kWhole; k < K; k++)
            if (!small && 2 * (k + 1) * V > in) {
                const int past = (2 * k * V + first - min(2 * k * V + first, in - V)) * static_cast<int>(sizeof(T));
                f[k] = past < 16 ? moved_down<T>(f[k], past) : Frag<T>(0);
            }
    }
};

// K steps of 32 bytes a row. A wave takes 32 rows at a time; the next 32 are on their way meanwhile. Bound by the rows' bytes:
// 1 M rows, 48 to 64 bfloat16 39 us (5.7 TB/s); 64 to 64 with gelu and pre 78 (4.9); in 200 groups 86 (4.5).
template <class T, int K>
__global__ void __launch_bounds__(512) k_narrow_fwd(NarrowArgs a) {
    constexpr int V = kPer<T>;
    extern __shared__ __attribute__((aligned(128))) char lds[];
    const int tiles = static_cast<int>((a.out + 32 * kUnitTiles<T> - 1) / (32 * kUnitTiles<T>)) * kUnitTiles<T>;
    const int lane = threadIdx.x % 64, wave = wave_of(), rows_at_once = blockDim.x / 2;
    Frag<T>* const weights = reinterpret_cast<Frag<T>*>(lds);
    float* const bias = reinterpret_cast<float*>(lds + tiles * K * 1024);
    char* const mine = lds + tiles * (K * 1024 + 128) + wave * kUnitBytes<T>;
    const RowLoad<T, K> load(a.in);
    const T* const x = static_cast<const T*>(a.x);
    // without groups the workgroups' rows lie between each other's, so that all work in one place of memory at a time
    const bool grouped = a.groups.ends;
    const int64_t last = grouped ? min(a.groups.rows, (blockIdx.x + int64_t{1}) * a.chunk) : a.groups.rows;
    const int64_t step = grouped ? rows_at_once : int64_t{gridDim.x} * rows_at_once;
    for (int64_t first = blockIdx.x * (grouped ? a.chunk : rows_at_once); first < last;) {
        const int group = group_of(a.groups, first);
        if (group >= a.groups.groups) {
            for (int64_t r = first + threadIdx.x / 8; r < last; r += blockDim.x / 8)
                for (int64_t c = threadIdx.x % 8 * 4; c < a.out; c += 32) clear4<T>(a.to, r, c);
            return;
        }
        const int64_t stop = max(first + 1, min(last, a.groups.end(group)));  // (a row at least, whatever the ends are)
        Frag<T> now[K], next[K];
        int64_t base = first + wave * 32;
        load(next, x + min(base + lane % 32, stop - 1) * a.x_stride);
        lds_barrier();
        const T* const w = static_cast<const T*>(a.weight) + group * a.in * a.out;
        for (int i = threadIdx.x; i < tiles * K * 64; i += blockDim.x) {
            const int n = i / 64 / K * 32 + i % 32, k = (2 * (i / 64 % K) + i % 64 / 32) * V;
            const T* const p = w + min(int64_t{n}, a.out - 1) * a.in;
            const Frag<T> f = a.in >= V ? load_clamped(p, k, a.in) : load_within(p, k, a.in);
            weights[i] = n < a.out ? f : Frag<T>(0);
        }
        for (int i = threadIdx.x; i < tiles * 32; i += blockDim.x)
            bias[i] = a.bias && i < a.out ? static_cast<float>(static_cast<const T*>(a.bias)[group * a.out + i]) : 0.0f;
        lds_barrier();
        for (; base < stop; base += step) {
#pragma unroll
            for (int k = 0; k < K; k++) now[k] = next[k];
            load.cut(now);
            if (base + step < stop) load(next, x + min(base + step + lane % 32, stop - 1) * a.x_stride);
            for (int t = 0; t < tiles; t += kUnitTiles<T>) {
                Unit<T> to(a.to, base, stop, t * 32);
                Sums unit[kUnitTiles<T>];
#pragma unroll
                for (int u = 0; u < kUnitTiles<T>; u++) {
#pragma unroll
                    for (int q = 0; q < 4; q++) {
                        const Floats<4> b = *reinterpret_cast<const Floats<4>*>(bias + (t + u) * 32 + 8 * q + lane / 32 * 4);
#pragma unroll
                        for (int e = 0; e < 4; e++) unit[u][4 * q + e] = b[e];
                    }
#pragma unroll
                    for (int k = 0; k < K; k++) mma(unit[u], weights[((t + u) * K + k) * 64 + lane], now[k]);
                }
                if (t == 0) arrived<T>(next);
                if (a.to.residual) arrived<T>(to.residual);
                to.finish(unit, mine);
            }
        }
        first = stop;
    }
}

// Longer rows of floats, up to Tiles times 32 outputs: a row's fragments do not fit a lane's registers, and 16 bytes of each of 32 rows
// a load would have the rows read in pieces. A wave takes 32 rows as whole lines, 128 bytes of each at a time, through registers
// (two of them on their way) and LDS of its own, which its outputs take afterwards. Bound by the rows' bytes, as far as sixteen waves
// a unit keep on their way: 1,129,273 rows of 192 to 32 234 us (4.3 TB/s).
template <class T, int Tiles>
__global__ void __launch_bounds__(512) k_long_fwd(NarrowArgs a, int lines) {
    static_assert(kUnitTiles<T> == 1 && kUnitBytes<T> >= 4096);
    constexpr int V = kPer<T>, kLine = 128 / static_cast<int>(sizeof(T));
    extern __shared__ __attribute__((aligned(128))) char lds[];
    const int lane = threadIdx.x % 64, half = lane / 32, wave = wave_of(), rows_at_once = blockDim.x / 2, steps = lines * 4;
    Frag<T>* const weights = reinterpret_cast<Frag<T>*>(lds);
    float* const bias = reinterpret_cast<float*>(lds + Tiles * steps * 1024);
    char* const mine = lds + Tiles * (steps * 1024 + 128) + wave * kUnitBytes<T>;
    const T* const x = static_cast<const T*>(a.x);
    const bool grouped = a.groups.ends;
    const int64_t last = grouped ? min(a.groups.rows, (blockIdx.x + int64_t{1}) * a.chunk) : a.groups.rows;
    const int64_t stride = grouped ? rows_at_once : int64_t{gridDim.x} * rows_at_once;
    int chunk[4];  // the lane's, of a line of row i * 8 + lane / 8
#pragma unroll
    for (int i = 0; i < 4; i++) chunk[i] = (plain_at(i * 8 + lane / 8, lane % 8) - (i * 8 + lane / 8) * 128) / 16 * V;
    for (int64_t first = blockIdx.x * (grouped ? a.chunk : rows_at_once); first < last;) {
        const int group = group_of(a.groups, first);
        if (group >= a.groups.groups) {
            for (int64_t r = first + threadIdx.x / 8; r < last; r += blockDim.x / 8)
                for (int64_t c = threadIdx.x % 8 * 4; c < a.out; c += 32) clear4<T>(a.to, r, c);
            return;
        }
        const int64_t stop = max(first + 1, min(last, a.groups.end(group)));  // (a row at least, whatever the ends are)
        const T* const w = static_cast<const T*>(a.weight) + group * a.in * a.out;
        struct Line {
            Frag<T> v[4];
        } even, odd;
        // what is loaded next, and what is worked on
        int64_t ahead = first + wave * 32, base = ahead;
        int line_ahead = 0, line = 0;
        const auto load = [&](Line& to) {
            if (ahead >= stop) return;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const T* const row = x + min(ahead + i * 8 + lane / 8, stop - 1) * a.x_stride;
                const int at = line_ahead * kLine + chunk[i];
                to.v[i] = line_ahead + 1 < lines ? load_raw<V>(row + at) : load_clamped(row, at, a.in);
            }
            if (++line_ahead == lines) line_ahead = 0, ahead += stride;
        };
        load(even);
        load(odd);
        lds_barrier();  // the group's before have been worked on
        for (int i = threadIdx.x; i < Tiles * steps * 64; i += blockDim.x) {
            const int n = i / 64 / steps * 32 + i % 32, k = (2 * (i / 64 % steps) + i % 64 / 32) * V;
            const Frag<T> f = load_clamped(w + min(int64_t{n}, a.out - 1) * a.in, k, a.in);
            weights[i] = n < a.out ? f : Frag<T>(0);
        }
        for (int i = threadIdx.x; i < Tiles * 32; i += blockDim.x)
            bias[i] = a.bias && i < a.out ? static_cast<float>(static_cast<const T*>(a.bias)[group * a.out + i]) : 0.0f;
        lds_barrier();
        Sums sums[Tiles];
        const auto step = [&](Line& v) {
            if (line == 0)
#pragma unroll
                for (int t = 0; t < Tiles; t++)
#pragma unroll
                    for (int q = 0; q < 4; q++) {
                        const Floats<4> b = *reinterpret_cast<const Floats<4>*>(bias + t * 32 + 8 * q + half * 4);
#pragma unroll
                        for (int e = 0; e < 4; e++) sums[t][4 * q + e] = b[e];
                    }
            wave_sees();  // (what was there has been read)
#pragma unroll
            for (int i = 0; i < 4; i++) *reinterpret_cast<Frag<T>*>(mine + i * 1024 + lane * 16) = v.v[i];
            load(v);
            wave_sees();
#pragma unroll
            for (int s = 0; s < 4; s++) {
                const Frag<T> row = *reinterpret_cast<const Frag<T>*>(mine + plain_at(lane % 32, 2 * s + half));
#pragma unroll
                for (int t = 0; t < Tiles; t++) mma(sums[t], weights[(t * steps + line * 4 + s) * 64 + lane], row);
            }
            if (++line < lines) return;
#pragma unroll
            for (int t = 0; t < Tiles; t++) Unit<T>(a.to, base, stop, t * 32).finish({sums[t]}, mine);
            line = 0;
            base += stride;
        };
        while (base < stop) {
            step(even);
            if (base >= stop) break;
            step(odd);
        }
        first = stop;
    }
}

struct NarrowBwdArgs {
    const void *dy, *pre, *x, *weight;  // x: null where dweight is not wanted
    int64_t dy_stride, pre_stride, x_stride;
    Finish to;       // dx; its out may be null
    float* partial;  // slabs of dweight and dbias, or null
    int64_t size;    // of a slab
    int64_t in, out, chunk;
    Groups groups;
    int act;
};
template <class T>
constexpr int kBlockRows = block_rows(sizeof(T));

// The lane's fragment of a column of a block: the lines along it, step s of eight.
template <class T, int Tiles>
__device__ inline Frag<T> across_fragment(const char* block, int column, int s) {
    constexpr int kLine = line_bytes(Tiles, sizeof(T));
    const int lane = threadIdx.x % 64, half = lane / 32;
    if constexpr (sizeof(T) == 4) {
        Frag<T> f;
#pragma unroll
        for (int i = 0; i < 4; i++) f[i] = *reinterpret_cast<const float*>(block + (s * 8 + half * 4 + i) * kLine + (column + lane % 32) * 4);
        return f;
    } else {
        using Four = short __attribute__((ext_vector_type(4)));
        using Lds = __attribute__((address_space(3))) Four*;
        const int group = lane % 16;
        Four part[2];
#pragma unroll
        for (int j = 0; j < 2; j++)
            part[j] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (Lds)(block + (s * 16 + half * 8 + j * 4 + group / 4) * kLine + (column + lane % 32 / 16 * 16 + group % 4 * 4) * 2));
        return __builtin_bit_cast(Frag<T>, __builtin_shufflevector(part[0], part[1], 0, 1, 2, 3, 4, 5, 6, 7));
    }
}

// A thread's fragments of a block's rows, Tiles times 32 columns of them, on their way from memory.
template <class T, int Tiles, int Threads>
struct BlockPart {
    static constexpr int V = kPer<T>, kLanes = Tiles * 32 / V, kLines = Threads / kLanes, N = kBlockRows<T> / kLines;
    static_assert(Threads % kLanes == 0 && kBlockRows<T> % kLines == 0);
    Frag<T> v[N];
    static __device__ int chunk() { return threadIdx.x % kLanes; }
    static __device__ int line(int i) { return threadIdx.x / kLanes + i * kLines; }
    // Rows [first, stop), at most a block of them. (Of rows and chunks there are not others are read, of a chunk that reaches past
    // its row's end the last elements of the row: `get` moves them to their place.)
    __device__ void load(const void* from, int64_t stride, int64_t width, int64_t first, int64_t stop) {
        const T* const base = static_cast<const T*>(from) + first * stride;
        const int most = static_cast<int>(min(stop - 1 - first, int64_t{kBlockRows<T>})), n = static_cast<int>(width);
        if (n >= V) {
            const T* const at = base + min(chunk() * V, n - V);
#pragma unroll
            for (int i = 0; i < N; i++) v[i] = load_raw<V>(at + min(line(i), most) * stride);
        } else {
#pragma unroll
            for (int i = 0; i < N; i++) v[i] = load_within(base + min(line(i), most) * stride, chunk() * V, width);
        }
    }
    // Its i-th chunk: zeros behind the row's end and in lines from `lines` on.
    __device__ Frag<T> get(int i, int64_t width, int lines) const {
        const int n = static_cast<int>(width), past = n < V ? 0 : chunk() * V - min(chunk() * V, n - V);
        Frag<T> f = v[i];
        if (n % V) f = moved_down<T>(f, past * static_cast<int>(sizeof(T)) & 15);
        return line(i) < lines && chunk() * V < n ? f : Frag<T>(0);
    }
};

// d as two terms of the type: the first is rounded from a little less than d, so that the second has d's sign and is not zero
// where d is not (a product with an infinite x or weight then stays infinite in their sum). Of half below 2^-14, where all values are
// 2^-24 apart, from half of d; only within 1.5 of those steps of 0 a term may vanish. Of what is not finite both are that.
template <class T>
__device__ inline void two_terms(Floats<8> d, char* first, char* second) {
    constexpr bool kHalf = std::is_same_v<T, _Float16>;
    constexpr float kLess = kHalf ? 1.0f - 1.0f / 512 : 1.0f - 1.0f / 64;
    Floats<8> less = d * kLess;
    if constexpr (kHalf)
#pragma unroll
        for (int e = 0; e < 8; e++)
            if (__builtin_fabsf(d[e]) < 0x1p-14f) less[e] = d[e] * 0.5f;
    const Frag<T> high = raw<T, 8>(less);
    const Floats<8> h = floats<T, 8>(high);
    Floats<8> low = d - h;
#pragma unroll
    for (int e = 0; e < 8; e++)
        if (!(__builtin_fabsf(h[e]) < INFINITY)) low[e] = h[e];
    *reinterpret_cast<Frag<T>*>(first) = high;
    *reinterpret_cast<Frag<T>*>(second) = raw<T, 8>(low);
}

// All three gradients in one pass: a block of rows of dz and x lies in LDS, its products with the weight are dx's rows, and the
// products of its columns with one another stay in registers over the rows of a group, tiles of 32 x 32 of dweight. The next
// block is on its way meanwhile. Up to ZT tiles of 32 outputs (Fine, of dz in two terms: half as many) and XT of 32 inputs. Bound
// by the rows' bytes, as far as two workgroups a unit, which is what LDS and registers hold, keep on their way: 1 M rows, 64 to 64
// bfloat16 with gelu 119 us (4.3 TB/s), 300,000 of floats, 48 to 64, in groups 109 (floats' products take 26 of them).
template <class T, int Waves, int ZT, int XT, bool Fine>
__global__ void __launch_bounds__(Waves * 64) k_narrow_bwd(NarrowBwdArgs a) {
    constexpr int V = kPer<T>, kRows = kBlockRows<T>, kThreads = Waves * 64;
    constexpr int kSteps = ZT * static_cast<int>(sizeof(T)), kTiles = (ZT * XT + Waves - 1) / Waves, kZ = line_bytes(ZT, sizeof(T)), kX = line_bytes(XT, sizeof(T));
    constexpr int kLow = ZT * 32 / 2 * static_cast<int>(sizeof(T));  // from a first term to its second
    static_assert(XT % kUnitTiles<T> == 0);
    extern __shared__ __attribute__((aligned(128))) char lds[];
    const int lane = threadIdx.x % 64, wave = wave_of();
    const int nt = static_cast<int>((a.out + 31) / 32), kt = static_cast<int>((a.in + 31) / 32);
    char *const dz = lds, *const xs = dz + kRows * kZ, *const mine = xs + kRows * kX + wave * kBareBytes;
    Frag<T>* const weights = reinterpret_cast<Frag<T>*>(xs + kRows * kX + Waves * kBareBytes);
    BlockPart<T, ZT, kThreads> dy, pre;
    BlockPart<T, XT, kThreads> x;
    const auto load = [&](int64_t first, int64_t stop) {
        dy.load(a.dy, a.dy_stride, a.out, first, stop);
        if (a.act) pre.load(a.pre, a.pre_stride, a.out, first, stop);
        if (a.x) x.load(a.x, a.x_stride, a.in, first, stop);
    };
    const int zc = dy.chunk(), xc = x.chunk();
    const bool grouped = a.groups.ends;
    const int64_t last = grouped ? min(a.groups.rows, (blockIdx.x + int64_t{1}) * a.chunk) : a.groups.rows;
    const int64_t step = grouped ? kRows : int64_t{gridDim.x} * kRows;
    for (int64_t first = blockIdx.x * (grouped ? a.chunk : kRows); first < last;) {
        const int group = group_of(a.groups, first);
        if (group >= a.groups.groups) {
            if (a.to.out)
                for (int64_t r = first + threadIdx.x / 8; r < last; r += kThreads / 8)
                    for (int64_t c = threadIdx.x % 8 * 4; c < a.in; c += 32) clear4<T>(a.to, r, c);
            return;
        }
        const int64_t stop = max(first + 1, min(last, a.groups.end(group)));
        load(first, stop);
        lds_barrier();  // the group's before have been worked on
        if (a.to.out) {
            const T* const w = static_cast<const T*>(a.weight) + group * a.in * a.out;
            for (int i = threadIdx.x; i < XT * kSteps * 64; i += kThreads) {
                const int k = i / 64 / kSteps * 32 + i % 32, n = (2 * (i / 64 % kSteps) + i % 64 / 32) * V;
                Frag<T> f;
#pragma unroll
                for (int e = 0; e < V; e++) f[e] = w[min(int64_t{n + e}, a.out - 1) * a.in + min(int64_t{k}, a.in - 1)];
#pragma unroll
                for (int e = 0; e < V; e++)
                    if (n + e >= a.out || k >= a.in) f[e] = static_cast<T>(0.0f);
                weights[i] = f;
            }
        }
        Sums sums[kTiles];
        Floats<V> db(0.0f);
#pragma unroll
        for (int t = 0; t < kTiles; t++) sums[t] = Sums(0.0f);
        for (int64_t block = first; block < stop; block += step) {
            const int rows = static_cast<int>(min(stop - block, int64_t{kRows}));
#pragma unroll
            for (int i = 0; i < dy.N; i++) {
                Floats<V> d = floats<T, V>(dy.get(i, a.out, rows));
                if (a.act) through<T, V>(d, floats<T, V>(pre.get(i, a.out, rows)), a.act);
                db += d;
                char* const at = dz + dy.line(i) * kZ + zc * 16;
                if constexpr (Fine) {
                    if (zc < dy.kLanes / 2) two_terms<T>(d, at, at + kLow);
                } else {
                    *reinterpret_cast<Frag<T>*>(at) = raw<T, V>(d);
                }
            }
            if (a.x)
#pragma unroll
                for (int i = 0; i < x.N; i++)
                    *reinterpret_cast<Frag<T>*>(xs + x.line(i) * kX + xc * 16) = x.get(i, a.in, rows);
            lds_barrier();
            if (block + step < stop) load(block + step, stop);
            if (a.x)
#pragma unroll
                for (int i = 0; i < kTiles; i++) {
                    const int t = wave + i * Waves;
                    if (t / XT < nt && t % XT < kt)
#pragma unroll
                        for (int s = 0; s < 8; s++) {
                            const Frag<T> col = across_fragment<T, XT>(xs, t % XT * 32, s);
                            mma(sums[i], col, across_fragment<T, ZT>(dz, t / XT * 32, s));
                            if constexpr (Fine) mma(sums[i], col, across_fragment<T, ZT>(dz + kLow, t / XT * 32, s));
                        }
                }
            if (a.to.out)
                for (int i = wave; i < kRows / 32 * (XT / kUnitTiles<T>); i += Waves) {
                    const int strip = i / (XT / kUnitTiles<T>) * 32, t = i % (XT / kUnitTiles<T>) * kUnitTiles<T>;
                    if (strip >= rows) break;
                    if (t >= kt) continue;
                    Sums unit[kUnitTiles<T>];
#pragma unroll
                    for (int u = 0; u < kUnitTiles<T>; u++) unit[u] = Sums(0.0f);
                    for (int s = 0; s < nt * static_cast<int>(sizeof(T)); s++) {
                        const char* const at = dz + (strip + lane % 32) * kZ + (2 * s + lane / 32) * 16;
                        const Frag<T> row = *reinterpret_cast<const Frag<T>*>(at);
#pragma unroll
                        for (int u = 0; u < kUnitTiles<T>; u++) mma(unit[u], weights[((t + u) * kSteps + s) * 64 + lane], row);
                        if constexpr (Fine) {
                            const Frag<T> low = *reinterpret_cast<const Frag<T>*>(at + kLow);
#pragma unroll
                            for (int u = 0; u < kUnitTiles<T>; u++) mma(unit[u], weights[((t + u) * kSteps + s) * 64 + lane], low);
                        }
                    }
                    if (i == wave) {  // before the first stores
                        arrived<T>(dy.v);
                        if (a.act) arrived<T>(pre.v);
                        if (a.x) arrived<T>(x.v);
                    }
                    store_unit<T>(a.to, block + strip, stop, t * 32, unit, mine);
                }
            lds_barrier();
        }
        if (a.partial) {
            float* const slab = a.partial + (int64_t{blockIdx.x} + group) * a.size;
#pragma unroll
            for (int i = 0; i < kTiles; i++) {
                const int t = wave + i * Waves;
                const int64_t n = t / XT * 32 + lane % 32;
                if (a.x && t % XT < kt && n < a.out)
#pragma unroll
                    for (int q = 0; q < 4; q++) {
                        const int64_t k = t % XT * 32 + 8 * q + lane / 32 * 4;
                        const Floats<4> v = {sums[i][4 * q], sums[i][4 * q + 1], sums[i][4 * q + 2], sums[i][4 * q + 3]};
                        store_some<float, 4>(slab + n * a.in + k, v, static_cast<int>(max(int64_t{0}, min(a.in - k, int64_t{4}))));
                    }
            }
            Floats<V>* const parts = reinterpret_cast<Floats<V>*>(lds);
            static_assert(kThreads * sizeof(Floats<V>) <= kRows * (kZ + kX));
            parts[threadIdx.x] = db;
            lds_barrier();
            if (static_cast<int>(threadIdx.x) < dy.kLanes && zc * V < a.out) {
                for (int l = 1; l < dy.kLines; l++) db += parts[l * dy.kLanes + zc];
                store_some<float, V>(slab + a.in * a.out + zc * V, db, static_cast<int>(min(a.out - zc * V, int64_t{V})));
            }
        }
        first = stop;
    }
}

// ---- few rows ---------------------------------------------------------------------------------------------
//
// A layer of few rows is bound by its weight's bytes, each read once. Forward: a workgroup has 32 outputs, its waves share the
// sums' length, 128 bytes of each weight's row at a time in turn, and add their sums in LDS at the end. What they read comes
// through LDS of the wave's own, straight there where all lines begin on 16 bytes, else through registers: a load of 16 bytes each
// from 32 rows takes four times as long as one of whole lines, and half of them are x's, again and again. (9 rows to 8192 in half
// precision, us: of 2048 15 by tiles, 10.5 by such loads, 8.9 so, 3.7 TB/s; of 2049 19.5 by such loads, 9.6 so. 2 rows of 7187 to
// 2267 in floats 35 and 20.4, the library's product 28.)
struct FewArgs {
    const void *x, *weight, *bias;
    int64_t x_stride;
    Finish to;
    int64_t in, out;
    Groups groups;
    float* partial;  // [slices][rows][out] in place of y, or null
    int64_t rows, slice;  // of the sums' length, whole lines of every wave
};
template <class T, bool Lines>
__global__ void __launch_bounds__(kFewWaves * 64) k_few_fwd(FewArgs a) {
    constexpr int V = kPer<T>, kLine = 128 / static_cast<int>(sizeof(T)), kPitch = 36;
    // (two arrays, so that a load into one is seen to be no store into the other)
    __shared__ __attribute__((aligned(128))) char lds[kFewWaves * 8192], lds1[Lines ? kFewWaves * 8192 : 16];
    static_assert(sizeof(float) * 32 * kPitch <= 8192);
    const Part part = part_of(a.groups, blockIdx.y, kFewShift);
    if (part.begin >= part.end) return;
    const int64_t c0 = int64_t{blockIdx.x} * 32;
    const int lane = threadIdx.x % 64, half = lane / 32, wave = wave_of();
    // (in the end a thread of the first half has four outputs)
    const int64_t r = part.begin + threadIdx.x / 8, c = c0 + threadIdx.x % 8 * 4;
    if (part.group >= a.groups.groups) {
        if (a.partial) return;
        if (threadIdx.x < 256 && r < part.end) clear4<T>(a.to, r, c);
        return;
    }
    const int64_t first = blockIdx.z * a.slice, length = min(a.slice, a.in - first);
    const T* const weight = static_cast<const T*>(a.weight) + part.group * a.out * a.in + first;
    const T* const xs = static_cast<const T*>(a.x) + first;
    const T* const w = weight + min(c0 + lane % 32, a.out - 1) * a.in;
    const T* const x = xs + min(part.begin + lane % 32, part.end - 1) * a.x_stride;
    Sums s(0.0f);
    // The wave's lines: `wave` and every eighth after it. A load of the wave's takes eight rows', as they lie in a tile (plain_at).
    const int64_t lines = length / kLine, mine = (lines - wave + kFewWaves - 1) / kFewWaves;
    const T *from_w[4], *from_x[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int row = i * 8 + lane / 8, chunk = (plain_at(row, lane % 8) - row * 128) / 16 * V;
        from_w[i] = weight + min(c0 + row, a.out - 1) * a.in + wave * kLine + chunk;
        from_x[i] = xs + min(part.begin + row, part.end - 1) * a.x_stride + wave * kLine + chunk;
    }
    const auto product = [&](const char* now) {
        Frag<T> fw[4], fx[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            fw[i] = *reinterpret_cast<const Frag<T>*>(now + wave * 8192 + plain_at(lane % 32, 2 * i + half));
            fx[i] = *reinterpret_cast<const Frag<T>*>(now + wave * 8192 + 4096 + plain_at(lane % 32, 2 * i + half));
        }
#pragma unroll
        for (int i = 0; i < 4; i++) mma(s, fw[i], fx[i]);
    };
    int64_t loaded = 0;
    // (after the last line that again, so that as many loads are always on their way)
    const auto onwards = [&] {
        const int64_t next = ++loaded < mine ? kFewWaves * kLine : 0;
#pragma unroll
        for (int i = 0; i < 4; i++) from_w[i] += next, from_x[i] += next;
    };
    if constexpr (Lines) {
        using Global = __attribute__((address_space(1))) const void*;
        using Lds = __attribute__((address_space(3))) void*;
        const auto load = [&](char* to) {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                __builtin_amdgcn_global_load_lds((Global)from_w[i], (Lds)(to + wave * 8192 + i * 1024), 16, 0, 0);
                __builtin_amdgcn_global_load_lds((Global)from_x[i], (Lds)(to + wave * 8192 + 4096 + i * 1024), 16, 0, 0);
            }
            onwards();
        };
        const auto step = [&](const char* now, char* next) {
            wait_for<63>();  // (what was read of that place is there)
            load(next);
            wait_for<8>();
            product(now);
        };
        if (mine > 0) {
            load(lds);
            for (int64_t t = 0;;) {
                step(lds, lds1);
                if (++t == mine) break;
                step(lds1, lds);
                if (++t == mine) break;
            }
            wait_for<0>();
        }
    } else if (mine > 0) {
        // Of rows that begin anywhere the lines go through registers, two of them on their way; of x only the rows there are, eight at
        // a time. (What LDS holds in place of others goes into sums that nothing takes.)
        const auto pass = [&](auto eights) {
            constexpr int X = eights.value;
            struct Line {
                Frag<T> w[4], x[X];
            } first, second;
            const auto load = [&](Line& v) {
#pragma unroll
                for (int i = 0; i < 4; i++) v.w[i] = load_raw<V>(from_w[i]);
#pragma unroll
                for (int i = 0; i < X; i++) v.x[i] = load_raw<V>(from_x[i]);
                onwards();
            };
            const auto step = [&](Line& v) {
                char* const to = lds + wave * 8192 + lane * 16;
                wave_sees();  // (what was there has been read)
#pragma unroll
                for (int i = 0; i < 4; i++) *reinterpret_cast<Frag<T>*>(to + i * 1024) = v.w[i];
#pragma unroll
                for (int i = 0; i < X; i++) *reinterpret_cast<Frag<T>*>(to + 4096 + i * 1024) = v.x[i];
                load(v);
                wave_sees();
                product(lds);
            };
            load(first);
            load(second);
            for (int64_t t = 0;;) {
                step(first);
                if (++t == mine) break;
                step(second);
                if (++t == mine) break;
            }
        };
        const int64_t rows = part.end - part.begin;
        if (rows <= 8) pass(std::integral_constant<int, 1>{});
        else if (rows <= 16) pass(std::integral_constant<int, 2>{});
        else pass(std::integral_constant<int, 4>{});
    }
    // what is left of the length, less than a line
    if (const int64_t k = lines * kLine; wave == 0 && k < length) {
        Frag<T> fw[4], fx[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int64_t at = k + (2 * i + half) * V;
            fw[i] = length >= V ? load_clamped(w, at, length) : load_within(w, at, length);
            fx[i] = length >= V ? load_clamped(x, at, length) : load_within(x, at, length);
        }
#pragma unroll
        for (int i = 0; i < 4; i++) mma(s, fw[i], fx[i]);
    }
    float* const sums = reinterpret_cast<float*>(lds + wave * 8192);
#pragma unroll
    for (int q = 0; q < 4; q++)
        *reinterpret_cast<Floats<4>*>(sums + lane % 32 * kPitch + half * 4 + q * 8) = Floats<4>{s[4 * q], s[4 * q + 1], s[4 * q + 2], s[4 * q + 3]};
    __syncthreads();
    if (threadIdx.x >= 256 || r >= part.end || c >= a.out) return;
    Floats<4> v(0.0f);
#pragma unroll
    for (int k = 0; k < kFewWaves; k++) v += *reinterpret_cast<const Floats<4>*>(lds + k * 8192 + (threadIdx.x / 8 * kPitch + threadIdx.x % 8 * 4) * 4);
    if (a.partial) {
        store_some<float, 4>(a.partial + (blockIdx.z * a.rows + r) * a.out + c, v, static_cast<int>(min(a.out - c, int64_t{4})));
        return;
    }
    if (a.bias) v += load_some<T, 4>(static_cast<const T*>(a.bias) + part.group * a.out + c, static_cast<int>(min(a.out - c, int64_t{4})));
    finish4<T>(a.to, r, c, v);
}

// The backward of few rows, in floats: dz of the rows lies in LDS, a thread has the columns of 16 bytes.
struct FewBwdArgs {
    const void *dy, *pre, *x, *weight;
    int64_t dy_stride, pre_stride, x_stride;
    void *dweight, *dbias;
    float* partial;  // [slices][rows][in] of dx
    int64_t in, out, slice;
    Groups groups;
    int act;
};
// dz of rows [r, r + rows) and outputs [n, n + outputs) before `end` as [outputs][pitch] floats, zeros past them
template <class T>
__device__ inline void few_dz(const FewBwdArgs& a, float* dz, int64_t r, int rows, int pitch, int64_t n, int outputs, int64_t end) {
    for (int i = threadIdx.x; i < outputs * pitch; i += kFewBlock) {
        const int m = i / outputs, o = i % outputs;  // (threads side by side: outputs side by side)
        Floats<1> d(0.0f);
        if (m < rows && n + o < end) {
            d[0] = static_cast<float>(static_cast<const T*>(a.dy)[(r + m) * a.dy_stride + n + o]);
            if (a.act) through<T, 1>(d, Floats<1>(static_cast<float>(static_cast<const T*>(a.pre)[(r + m) * a.pre_stride + n + o])), a.act);
        }
        dz[o * pitch + m] = d[0];
    }
}
// The thread's chunks of N rows from `first` on, of those before `end`, on their way together.
template <class T, int N>
__device__ inline void few_chunks(Frag<T> (&v)[N], const T* base, int64_t stride, int64_t first, int64_t end, int64_t c, int64_t n) {
    constexpr int V = kPer<T>;
    if (n < V) {
#pragma unroll
        for (int i = 0; i < N; i++) v[i] = load_within(base + min(first + i, end - 1) * stride, c, n);
        return;
    }
    const int64_t at = min(c, n - V);
#pragma unroll
    for (int i = 0; i < N; i++) v[i] = load_raw<V>(base + min(first + i, end - 1) * stride + at);
    if (n % V)
#pragma unroll
        for (int i = 0; i < N; i++) v[i] = moved_down<T>(v[i], static_cast<int>(c - at) * static_cast<int>(sizeof(T)) & 15);
}

// dx = dz W of a slice of the outputs, sixteen rows at a time: the weight's rows pass by once for each sixteen. With floats' own
// products: dz stays unrounded, and the weight's bytes are what it takes (the gradients of 6 rows in 3 groups, 1984 to 5536 float,
// by tiles 134 us, so 58; of 3 rows, 1856 to 992, 29 and 15).
template <class T>
__global__ void __launch_bounds__(kFewBlock) k_few_dx(FewBwdArgs a) {
    constexpr int V = kPer<T>, kAtOnce = 16, kOutputs = 32, kBatch = 16;
    __shared__ __attribute__((aligned(16))) float dz[kOutputs * kAtOnce];
    const Part part = part_of(a.groups, blockIdx.z, kFewShift);
    if (part.group >= a.groups.groups || part.begin >= part.end) return;
    const int64_t c = (int64_t{blockIdx.x} * kFewBlock + threadIdx.x) * V;
    const int64_t n0 = blockIdx.y * a.slice, n1 = min(a.out, n0 + a.slice);
    const T* const w = static_cast<const T*>(a.weight) + part.group * a.in * a.out;
    for (int64_t r = part.begin; r < part.end; r += kAtOnce) {
        const int rows = static_cast<int>(min(part.end - r, int64_t{kAtOnce}));
        Floats<V> sum[kAtOnce];
#pragma unroll
        for (int m = 0; m < kAtOnce; m++) sum[m] = Floats<V>(0.0f);
        for (int64_t n = n0; n < n1; n += kOutputs) {
            __syncthreads();
            few_dz<T>(a, dz, r, rows, kAtOnce, n, kOutputs, n1);
            __syncthreads();
            const int here = static_cast<int>(min(n1 - n, int64_t{kOutputs}));
            if (c < a.in)
                for (int o = 0; o < here; o += kBatch) {
                    Frag<T> v[kBatch];
                    few_chunks<T, kBatch>(v, w, a.in, n + o, n1, c, a.in);
#pragma unroll
                    for (int b = 0; b < kBatch; b++) {
                        if (o + b >= here) break;  // (past the slice's end lies its last row again, and an infinity times 0 is none)
                        const Floats<V> f = floats<T, V>(v[b]);
#pragma unroll
                        for (int q = 0; q < kAtOnce; q += 4) {
                            if (q >= rows) break;
                            const Floats<4> d = *reinterpret_cast<const Floats<4>*>(dz + (o + b) * kAtOnce + q);
#pragma unroll
                            for (int m = 0; m < 4; m++)
#pragma unroll
                                for (int e = 0; e < V; e++) sum[q + m][e] = __builtin_fmaf(d[m], f[e], sum[q + m][e]);
                        }
                    }
                }
        }
        if (c >= a.in) continue;
#pragma unroll
        for (int m = 0; m < kAtOnce; m++)
            if (m < rows)
                store_some<float, V>(a.partial + (blockIdx.y * a.groups.rows + r + m) * a.in + c, sum[m], static_cast<int>(min(a.in - c, int64_t{V})));
    }
}

// dweight = dz^T x and dbias of eight outputs.
template <class T>
__global__ void __launch_bounds__(kFewBlock) k_few_dw(FewBwdArgs a) {
    constexpr int V = kPer<T>, kOutputs = 8, kBatch = 8;
    __shared__ __attribute__((aligned(16))) float dz[kOutputs * kFewRows];
    const int group = blockIdx.z;
    const int64_t begin = a.groups.begin(group);
    const int rows = static_cast<int>(max(int64_t{0}, min(a.groups.end(group) - begin, int64_t{kFewRows})));
    const int64_t n = int64_t{blockIdx.y} * kOutputs, c = (int64_t{blockIdx.x} * kFewBlock + threadIdx.x) * V;
    few_dz<T>(a, dz, begin, rows, kFewRows, n, kOutputs, a.out);
    __syncthreads();
    if (a.dbias && blockIdx.x == 0 && threadIdx.x < kOutputs && n + threadIdx.x < a.out) {
        float sum = 0.0f;
        for (int m = 0; m < rows; m++) sum += dz[threadIdx.x * kFewRows + m];
        static_cast<T*>(a.dbias)[group * a.out + n + threadIdx.x] = static_cast<T>(sum);
    }
    if (!a.dweight || c >= a.in) return;
    Floats<V> sum[kOutputs];
#pragma unroll
    for (int o = 0; o < kOutputs; o++) sum[o] = Floats<V>(0.0f);
    for (int m = 0; m < rows; m += kBatch) {
        Frag<T> v[kBatch];
        few_chunks<T, kBatch>(v, static_cast<const T*>(a.x), a.x_stride, begin + m, begin + rows, c, a.in);
#pragma unroll
        for (int b = 0; b < kBatch; b++) {
            if (m + b >= rows) break;
            const Floats<V> f = floats<T, V>(v[b]);
#pragma unroll
            for (int o = 0; o < kOutputs; o++) {
                const float d = dz[o * kFewRows + m + b];
#pragma unroll
                for (int e = 0; e < V; e++) sum[o][e] = __builtin_fmaf(d, f[e], sum[o][e]);
            }
        }
    }
#pragma unroll
    for (int o = 0; o < kOutputs; o++)
        if (n + o < a.out)
            store_some<T, V>(static_cast<T*>(a.dweight) + (group * a.out + n + o) * a.in + c, sum[o], static_cast<int>(min(a.in - c, int64_t{V})));
}

// ---- dz = dy act'(pre), and its columns' sums ------------------------------------------------------------

struct SlopeArgs {
    const void *dy, *pre;
    void* dz;            // [rows][dz_stride], or null
    float* partial;      // [slots][cols], or null
    int64_t dy_stride, pre_stride, dz_stride, cols;
    Groups groups;
    int shift, act;
};

// A part of the rows and up to 256 vectors of columns a workgroup; `lanes` threads go along a row, as many as it has vectors (by
// the next power of two: 800,000 rows, 64 to 300 bfloat16, gradients 878 us for 826), four rows at a time (their loads on their
// way together). Bound by its bytes: those 403 MB in 87 us, 4.6 TB/s.
template <class T>
__global__ void __launch_bounds__(256) k_slope(SlopeArgs a, int lanes) {
    constexpr int V = kPer<T>, kAtOnce = 4;
    __shared__ Floats<V> sums[256];
    const Part part = part_of(a.groups, blockIdx.x, a.shift);
    if (part.group >= a.groups.groups || part.begin >= part.end) return;
    const int64_t c = (int64_t{blockIdx.y} * lanes + threadIdx.x % lanes) * V;
    const int step = 256 / lanes;
    Floats<V> sum(0.0f);
    if (c < a.cols && static_cast<int>(threadIdx.x) < step * lanes) {
        const int n = static_cast<int>(min(a.cols - c, int64_t{V}));
        // (a vector that reaches past the row's end is read so that it ends there, and moved to its place)
        const bool small = a.cols < V;
        const int64_t at = min(c, a.cols - V);
        const int past = small ? 0 : static_cast<int>(c - at) * static_cast<int>(sizeof(T));
        for (int64_t first = part.begin + threadIdx.x / lanes; first < part.end; first += kAtOnce * step) {
            Frag<T> dy[kAtOnce], pre[kAtOnce];
            const auto load = [&](Frag<T> (&v)[kAtOnce], const void* from, int64_t stride) {
#pragma unroll
                for (int i = 0; i < kAtOnce; i++) {
                    const T* const p = static_cast<const T*>(from) + min(first + i * step, part.end - 1) * stride;
                    v[i] = small ? load_within(p, c, a.cols) : load_raw<V>(p + at);
                }
            };
            load(dy, a.dy, a.dy_stride);
            if (a.act) load(pre, a.pre, a.pre_stride);
#pragma unroll
            for (int i = 0; i < kAtOnce; i++) {
                const int64_t r = first + i * step;
                if (r >= part.end) break;
                if (past) {
                    dy[i] = moved_down<T>(dy[i], past);
                    if (a.act) pre[i] = moved_down<T>(pre[i], past);
                }
                Floats<V> d = floats<T, V>(dy[i]);
                if (a.act) through<T, V>(d, floats<T, V>(pre[i]), a.act);
                if (a.dz) {
                    store_some<T, V>(static_cast<T*>(a.dz) + r * a.dz_stride + c, d, n);
                }
                sum += d;
            }
        }
    }
    if (!a.partial) return;
    sums[threadIdx.x] = sum;
    __syncthreads();
    if (static_cast<int>(threadIdx.x) >= lanes || c >= a.cols) return;
    for (int t = threadIdx.x + lanes; t < step * lanes; t += lanes) sum += sums[t];
    store_some<float, V>(a.partial + int64_t{blockIdx.x} * a.cols + c, sum, static_cast<int>(min(a.cols - c, int64_t{V})));
}

// ---- launches ---------------------------------------------------------------------------------------------

// A call's workspace, handed out from its beginning; without memory only how much there has to be.
class Work {
  public:
    explicit Work(void* base) : base_(static_cast<char*>(base)) {}
    char* take(int64_t bytes) {
        char* const p = base_ ? base_ + used_ : nullptr;
        used_ += (bytes + 255) / 256 * 256;
        most_ = std::max(most_, used_);
        return p;
    }
    int64_t used() const { return used_; }
    void back_to(int64_t used) { used_ = used; }
    int64_t most() const { return most_; }

  private:
    char* base_;
    int64_t used_ = 0, most_ = 0;
};
// Where a call is enqueued, or that it is only measured.
struct Run {
    Work work;
    hipStream_t stream;
    bool real;
};

void check_grid(int64_t blocks, int64_t threads) {
    if (blocks * threads >= int64_t{1} << 32) throw std::runtime_error("linear: more workgroups than a launch holds");
}

template <class T>
void launch_slope(const SlopeArgs& a, const Slope& p, hipStream_t s) {
    check_grid(p.slots * p.columns, 256);
    k_slope<T><<<dim3(static_cast<uint32_t>(p.slots), static_cast<uint32_t>(p.columns)), 256, 0, s>>>(a, p.lanes);
}

// A product's operand as k_tile reads it: lines that begin on 16 bytes, their places in a tile in 32 bits, and across them whole
// fragments. What lies otherwise is copied first, which takes two passes over it where loads of its own kind took the product three
// times as long (377 rows of 5996 to 1162 bfloat16, the gradients 98 us, with the copies 66; but see staged_pays).
struct Operand {
    const void* p;
    int64_t stride, width;
};
template <class T>
bool lies_for_tiles(const void* p, int64_t width, int64_t stride, bool across) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride * static_cast<int64_t>(sizeof(T)) % 16 == 0 &&
           stride <= kMostLine / static_cast<int>(sizeof(T)) && (!across || width % kPer<T> == 0);
}
template <class T>
Operand operand(const void* p, int64_t rows, int64_t width, int64_t stride, bool across, Run& run) {
    if (lies_for_tiles<T>(p, width, stride, across) || !rows) return {p, stride, width};
    const Slope plan = plan_slope(rows, width, 1, false, sizeof(T));
    SlopeArgs a{};
    a.dy = p; a.dy_stride = stride; a.dz = run.work.take(plan.dz_bytes); a.dz_stride = plan.dz_stride;
    a.cols = width; a.groups = {nullptr, 1, rows}; a.shift = plan.shift;
    if (run.real) launch_slope<T>(a, plan, run.stream);
    return {a.dz, plan.dz_stride, plan.dz_stride};
}

template <class T, bool RowAcross, bool ColAcross>
void launch_tiles(const TileArgs& a, int side, int64_t slabs, bool staged, hipStream_t s) {
    const int64_t down = RowAcross ? up(a.rows, side) : a.slots, tiles = up(down * up(a.to.cols, side == 256 ? 256 : 128), 8) * 8;
    check_grid(tiles * slabs, side == 256 ? 512 : 256);
    const dim3 grid(static_cast<uint32_t>(tiles), static_cast<uint32_t>(slabs));
    if constexpr (sizeof(T) == 2) {
        if (side == 256) {
            k_tile<T, 256, 256, 128, 64, RowAcross, ColAcross, false><<<grid, 512, 0, s>>>(a);
            return;
        }
    } else if constexpr (!RowAcross && !ColAcross) {
        if (staged) {
            if (side == 128) k_tile<T, 128, 128, 64, 64, false, false, true><<<grid, 256, 0, s>>>(a);
            else k_tile<T, 64, 128, 32, 64, false, false, true><<<grid, 256, 0, s>>>(a);
            return;
        }
    }
    if (side == 128) k_tile<T, 128, 128, 64, 64, RowAcross, ColAcross, false><<<grid, 256, 0, s>>>(a);
    else k_tile<T, 64, 128, 32, 64, RowAcross, ColAcross, false><<<grid, 256, 0, s>>>(a);
}

// `slabs`: of a group, on average
template <class T>
void join_weights(JoinArgs a, int64_t slabs, hipStream_t s) {
    a.turns = 1;
    while (a.turns < 64 && a.turns * 4 <= slabs) a.turns *= 2;
    const int64_t blocks = std::min<int64_t>(up(up(a.wanted, 4), 256 / a.turns), 65536);
    k_weights_join<T><<<dim3(static_cast<uint32_t>(blocks), static_cast<uint32_t>(a.groups.groups)), 256, 0, s>>>(a);
}

template <class T>
void launch_narrow_bwd(const NarrowBwdArgs& a, const NarrowBwd& p, hipStream_t s) {
    const auto go = [&](auto kernel) { kernel<<<static_cast<uint32_t>(p.blocks), p.waves * 64, p.lds, s>>>(a); };
    if constexpr (sizeof(T) == 4) {
        if (p.waves == 4) go(k_narrow_bwd<T, 4, 2, 2, false>);
        else if (p.zt == 4) go(k_narrow_bwd<T, 8, 4, 2, false>);
        else go(k_narrow_bwd<T, 8, 2, 4, false>);
    } else {
        const auto by_terms = [&](auto fine) {
            if (p.waves == 4) go(k_narrow_bwd<T, 4, 2, 2, fine.value>);
            else if (p.zt == 4) go(k_narrow_bwd<T, 8, 4, 4, fine.value>);
            else if (p.zt == 2) go(k_narrow_bwd<T, 8, 2, 8, fine.value>);
            else go(k_narrow_bwd<T, 8, 8, 2, fine.value>);
        };
        if (p.fine) by_terms(std::true_type{});
        else by_terms(std::false_type{});
    }
}

template <class T>
void launch_narrow(const NarrowArgs& a, const Narrow& p, hipStream_t s) {
    const auto go = [&](auto kernel) { kernel<<<static_cast<uint32_t>(p.blocks), p.threads, p.lds, s>>>(a); };
    switch (p.steps) {
        case 1: return go(k_narrow_fwd<T, 1>);
        case 2: return go(k_narrow_fwd<T, 2>);
        case 3: return go(k_narrow_fwd<T, 3>);
        case 4: return go(k_narrow_fwd<T, 4>);
        case 6: return go(k_narrow_fwd<T, 6>);
        case 8: return go(k_narrow_fwd<T, 8>);
        case 12: return go(k_narrow_fwd<T, 12>);
        default: return go(k_narrow_fwd<T, 16>);
    }
}

template <class T>
void join_splits(const TileArgs& a, hipStream_t s) {
    int turns = 1;
    while (turns < 32 && turns * 4 <= a.splits) turns *= 2;
    const int64_t blocks = std::min<int64_t>(up(a.rows * up(a.to.cols, 4), 256 / turns), 4096);
    k_split_join<T><<<static_cast<uint32_t>(blocks), 256, 0, s>>>(a, turns);
}

// out = row col^T over the groups' rows (see TileArgs), with what follows.
template <class T, bool ColAcross>
void over_depth(TileArgs a, bool ragged, bool staged, Run& run) {
    const Plan p = plan_rows(a.rows, a.to.cols, a.depth, a.groups.groups, ragged, sizeof(T));
    a.shift = log2_up(p.side);
    a.slots = slots_of(a.rows, a.groups.groups, a.shift, ragged);
    a.split = p.split;
    a.splits = p.splits;
    a.partial = p.splits > 1 ? reinterpret_cast<float*>(run.work.take(p.bytes)) : nullptr;
    if (!run.real) return;
    launch_tiles<T, false, ColAcross>(a, p.side, p.splits, staged, run.stream);
    if (a.partial) join_splits<T>(a, run.stream);
}

template <class T>
void forward(const LinearFwdArgs& f, Run& run) {
    const Finish to{f.y, f.y_stride, f.out, f.residual, f.residual_stride, f.pre, f.pre_stride, f.act, f.clear};
    const Groups groups{f.ends, f.groups, f.rows};
    const bool ragged = f.ends != nullptr;
    if (const Narrow p = plan_narrow(f.rows, f.in, f.out, ragged, sizeof(T)); p.blocks) {
        if (run.real) launch_narrow<T>({f.x, f.weight, f.bias, f.x_stride, to, f.in, f.out, p.chunk, groups}, p, run.stream);
        return;
    }
    if constexpr (sizeof(T) == 4)
        if (const Long p = plan_long(f.rows, f.in, f.out, f.groups, ragged); p.blocks) {
            const NarrowArgs a{f.x, f.weight, f.bias, f.x_stride, to, f.in, f.out, p.chunk, groups};
            const auto go = [&](auto kernel) { kernel<<<static_cast<uint32_t>(p.blocks), p.threads, p.lds, run.stream>>>(a, p.lines); };
            if (run.real) p.tiles == 1 ? go(k_long_fwd<T, 1>) : go(k_long_fwd<T, 2>);
            return;
        }
    const auto whole_lines = [](const void* p, int64_t stride) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride * sizeof(T) % 16 == 0; };
    const bool whole = whole_lines(f.x, f.x_stride) && whole_lines(f.weight, f.in);
    if (few_rows(f.rows, f.out, f.groups, sizeof(T), whole)) {
        const int64_t slots = slots_of(f.rows, f.groups, kFewShift, ragged), blocks = up(f.out, 32);
        // Where that leaves units without work and a wave has eight lines and more (sixteen, of those that go straight into LDS), slices
        // of the sums' length, of two lines a wave at least, are workgroups of their own. (31 rows of 2274 to 906 float, nine lines, 15.5 us
        // whole, 12.5 in slices; 8 rows of 4096 to 1024 bfloat16, eight lines straight into LDS, 7.9 and 9.5.)
        constexpr int64_t line = kFewWaves * 128 / static_cast<int>(sizeof(T));
        const int64_t lines = up(f.in, line), most = lines < (whole ? 16 : 8) ? 1 : std::min(lines / 2, 256 / std::max<int64_t>(blocks * slots, 1));
        const int64_t slice = up(lines, std::max<int64_t>(most, 1)) * line, slices = up(f.in, slice);
        TileArgs t{};  // (what joins the slices)
        t.to = to; t.rows = f.rows; t.groups = groups; t.bias = f.bias; t.bias_group = f.out; t.splits = static_cast<int>(slices);
        if (slices > 1) t.partial = reinterpret_cast<float*>(run.work.take(slices * f.rows * f.out * 4));
        if (!run.real || !f.rows) return;
        check_grid(blocks * slots * slices, kFewWaves * 64);
        const dim3 grid(static_cast<uint32_t>(blocks), static_cast<uint32_t>(slots), static_cast<uint32_t>(slices));
        const FewArgs a{f.x, f.weight, f.bias, f.x_stride, to, f.in, f.out, groups, t.partial, f.rows, slice};
        if (whole) k_few_fwd<T, true><<<grid, kFewWaves * 64, 0, run.stream>>>(a);
        else k_few_fwd<T, false><<<grid, kFewWaves * 64, 0, run.stream>>>(a);
        if (slices > 1) join_splits<T>(t, run.stream);
        return;
    }
    const bool x_lies = lies_for_tiles<T>(f.x, f.in, f.x_stride, false), w_lies = lies_for_tiles<T>(f.weight, f.in, f.in, false);
    const bool staged = sizeof(T) == 4 && staged_pays(f.rows, f.in, f.out, f.groups, !x_lies, !w_lies);
    const Operand x = staged ? Operand{f.x, f.x_stride, f.in} : operand<T>(f.x, f.rows, f.in, f.x_stride, false, run);
    const Operand w = staged ? Operand{f.weight, f.in, f.in} : operand<T>(f.weight, f.groups * f.out, f.in, f.in, false, run);
    TileArgs a{};
    a.row = x.p; a.row_stride = x.stride; a.col = w.p; a.col_stride = w.stride; a.col_group = w.stride * f.out;
    a.rows = f.rows; a.depth = f.in; a.groups = groups; a.bias = f.bias; a.bias_group = f.out; a.to = to;
    over_depth<T, false>(a, ragged, staged, run);
}

template <class T>
void backward_narrow(const LinearBwdArgs& f, const NarrowBwd& p, Run& run) {
    NarrowBwdArgs a{};
    a.dy = f.dy; a.pre = f.pre; a.x = f.dweight ? f.x : nullptr; a.weight = f.weight;
    a.dy_stride = f.dy_stride; a.pre_stride = f.pre_stride; a.x_stride = f.x_stride;
    a.to.out = f.dx; a.to.out_stride = f.dx_stride; a.to.cols = f.in; a.to.clear = f.clear;
    a.in = f.in; a.out = f.out; a.chunk = p.chunk; a.size = p.size; a.groups = {f.ends, f.groups, f.rows}; a.act = f.act;
    const bool sums = f.dweight || f.dbias;
    if (sums) a.partial = reinterpret_cast<float*>(run.work.take(p.bytes));
    if (!run.real) return;
    if (f.rows) launch_narrow_bwd<T>(a, p, run.stream);
    if (!sums) return;
    JoinArgs j{};
    j.partial = a.partial; j.dweight = f.dweight; j.dbias = f.dbias; j.weights = f.in * f.out; j.size = p.size;
    j.wanted = f.dbias ? p.size : j.weights;
    j.groups = a.groups; j.step = p.chunk; j.slabs = f.ends || !f.rows ? 0 : p.blocks;
    join_weights<T>(j, p.blocks / f.groups + 1, run.stream);
}

template <class T>
void backward_few(const LinearBwdArgs& f, Run& run) {
    FewBwdArgs a{};
    a.dy = f.dy; a.pre = f.pre; a.x = f.x; a.weight = f.weight; a.dy_stride = f.dy_stride; a.pre_stride = f.pre_stride; a.x_stride = f.x_stride;
    a.dweight = f.dweight; a.dbias = f.dbias; a.in = f.in; a.out = f.out; a.groups = {f.ends, f.groups, f.rows}; a.act = f.act;
    const int64_t across = up(f.in, kFewBlock * kPer<T>);
    if (f.dx && f.rows) {
        // (slices of 32 outputs, of 16 where those were too few workgroups)
        a.slice = across * up(f.out, 32) * std::min<int64_t>(f.groups, f.rows) < 512 ? 16 : up(up(f.out, 256), 32) * 32;
        const int64_t slices = up(f.out, a.slice), slots = slots_of(f.rows, f.groups, kFewShift, f.ends != nullptr);
        a.partial = reinterpret_cast<float*>(run.work.take(slices * f.rows * f.in * 4));
        TileArgs t{};  // (what joins the slices)
        t.to.out = f.dx; t.to.out_stride = f.dx_stride; t.to.cols = f.in; t.to.clear = f.clear;
        t.rows = f.rows; t.groups = a.groups; t.partial = a.partial; t.splits = static_cast<int>(slices);
        if (run.real) {
            check_grid(across * slices * slots, kFewBlock);
            k_few_dx<T><<<dim3(static_cast<uint32_t>(across), static_cast<uint32_t>(slices), static_cast<uint32_t>(slots)), kFewBlock, 0, run.stream>>>(a);
            join_splits<T>(t, run.stream);
        }
    }
    if ((f.dweight || f.dbias) && run.real) {
        const int64_t down = up(f.out, 8), wide = f.dweight ? across : 1;
        check_grid(wide * down * f.groups, kFewBlock);
        k_few_dw<T><<<dim3(static_cast<uint32_t>(wide), static_cast<uint32_t>(down), static_cast<uint32_t>(f.groups)), kFewBlock, 0, run.stream>>>(a);
    }
}

template <class T>
void backward(const LinearBwdArgs& f, Run& run) {
    const bool ragged = f.ends != nullptr;
    const Groups groups{f.ends, f.groups, f.rows};
    if (const NarrowBwd p = plan_narrow_bwd(f.rows, f.in, f.out, f.groups, f.act != kNone && f.act != kRelu, sizeof(T)); p.blocks) {
        backward_narrow<T>(f, p, run);
        return;
    }
    if (few_rows_backward(f.rows, f.in, f.out, f.groups, sizeof(T))) {
        backward_few<T>(f, run);
        return;
    }
    // dz, where it is not dy itself, and its columns' sums
    Operand dz{f.dy, f.dy_stride, f.out};
    const bool products = f.dx || f.dweight, slopes = products && f.act;
    if (f.dbias || slopes) {
        const Slope slope = plan_slope(f.rows, f.out, f.groups, ragged, sizeof(T));
        SlopeArgs a{};
        a.dy = f.dy; a.pre = f.pre; a.dy_stride = f.dy_stride; a.pre_stride = f.pre_stride;
        a.cols = f.out; a.groups = groups; a.shift = slope.shift; a.act = f.act;
        if (slopes) {
            a.dz = run.work.take(slope.dz_bytes);
            a.dz_stride = slope.dz_stride;
            dz = {a.dz, slope.dz_stride, slope.dz_stride};
        }
        if (f.dbias) a.partial = reinterpret_cast<float*>(run.work.take(slope.bytes));
        if (run.real && f.rows) launch_slope<T>(a, slope, run.stream);
        if (run.real && f.dbias) {
            JoinArgs j{};
            j.partial = a.partial; j.dbias = f.dbias; j.wanted = j.size = f.out;
            j.groups = groups; j.step = int64_t{1} << slope.shift; j.from_begin = true;
            join_weights<T>(j, slope.slots / f.groups, run.stream);
        }
    }
    if (!products) return;
    if (!slopes) dz = operand<T>(f.dy, f.rows, f.out, f.dy_stride, f.dweight != nullptr, run);
    const int64_t kept = run.work.used();
    if (f.dx && f.rows) {
        const Operand w = operand<T>(f.weight, f.groups * f.out, f.in, f.in, true, run);
        TileArgs a{};
        a.row = dz.p; a.row_stride = dz.stride; a.col = w.p; a.col_stride = w.stride; a.col_group = w.stride * f.out; a.col_width = w.width;
        a.to.out = f.dx; a.to.out_stride = f.dx_stride; a.to.cols = f.in; a.to.clear = f.clear;
        a.rows = f.rows; a.depth = f.out; a.groups = groups;
        over_depth<T, true>(a, ragged, false, run);
        run.work.back_to(kept);
    }
    if (f.dweight) {
        const Operand x = operand<T>(f.x, f.rows, f.in, f.x_stride, true, run);
        const Over p = plan_over(f.rows, f.out, f.in, f.groups, ragged, sizeof(T));
        TileArgs a{};
        a.row = dz.p; a.row_stride = dz.stride; a.row_width = dz.width; a.col = x.p; a.col_stride = x.stride; a.col_width = x.width;
        a.to.out = f.dweight; a.to.out_stride = f.in; a.to.cols = f.in; a.out_group = f.in * f.out; a.rows = f.out; a.depth = f.rows;
        a.groups = groups; a.shift = p.shift; a.slots = p.slots;
        a.partial = p.bytes ? reinterpret_cast<float*>(run.work.take(p.bytes)) : nullptr;
        if (!run.real) return;
        launch_tiles<T, true, true>(a, p.side, p.slots, false, run.stream);
        if (a.partial) {
            JoinArgs j{};
            j.partial = a.partial; j.dweight = f.dweight; j.weights = j.wanted = j.size = f.in * f.out;
            j.groups = groups; j.step = int64_t{1} << p.shift; j.from_begin = true;
            join_weights<T>(j, p.slots / f.groups, run.stream);
        }
    }
}

}  // namespace
}  // namespace sxk
