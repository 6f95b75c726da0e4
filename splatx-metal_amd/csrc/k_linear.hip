// k_linear.hip — linear layers over rows, forward and backward, all rows with one weight or groups of rows with their own
// (include/splatx_hip.h has the formulas).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <stdexcept>
#include <string>

#include "sx_mma.h"

namespace sxk {
using namespace sxd;
namespace {

// ---- tiles ------------------------------------------------------------------------------------------------
//
// out[r][c] = sum over d of row(r, d) col(c, d): x W^T, dz W and dz^T x, each operand either with its sums' elements side by
// side in memory (plain) or with its rows side by side (Across: W's columns, dz's and x's).

struct TileArgs {
    const void *row, *col;
    int64_t row_stride, col_stride;  // elements between the rows in memory
    int64_t col_group;               // elements between the groups' col operands
    void* out;
    int64_t out_stride, out_group;
    int64_t rows, cols, depth;       // rows (of the products over rows), depth (of those over groups' rows): all groups'
    Groups groups;
    int shift;                       // the parts' rows, log2
    int64_t slots;
    float* partial;                  // [slabs][rows][cols] in place of out, or null
    int64_t split;                   // depth of a slab
    int splits;
    const void *bias, *residual;     // of out
    void* pre;
    int64_t bias_group, residual_stride, pre_stride;
    int act;
    bool clear;                      // rows behind the last group become zero
};

// Where the 16 bytes (row r, chunk c) of a plain operand's tile lie: 128 bytes a row, the chunks of eight rows in different
// places, so that lanes that read one chunk of several rows read different banks.
__device__ inline int plain_at(int r, int c) { return r * 128 + (c ^ (r & 7)) * 16; }
// Of an Across operand's tile: `row_bytes` a row of the sums' dimension; four rows' 32 bytes in different places.
template <class T>
__device__ inline int across_at(int m, int byte, int row_bytes) {
    return m * row_bytes + (sizeof(T) == 2 ? byte ^ ((m & 3) << 5) : byte);
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
    // Of the sums' dimension [d, d + kDepth), zeros from `end` on.
    __device__ void load(int64_t d, int64_t end) {
#pragma unroll
        for (int i = 0; i < N; i++) {
            const int l = line + i * kLines;
            if constexpr (Across) {
                v[i] = d + l < end ? load_within(base + (d + l) * stride, first + chunk * V, limit) : Frag<T>(0);
            } else {
                v[i] = load_within(base + min(first + l, limit - 1) * stride, d + chunk * V, end);
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

// What follows the sums: four columns from c on of row r.
template <class T>
__device__ inline void finish(const TileArgs& a, int group, int64_t r, int64_t c, Floats<4> v) {
    const int n = static_cast<int>(min(a.cols - c, int64_t{4}));
    if (n <= 0) return;
    if (a.bias) v += load_some<T, 4>(static_cast<const T*>(a.bias) + group * a.bias_group + c, n);
    if (a.pre) store_some<T, 4>(static_cast<T*>(a.pre) + r * a.pre_stride + c, v, n);
    if (a.act)
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] = activated<T>(v[e], a.act);
    if (a.residual) v += load_some<T, 4>(static_cast<const T*>(a.residual) + r * a.residual_stride + c, n);
    store_some<T, 4>(static_cast<T*>(a.out) + group * a.out_group + r * a.out_stride + c, v, n);
}
// The same of a row behind the last group.
template <class T>
__device__ inline void clear(const TileArgs& a, int64_t r, int64_t c) {
    const int n = static_cast<int>(min(a.cols - c, int64_t{4}));
    if (n <= 0 || !a.clear) return;
    store_some<T, 4>(static_cast<T*>(a.out) + r * a.out_stride + c, Floats<4>(0.0f), n);
    if (a.pre) store_some<T, 4>(static_cast<T*>(a.pre) + r * a.pre_stride + c, Floats<4>(0.0f), n);
}

// BR x BC outputs a workgroup, WR x WC a wave. OverRows: the sums go over a group's rows (dW), else the outputs' rows are the
// groups' rows.
template <class T, int BR, int BC, int WR, int WC, bool RowAcross, bool ColAcross>
__global__ void __launch_bounds__(BR / WR * (BC / WC) * 64) k_tile(TileArgs a) {
    constexpr bool OverRows = RowAcross;
    constexpr int kWaves = BR / WR * (BC / WC), kThreads = kWaves * 64, kDepth = 128 / static_cast<int>(sizeof(T));
    constexpr int kBuffer = (BR + BC) * 128, I = WR / 32, J = WC / 32;
    __shared__ __attribute__((aligned(128))) char lds[2 * kBuffer];
    // Which tile: workgroups go round the eight dies, and each die takes tiles side by side, eight rows of tiles at a time.
    const int64_t across = (a.cols + BC - 1) / BC, down = OverRows ? (a.rows + BR - 1) / BR : a.slots, tiles = across * down;
    const int64_t each = (tiles + 7) / 8, tile = blockIdx.x % 8 * each + blockIdx.x / 8;
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
    const int wave = threadIdx.x / 64, lane = threadIdx.x % 64;
    const int wr = wave / (BC / WC) * WR, wc = wave % (BC / WC) * WC;
    if (!OverRows && part.group >= a.groups.groups) {
        if (a.partial) return;
        for (int64_t r = r0 + threadIdx.x / 32; r < r1; r += kThreads / 32)
            for (int c = threadIdx.x % 32 * 4; c < BC; c += 128) clear<T>(a, r, c0 + c);
        return;
    }
    Sums sums[I][J];
#pragma unroll
    for (int i = 0; i < I; i++)
#pragma unroll
        for (int j = 0; j < J; j++) sums[i][j] = Sums(0.0f);
    Stage<T, BR, RowAcross, kThreads> row(static_cast<const T*>(a.row), a.row_stride, r0, r1);
    Stage<T, BC, ColAcross, kThreads> col(static_cast<const T*>(a.col) + part.group * a.col_group, a.col_stride, c0, a.cols);
    if (d0 < d1) {
        row.load(d0, d1);
        col.load(d0, d1);
        row.store(lds);
        col.store(lds + BR * 128);
    }
    __syncthreads();
    int now = 0;
    for (int64_t d = d0; d < d1; d += kDepth) {
        const bool more = d + kDepth < d1;
        if (more) {
            row.load(d + kDepth, d1);
            col.load(d + kDepth, d1);
        }
        const char* buffer = lds + now * kBuffer;
#pragma unroll
        for (int s = 0; s < 4; s++) {
            Frag<T> fr[I], fc[J];
#pragma unroll
            for (int i = 0; i < I; i++) fr[i] = fragment<T, BR, RowAcross>(buffer, wr + i * 32, s);
#pragma unroll
            for (int j = 0; j < J; j++) fc[j] = fragment<T, BC, ColAcross>(buffer + BR * 128, wc + j * 32, s);
#pragma unroll
            for (int i = 0; i < I; i++)
#pragma unroll
                for (int j = 0; j < J; j++) mma(sums[i][j], fc[j], fr[i]);
        }
        now ^= 1;
        if (more) {
            row.store(lds + now * kBuffer);
            col.store(lds + now * kBuffer + BR * 128);
        }
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < I; i++) {
        const int64_t r = r0 + wr + i * 32 + lane % 32;
        if (r >= r1) continue;
#pragma unroll
        for (int j = 0; j < J; j++)
#pragma unroll
            for (int q = 0; q < 4; q++) {
                const int64_t c = c0 + wc + j * 32 + 8 * q + lane / 32 * 4;
                const Floats<4> v = {sums[i][j][4 * q], sums[i][j][4 * q + 1], sums[i][j][4 * q + 2], sums[i][j][4 * q + 3]};
                if (a.partial) {
                    const int n = static_cast<int>(min(a.cols - c, int64_t{4}));
                    if (n > 0) store_some<float, 4>(a.partial + (int64_t{blockIdx.y} * a.rows + r) * a.cols + c, v, n);
                } else {
                    finish<T>(a, part.group, r, c, v);
                }
            }
    }
}

// The slabs of partial sums, added in order. Over rows: group blockIdx.z's slots, else all splits.
template <class T, bool OverRows>
__global__ void __launch_bounds__(256) k_tile_join(TileArgs a) {
    const int64_t quads = (a.cols + 3) / 4;
    int group = OverRows ? blockIdx.y : 0;
    int64_t first = 0, slabs = a.splits;
    if constexpr (OverRows) {
        const int64_t begin = a.groups.begin(group), end = a.groups.end(group);
        first = group + (begin >> a.shift);
        slabs = end > begin ? ((end - begin - 1) >> a.shift) + 1 : 0;
    }
    for (int64_t i = blockIdx.x * int64_t{256} + threadIdx.x; i < a.rows * quads; i += gridDim.x * int64_t{256}) {
        const int64_t r = i / quads, c = i % quads * 4;
        const int n = static_cast<int>(min(a.cols - c, int64_t{4}));
        if constexpr (!OverRows) {
            if (a.groups.ends) {
                int lo = 0, hi = a.groups.groups;  // the first group that ends behind the row
                while (lo < hi) {
                    const int mid = (lo + hi) / 2;
                    if (a.groups.end(mid) <= r) lo = mid + 1;
                    else hi = mid;
                }
                group = lo;
                if (group >= a.groups.groups) {
                    clear<T>(a, r, c);
                    continue;
                }
            }
        }
        Floats<4> sum(0.0f);
        for (int64_t s = 0; s < slabs; s++) sum += load_some<float, 4>(a.partial + ((first + s) * a.rows + r) * a.cols + c, n);
        finish<T>(a, group, r, c, sum);
    }
}

// ---- dz = dy act'(pre), and its columns' sums ------------------------------------------------------------

struct SlopeArgs {
    const void *dy, *pre;
    void* dz;            // [rows][dz_stride], or null
    float* partial;      // [slots][cols], or null
    void* dbias;
    int64_t dy_stride, pre_stride, dz_stride, cols;
    Groups groups;
    int shift, act;
};

// A part of the rows and up to 256 vectors of columns a workgroup; `lanes` threads go along a row.
template <class T>
__global__ void __launch_bounds__(256) k_slope(SlopeArgs a, int lanes) {
    constexpr int V = kPer<T>;
    __shared__ Floats<V> sums[256];
    const Part part = part_of(a.groups, blockIdx.x, a.shift);
    if (part.group >= a.groups.groups || part.begin >= part.end) return;
    const int64_t c = (int64_t{blockIdx.y} * lanes + threadIdx.x % lanes) * V;
    Floats<V> sum(0.0f);
    if (c < a.cols) {
        const int n = static_cast<int>(min(a.cols - c, int64_t{V}));
        for (int64_t r = part.begin + threadIdx.x / lanes; r < part.end; r += 256 / lanes) {
            Floats<V> d = floats<T, V>(load_within(static_cast<const T*>(a.dy) + r * a.dy_stride, c, a.cols));
            if (a.act) {
                const Floats<V> z = floats<T, V>(load_within(static_cast<const T*>(a.pre) + r * a.pre_stride, c, a.cols));
#pragma unroll
                for (int e = 0; e < V; e++) d[e] = through<T>(d[e], z[e], a.act);
                if (a.dz) store_some<T, V>(static_cast<T*>(a.dz) + r * a.dz_stride + c, d, n);
            }
            sum += d;
        }
    }
    if (!a.partial) return;
    sums[threadIdx.x] = sum;
    __syncthreads();
    if (static_cast<int>(threadIdx.x) >= lanes || c >= a.cols) return;
    for (int t = threadIdx.x + lanes; t < 256; t += lanes) sum += sums[t];
    store_some<float, V>(a.partial + int64_t{blockIdx.x} * a.cols + c, sum, static_cast<int>(min(a.cols - c, int64_t{V})));
}

// A group's partial sums, added in order: sixteen columns a workgroup, as many threads a column.
template <class T>
__global__ void __launch_bounds__(256) k_slope_join(SlopeArgs a) {
    __shared__ float part[16][17];
    const int lane = threadIdx.x % 16, turn = threadIdx.x / 16;
    const int64_t c = int64_t{blockIdx.x} * 16 + lane;
    const int group = blockIdx.y;
    const int64_t begin = a.groups.begin(group), end = a.groups.end(group), first = group + (begin >> a.shift);
    const int64_t slabs = end > begin ? ((end - begin - 1) >> a.shift) + 1 : 0;
    float sum = 0.0f;
    if (c < a.cols)
        for (int64_t s = turn; s < slabs; s += 16) sum += a.partial[(first + s) * a.cols + c];
    part[turn][lane] = sum;
    __syncthreads();
    if (turn || c >= a.cols) return;
    for (int t = 1; t < 16; t++) sum += part[t][lane];
    static_cast<T*>(a.dbias)[group * a.cols + c] = static_cast<T>(sum);
}

// ---- plans ------------------------------------------------------------------------------------------------

constexpr int64_t kManyTiles = 512;  // two workgroups for each unit
int log2_up(int64_t n) {
    int k = 0;
    while ((int64_t{1} << k) < n) k++;
    return k;
}
int64_t up(int64_t n, int64_t to) { return (n + to - 1) / to; }

// out[rows][cols] over `depth`, rows in groups: the tile's side, and how many parts the depth is split into.
struct Plan {
    int side, splits;
    int64_t split, bytes;
};
Plan plan_rows(int64_t rows, int64_t cols, int64_t depth, int groups, bool ragged, int elem) {
    Plan p{128, 1, 0, 0};
    const auto tiles = [&](int side) { return slots_of(rows, groups, log2_up(side), ragged) * up(cols, side); };
    if (tiles(128) < kManyTiles) p.side = 64;
    const int64_t step = 128 / elem, steps = up(depth, step);
    if (p.side == 64) p.splits = static_cast<int>(std::max<int64_t>(1, std::min(kManyTiles / std::max<int64_t>(tiles(64), 1), steps / 4)));
    const int64_t each = up(steps, p.splits);
    p.split = each * step;
    p.splits = static_cast<int>(std::max<int64_t>(1, up(steps, std::max<int64_t>(each, 1))));
    p.bytes = p.splits > 1 ? p.splits * rows * cols * 4 : 0;
    return p;
}
// out[groups][out][in] over the groups' rows: the tile's side, and the parts of the rows (shift 62: each group's are one).
struct Over {
    int side, shift;
    int64_t slots, bytes;
};
Over plan_over(int64_t rows, int64_t out, int64_t in, int groups, bool ragged) {
    Over p{128, 62, groups, 0};
    if (std::max(out, in) <= 64) p.side = 64;
    const int64_t tiles = up(out, p.side) * up(in, p.side);
    const int64_t wanted = std::max<int64_t>(1, 2 * kManyTiles / tiles);
    const bool direct = tiles * groups >= kManyTiles && tiles >= 32;
    const int shift = std::max(8, log2_up(up(std::max<int64_t>(rows, 1), wanted)));
    if (!direct && rows > int64_t{1} << shift) {
        p.shift = shift;
        p.slots = slots_of(rows, groups, shift, ragged);
        p.bytes = p.slots * out * in * 4;
    }
    return p;
}
struct Slope {
    int shift, lanes;
    int64_t slots, columns, bytes, dz_stride, dz_bytes;
};
Slope plan_slope(int64_t rows, int64_t cols, int groups, bool ragged, int elem) {
    Slope p{};
    const int64_t vectors = up(cols, 16 / elem);
    p.lanes = 1 << std::min(8, log2_up(vectors));
    p.columns = up(vectors, p.lanes);
    p.shift = std::max({log2_up(256 / p.lanes), 4, log2_up(up(std::max<int64_t>(rows, 1), std::max<int64_t>(1, 2048 / p.columns)))});
    p.slots = slots_of(rows, groups, p.shift, ragged);
    p.bytes = p.slots * cols * 4;
    p.dz_stride = vectors * (16 / elem);
    p.dz_bytes = rows * p.dz_stride * elem;
    return p;
}

constexpr int64_t kAlign = 256;
int64_t aligned(int64_t bytes) { return (bytes + kAlign - 1) / kAlign * kAlign; }

void check_grid(int64_t blocks, int64_t threads) {
    if (blocks * threads >= int64_t{1} << 32) throw std::runtime_error("linear: more workgroups than a launch holds");
}

template <class T, bool RowAcross, bool ColAcross>
void launch_tiles(const TileArgs& a, int side, int64_t slabs, hipStream_t s) {
    const int64_t down = RowAcross ? up(a.rows, side) : a.slots, tiles = up(down * up(a.cols, side), 8) * 8;
    check_grid(tiles * slabs, 256);
    const dim3 grid(static_cast<uint32_t>(tiles), static_cast<uint32_t>(slabs));
    if (side == 128) k_tile<T, 128, 128, 64, 64, RowAcross, ColAcross><<<grid, 256, 0, s>>>(a);
    else k_tile<T, 64, 64, 32, 32, RowAcross, ColAcross><<<grid, 256, 0, s>>>(a);
}

template <class T, bool OverRows>
void join_tiles(const TileArgs& a, int groups, hipStream_t s) {
    const int64_t blocks = std::min<int64_t>(up(a.rows * up(a.cols, 4), 256), 4096);
    k_tile_join<T, OverRows><<<dim3(static_cast<uint32_t>(blocks), static_cast<uint32_t>(groups)), 256, 0, s>>>(a);
}

// out = row col^T over the groups' rows (see TileArgs), with what follows.
template <class T, bool ColAcross>
void over_depth(TileArgs a, bool ragged, float* work, hipStream_t s) {
    const Plan p = plan_rows(a.rows, a.cols, a.depth, a.groups.groups, ragged, sizeof(T));
    a.shift = log2_up(p.side);
    a.slots = slots_of(a.rows, a.groups.groups, a.shift, ragged);
    a.split = p.split;
    a.splits = p.splits;
    a.partial = p.splits > 1 ? work : nullptr;
    launch_tiles<T, false, ColAcross>(a, p.side, p.splits, s);
    if (a.partial) join_tiles<T, false>(a, 1, s);
}

template <class T>
void forward(const LinearFwdArgs& f, hipStream_t s) {
    TileArgs a{};
    a.row = f.x; a.row_stride = f.x_stride; a.col = f.weight; a.col_stride = f.in; a.col_group = f.in * f.out;
    a.out = f.y; a.out_stride = f.y_stride; a.rows = f.rows; a.cols = f.out; a.depth = f.in;
    a.groups = {f.ends, f.groups, f.rows};
    a.bias = f.bias; a.bias_group = f.out; a.residual = f.residual; a.residual_stride = f.residual_stride;
    a.pre = f.pre; a.pre_stride = f.pre_stride; a.act = f.act; a.clear = f.clear;
    over_depth<T, false>(a, f.ends != nullptr, static_cast<float*>(f.workspace), s);
}

template <class T>
void backward(const LinearBwdArgs& f, hipStream_t s) {
    const bool ragged = f.ends != nullptr;
    const Slope slope = plan_slope(f.rows, f.out, f.groups, ragged, sizeof(T));
    const Groups groups{f.ends, f.groups, f.rows};
    char* work = static_cast<char*>(f.workspace);
    const void* dz = f.dy;
    int64_t dz_stride = f.dy_stride;
    const bool products = f.dx || f.dweight;
    if (f.dbias || (f.act && products)) {
        SlopeArgs a{};
        a.dy = f.dy; a.pre = f.pre; a.dy_stride = f.dy_stride; a.pre_stride = f.pre_stride;
        a.cols = f.out; a.groups = groups; a.shift = slope.shift; a.act = f.act; a.dbias = f.dbias;
        if (f.act && products) {
            a.dz = work;
            dz = work;
            dz_stride = a.dz_stride = slope.dz_stride;
        }
        work += aligned(slope.dz_bytes);
        if (f.dbias) a.partial = reinterpret_cast<float*>(work);
        work += aligned(slope.bytes);
        check_grid(slope.slots * slope.columns, 256);
        if (f.rows)
            k_slope<T><<<dim3(static_cast<uint32_t>(slope.slots), static_cast<uint32_t>(slope.columns)), 256, 0, s>>>(a, slope.lanes);
        if (f.dbias) k_slope_join<T><<<dim3(static_cast<uint32_t>(up(f.out, 16)), static_cast<uint32_t>(f.groups)), 256, 0, s>>>(a);
    }
    if (f.dx && f.rows) {
        TileArgs a{};
        a.row = dz; a.row_stride = dz_stride; a.col = f.weight; a.col_stride = f.in; a.col_group = f.in * f.out;
        a.out = f.dx; a.out_stride = f.dx_stride; a.rows = f.rows; a.cols = f.in; a.depth = f.out;
        a.groups = groups; a.clear = f.clear;
        over_depth<T, true>(a, ragged, reinterpret_cast<float*>(work), s);
    }
    if (f.dweight) {
        const Over p = plan_over(f.rows, f.out, f.in, f.groups, ragged);
        TileArgs a{};
        a.row = dz; a.row_stride = dz_stride; a.col = f.x; a.col_stride = f.x_stride;
        a.out = f.dweight; a.out_stride = f.in; a.out_group = f.in * f.out; a.rows = f.out; a.cols = f.in; a.depth = f.rows;
        a.groups = groups; a.shift = p.shift; a.slots = p.slots;
        a.partial = p.bytes ? reinterpret_cast<float*>(work) : nullptr;
        launch_tiles<T, true, true>(a, p.side, p.slots, s);
        if (a.partial) join_tiles<T, true>(a, f.groups, s);
    }
}

template <class F>
void with_type(ElemType t, F&& f) {
    if (t == kF32) f(float{});
    else if (t == kBf16) f(__bf16{});
    else f(_Float16{});
}

}  // namespace

int64_t linear_fwd_workspace(int64_t rows, int64_t in, int64_t out, int groups, bool ragged, ElemType type) {
    return plan_rows(rows, out, in, groups, ragged, type == kF32 ? 4 : 2).bytes;
}
int64_t linear_bwd_workspace(int64_t rows, int64_t in, int64_t out, int groups, bool ragged, ElemType type) {
    const int elem = type == kF32 ? 4 : 2;
    const Slope slope = plan_slope(rows, out, groups, ragged, elem);
    return aligned(slope.dz_bytes) + aligned(slope.bytes) +
           std::max(plan_rows(rows, in, out, groups, ragged, elem).bytes, plan_over(rows, out, in, groups, ragged).bytes);
}
void linear_fwd(const LinearFwdArgs& a, ElemType type, hipStream_t s) {
    with_type(type, [&](auto t) { forward<decltype(t)>(a, s); });
}
void linear_bwd(const LinearBwdArgs& a, ElemType type, hipStream_t s) {
    with_type(type, [&](auto t) { backward<decltype(t)>(a, s); });
}

}  // namespace sxk
