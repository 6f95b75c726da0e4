// sx_linear_plan.h — how the linear layers' calls are divided (sx_linear.h has the kernels): which kernels take one, their tiles,
// parts, workgroups, LDS and workspace, from sizes and types alone. Plain C++, so that any compiler checks it over all sizes.
// `elem` is the elements' bytes, 4 or 2.
#pragma once

#include <algorithm>
#include <cmath>
#include <cstdint>

namespace sxk {
namespace {

int log2_up(int64_t n) {
    int k = 0;
    while ((int64_t{1} << k) < n) k++;
    return k;
}
int64_t up(int64_t n, int64_t to) { return (n + to - 1) / to; }
// Slots of a division of all groups' rows into parts of 2^shift (Groups and part_of in sx_mma.h).
int64_t slots_of(int64_t rows, int groups, int shift, bool ragged) {
    return ragged ? groups + 1 + (rows >> shift) : ((rows + (int64_t{1} << shift) - 1) >> shift);
}

// Few rows: a forward's workgroups have kFewWaves waves for a part of 2^kFewShift rows, a backward up to kFewRows rows and kFewBlock
// threads a workgroup.
constexpr int kFewWaves = 8, kFewShift = 5, kFewRows = 32, kFewBlock = 128;

// ---- LDS ----------------------------------------------------------------------------------------------------

constexpr int kLds = 160 * 1024;  // a workgroup's most

// A wave's outputs on their way to whole lines (Unit in sx_linear.h): `unit_tiles` tiles of 32 columns side by side, as floats, 32
// lines (of eight rows in different banks), and of sums that are the outputs in the type.
constexpr int unit_tiles(int elem) { return 4 / elem; }
constexpr int unit_line(int elem) { return unit_tiles(elem) * 128 + 16; }
constexpr int unit_bytes(int elem) { return 32 * unit_line(elem); }
constexpr int kBareLine = 128 + 16;
constexpr int kBareBytes = 32 * kBareLine;
// A narrow backward's block of rows, and the bytes between its lines: `tiles` times 32 elements, and what puts four lines (floats:
// the lanes' lines) into different banks.
constexpr int block_rows(int elem) { return 256 / elem; }
constexpr int line_bytes(int tiles, int elem) { return tiles * 32 * elem + (elem == 2 ? 32 : 16); }

// ---- tiles --------------------------------------------------------------------------------------------------

// The tiles to choose from: their rows and columns, how many run at once on 256 units, and what a step of 128 bytes of the
// sums' length then takes, in ns of 16-bit elements, and what a tile takes besides. Measured on layers of 16,383 rows, 8192 to
// 2048: 542, 623 and 712 us by tiles of 256, 128 and 64 rows; 20,001 rows in 16 groups, 1024 to 1408, whose tiles of 256 rows
// take three rounds for two: 121, 104 and 106.
struct TileKind {
    int rows, cols, at_once;
    double step, fixed, float_step;
};
constexpr TileKind kTileKinds[] = {{256, 256, 256, 1950, 6000, 0}, {128, 128, 512, 1150, 3000, 1860}, {64, 128, 768, 1050, 2500, 950}};
constexpr double kJoinFixed = 4000, kJoinBytes = 4;  // ns; bytes a ns
// `tiles` of `steps` each; a unit's only workgroup of a kind that shares it goes faster. Floats' sums over rows, whose operands both
// come from memory as long as they last, as 16-bit elements of 4.6 times the step: what runs side by side hides loads (300,000 rows of
// 64 to 144, gradients 465 us; 650 by the figures below, which choose parts that fill each unit once).
double tiles_take(const TileKind& k, double tiles, double steps, int elem) {
    const double step = k.step * (elem == 4 ? 4.6 : 1.0) * (tiles <= 256 && k.at_once > 256 ? 0.6 : 1.0);
    return std::max(1.0, std::ceil(tiles / k.at_once)) * (k.fixed + steps * step);
}
// The same of floats' sums over features, in `parts` whose sums are `bytes`. Their products fill a unit by one workgroup, and what shares
// it waits for them (one of 128 rows leaves a twelfth); loads and stores at the ends hide behind the others' products but for those
// that run at once. 429 rows of 5312 to 1072, us: 36 tiles of 128 rows whole 330, in 6 parts (216) 67, in 8 (288, more than units) 93;
// 63 tiles of 64 rows whole 168, in 4 parts (252) 52, in 8 54, in 12 (756, 22 MB of sums) 57, in 16 (more than run at once) 75.
// 4096 cubed 980 and 1017.
double float_tiles_take(const TileKind& k, double tiles, double steps, int64_t parts, int64_t bytes) {
    return 9000 + (std::ceil(std::max(1.0, tiles / k.at_once)) - 1) * 8000 +
           std::max(1.0, std::ceil(tiles / 256)) * steps * k.float_step * (k.rows == 128 && tiles <= 256 ? 1.08 : 1.0) +
           (parts > 1 ? 2000 + static_cast<double>(bytes) * 1e-4 : 0.0);
}

// A tile's lines in memory, those of an operand's rows, may be so many bytes apart: then what a lane adds to its load's beginning,
// which is 32 bits, is `plain_offset` or `across_offset`. (A row of the most elements, 2^24 floats.)
constexpr int64_t kMostLine = int64_t{1} << 26;
constexpr int kTileDepthBytes = 128;
// Plain: a load of a wave's takes 128 bytes of each of eight lines, from a beginning of its own. Across: whole rows of a tile's
// depth, from the tile's beginning.
constexpr int kLoadLines = 8;
constexpr int64_t plain_offset(int64_t lines, int64_t line, int chunk) { return lines * line + chunk * 16; }
constexpr int64_t across_offset(int64_t lines, int64_t line, int64_t byte) { return lines * line + byte; }

// out[rows][cols] over `depth`, rows in groups: the tile's rows, and how many parts the depth is split into.
struct Plan {
    int side, splits;
    int64_t split, bytes;
};
Plan plan_rows(int64_t rows, int64_t cols, int64_t depth, int groups, bool ragged, int elem) {
    const int64_t step = 128 / elem, steps = up(depth, step);
    Plan best{};
    double least = INFINITY;
    for (const TileKind& k : kTileKinds) {
        if (elem == 4 && k.rows == 256) continue;  // (floats' products are 16 times as long as their reads: 128 are enough)
        // (a group's last tile is half full)
        const double down = ragged ? static_cast<double>(rows) / k.rows + 0.5 * static_cast<double>(std::min<int64_t>(groups, rows)) : static_cast<double>(up(rows, k.rows));
        const double tiles = down * static_cast<double>(up(cols, k.cols));
        for (int64_t splits = 1; splits <= 64 && (splits == 1 || steps / splits >= 2); splits += elem == 2 ? splits : splits < 16 ? 1 : 4) {
            const int64_t each = up(steps, splits), parts = up(steps, each), bytes = parts > 1 ? parts * rows * cols * 4 : 0;
            if (bytes > int64_t{64} << 20) break;
            const double all = tiles * static_cast<double>(parts), length = static_cast<double>(each);
            const double time = elem == 4 ? float_tiles_take(k, all, length, parts, bytes)
                                          : tiles_take(k, all, length, elem) + (parts > 1 ? kJoinFixed + 2.0 * static_cast<double>(bytes) / kJoinBytes / 1000 : 0.0);
            if (time < least) {
                least = time;
                best = {k.rows, static_cast<int>(parts), each * step, bytes};
            }
        }
    }
    return best;
}
// Whether a forward of floats reads operands that do not lie for its tiles through registers rather than copy them first: the copies
// take two passes over them and a launch each, the registers a fifth of what the products take. (us so and with copies: 81 rows of
// 1835 to 7894 53 and 69, 44 of 6309 to 2451 45 and 66, 16,384 of 513 to 512 93 and 100; 4097 cubed 1294 and 1220. A backward's tiles,
// which read across the rows, took half as long again.)
bool staged_pays(int64_t rows, int64_t in, int64_t out, int groups, bool copy_x, bool copy_w) {
    const double passes = 2.0 * 4 * static_cast<double>(in) * (copy_x * static_cast<double>(rows) + copy_w * static_cast<double>(groups) * static_cast<double>(out));
    const double copies = passes / 4500 + 4000 * (copy_x + copy_w), products = 2.0 * static_cast<double>(rows) * static_cast<double>(in) * static_cast<double>(out) / 140'000;
    return copies > 0.2 * products;
}
// out[groups][out][in] over the groups' rows: the tile's rows, and the parts of the rows (shift 62: each group's are one).
struct Over {
    int side, shift;
    int64_t slots, bytes;
};
Over plan_over(int64_t rows, int64_t out, int64_t in, int groups, bool ragged, int elem) {
    const double step = 128.0 / elem, all = static_cast<double>(rows) / step;
    Over best{};
    double least = INFINITY;
    for (const TileKind& k : kTileKinds) {
        if (elem == 4 && k.rows == 256) continue;
        const double tiles = static_cast<double>(up(out, k.rows) * up(in, k.cols));
        // one part each: the largest group is taken to have three times an even share
        const double even = tiles_take(k, tiles * groups, all / groups, elem);
        double time = std::max(even, groups > 1 ? tiles_take(k, 1, std::min(all, 3 * all / groups), elem) : 0.0);
        if (time < least) {
            least = time;
            best = {k.rows, 62, groups, 0};
        }
        for (int shift = 8; (int64_t{1} << shift) < rows; shift++) {
            const int64_t slots = slots_of(rows, groups, shift, ragged), bytes = slots * out * in * 4;
            if (bytes > int64_t{256} << 20 || slots > 65535) continue;
            const double parts = ragged ? static_cast<double>(rows >> shift) + 0.5 * groups : static_cast<double>(slots);
            time = tiles_take(k, tiles * parts, static_cast<double>(int64_t{1} << shift) / step, elem) + kJoinFixed +
                   2.0 * parts * static_cast<double>(out * in) * 4 / kJoinBytes / 1000;
            if (time < least) {
                least = time;
                best = {k.rows, shift, slots, bytes};
            }
        }
    }
    return best;
}
struct Slope {
    int shift, lanes;
    int64_t slots, columns, bytes, dz_stride, dz_bytes;
};
Slope plan_slope(int64_t rows, int64_t cols, int groups, bool ragged, int elem) {
    Slope p{};
    const int64_t vectors = up(cols, 16 / elem);
    p.lanes = static_cast<int>(std::min<int64_t>(vectors, 256));
    p.columns = up(vectors, p.lanes);
    p.shift = std::max({log2_up(256 / p.lanes) + 2, log2_up(up(std::max<int64_t>(rows, 1), std::max<int64_t>(1, 1024 / p.columns)))});
    p.slots = slots_of(rows, groups, p.shift, ragged);
    p.bytes = p.slots * cols * 4;
    p.dz_stride = vectors * (16 / elem);
    p.dz_bytes = rows * p.dz_stride * elem;
    return p;
}

// ---- narrow layers ------------------------------------------------------------------------------------------

// The steps of 32 bytes of a row that k_narrow_fwd is built for, or 0.
int narrow_steps(int64_t in, int elem) {
    for (const int k : {1, 2, 3, 4, 6, 8, 12, 16})
        if (in * elem <= k * 32) return k;
    return 0;
}
// A layer whose weight a workgroup holds: its LDS and workgroups, or none.
struct Narrow {
    int steps, threads, lds;
    int64_t blocks, chunk;
};
Narrow plan_narrow(int64_t rows, int64_t in, int64_t out, bool ragged, int elem) {
    Narrow p{};
    const int steps = narrow_steps(in, elem);
    const int64_t tiles = elem == 4 ? up(out, 32) : up(out, 64) * 2, kib = tiles * steps;
    if (!steps || kib > 112 || (rows < 4096 && kib > 16)) return p;
    const int held = static_cast<int>(kib * 1024 + tiles * 128), eight = held + 8 * unit_bytes(elem);
    // Where eight waves' outputs have no room beside the weight four waves' have. Four waves alone on a unit hide less, and each
    // workgroup fetches the weight: they pay for short rows, many of them, of one group; else tiles take the layer. (bfloat16 and half,
    // us of four waves and by tiles: 1 M rows 64 to 768 462 and 630, 300,000 rows 96 to 512 136 and 194, 40,000 rows 38 and 33;
    // 100,000 rows 128 to 384 56 and 44; 4096 rows 64 to 768 26 and 8; 300,000 rows in 16 groups 64 to 768 396 and 217.)
    if (eight > kLds && (steps > 6 || ragged || rows < 65536)) return p;
    p.steps = steps;
    p.threads = kib > 32 && eight <= kLds ? 512 : 256;
    p.lds = held + p.threads / 64 * unit_bytes(elem);
    // with groups more workgroups than run at once: the rows worked on at a time lie closer together (1 M rows of 64 in 200 groups,
    // 3 for each unit 90 us, 8 86)
    const int64_t each = ragged ? 8 : std::min(p.threads == 512 ? 2 : 4, kLds / p.lds);
    p.blocks = std::max<int64_t>(1, std::min<int64_t>(256 * each, up(rows, p.threads / 2)));
    p.chunk = std::max<int64_t>(up(up(rows, p.blocks), 32) * 32, 32);
    p.blocks = std::max<int64_t>(up(rows, p.chunk), 1);
    return p;
}
// A layer of floats with longer rows than those (`lines` of 128 bytes, the last may end early) and up to two tiles of 32 outputs, whose
// weight a workgroup holds: or none. Each workgroup fetches the weight, and again for each group: it pays for many
// rows, a thousand of each group. (us so and by tiles: 158,303 rows of 178 to 2 43 and 138, 1 M of 192 to 64 301 and 570, 32,768 23
// and 24.8, 16,384 24 and 13; 300,000 in 200 groups of 200 to 32 119 and 192, 100,000 of 300 to 64 155 and 112.)
struct Long {
    int lines, tiles, threads, lds;
    int64_t blocks, chunk;
};
Long plan_long(int64_t rows, int64_t in, int64_t out, int groups, bool ragged) {
    Long p{};
    const int64_t lines = up(in, 32), tiles = up(out, 32), weight = tiles * (lines * 4096 + 128);
    // (four waves where eight would leave units a workgroup or two of all, and two of four fit: 66,580 rows of 288 to 16 36 us and 45; one
    // of four of 49,152 rows of 900 to 32 78 and 57)
    p.threads = rows < 256 * 512 && 2 * (weight + 4 * unit_bytes(4)) <= kLds ? 256 : 512;
    const int64_t lds = weight + p.threads / 64 * unit_bytes(4);
    if (narrow_steps(in, 4) || tiles > 2 || lds > kLds || rows < 32768 || rows / groups < 1024) return p;
    p.lines = static_cast<int>(lines);
    p.tiles = static_cast<int>(tiles);
    p.lds = static_cast<int>(lds);
    p.blocks = std::min<int64_t>(256 * (ragged ? 8 : std::min(p.threads == 512 ? 2 : 4, kLds / p.lds)), up(rows, p.threads / 2));
    p.chunk = up(up(rows, p.blocks), 32) * 32;
    p.blocks = up(rows, p.chunk);
    return p;
}
// A backward whose blocks of rows a workgroup holds.
struct NarrowBwd {
    int waves, zt, xt, lds;
    bool fine;
    int64_t blocks, chunk, size, bytes;
};
NarrowBwd plan_narrow_bwd(int64_t rows, int64_t in, int64_t out, int groups, bool curved, int elem) {
    NarrowBwd p{};
    const int64_t kt = up(in, 32);
    // dz is rounded to the type for its products, by which dx and dweight lose about what their own rounding takes, element for
    // element: of all together 1.4 times the error of floats' products. Of a gradient of few elements that sum of errors varies, and
    // may be more of the whole (11 rows of 26 to 62: dx's 1.5 times its own rounding's): under 1024 elements dz is two terms, where the
    // kernel holds those. (600,000 rows, 20 to 30, bfloat16: 76 us in one, 84 in two; 1 M of 64 to 64 125 and 224, for two terms
    // leave a unit one workgroup. Wider layers with such a gradient and more than 32 rows, 100 rows of 3 to 300, take one term.)
    // (dy itself, and what relu leaves of it, has no more digits than the type.)
    const bool wanted = elem == 2 && curved && std::min(in * out, rows * in) < 1024;
    p.fine = wanted && (out <= 32 || (out <= 64 && kt <= 4) || (out <= 128 && kt <= 2));
    if (wanted && !p.fine && rows <= kFewRows) return p;  // (the few rows' kernels keep floats)
    const int64_t nt = up(out, 32) * (p.fine ? 2 : 1);
    if (nt <= 2 && kt <= 2) p.waves = 4, p.zt = p.xt = 2;
    else if (elem == 4) {  // (blocks of 64 rows of more floats do not fit; 919,424 rows, 32 to 80, by tiles 2,400 us, so 500)
        if (nt <= 4 && kt <= 2) p.waves = 8, p.zt = 4, p.xt = 2;
        else if (nt <= 2 && kt <= 4) p.waves = 8, p.zt = 2, p.xt = 4;
        else return p;
    } else if (nt <= 4 && kt <= 4) p.waves = 8, p.zt = p.xt = 4;
    else if (nt <= 2 && kt <= 8) p.waves = 8, p.zt = 2, p.xt = 8;
    else if (nt <= 8 && kt <= 2) p.waves = 8, p.zt = 8, p.xt = 2;
    else return p;
    p.lds = block_rows(elem) * (line_bytes(p.zt, elem) + line_bytes(p.xt, elem)) + p.waves * kBareBytes + p.zt * p.xt * elem * 1024;
    static_assert(block_rows(2) * (line_bytes(2, 2) + line_bytes(8, 2)) + 8 * kBareBytes + 16 * 2048 <= kLds);
    const int64_t each = std::min(2, kLds / p.lds);
    p.blocks = std::max<int64_t>(1, std::min<int64_t>(256 * each, up(rows, block_rows(elem))));
    p.chunk = std::max<int64_t>(up(up(rows, p.blocks), 32) * 32, 32);
    p.blocks = std::max<int64_t>(up(rows, p.chunk), 1);
    p.size = in * out + out;
    p.bytes = (p.blocks + groups) * p.size * 4;
    return p;
}

// ---- few rows -----------------------------------------------------------------------------------------------

// Whether a forward's groups have so few rows that the weights' bytes are what it takes (and its workgroups fit a launch). Of floats,
// whose tiles are slower next to their bytes, more, and more again where their lines would have to be copied (us here and by tiles:
// 64 rows of 4096 to 4096 25.5 and 27.0, of 4097 25.7 and 34.2; 96 of 4096 45.4 and 41.7, of 4097 46.6 and 55.9; 81 of 1835 to 7894
// 46.0 and 53.4).
bool few_rows(int64_t rows, int64_t out, int groups, int elem, bool whole_lines) {
    return (rows <= (elem == 2 ? 32 : whole_lines ? 64 : 128) || rows / groups <= 16) && up(out, 32) * (groups + 1 + (rows >> kFewShift)) < int64_t{1} << 22;
}
// Whether a backward's rows are.
bool few_rows_backward(int64_t rows, int64_t in, int64_t out, int groups, int elem) {
    return rows <= kFewRows && out <= 8 * 65535 && up(in, kFewBlock * 16 / elem) * up(out, 8) * groups < int64_t{1} << 24;
}

}  // namespace
}  // namespace sxk
