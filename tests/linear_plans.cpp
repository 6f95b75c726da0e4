// Every plan of the linear layers over their sizes, against what a workgroup and a launch can hold: the plans that do not fit, one a
// line, and how many were looked at.
#include <cstdio>

#include "sx_linear_plan.h"

using namespace sxk;

namespace {

constexpr int kMostLds = 163840;  // of a workgroup, bytes
long looked = 0;

void narrow() {
    for (const int elem : {2, 4})
        for (int in = 1; in <= 520 / elem; in++)
            for (int out = 1; out <= 3700; out++)
                for (const long rows : {1L, 1000L, 4095L, 4096L, 100'000L, 40'000'000L})
                    for (const bool ragged : {false, true}) {
                        const Narrow p = plan_narrow(rows, in, out, ragged, elem);
                        if (!p.blocks) continue;
                        looked++;
                        // the weight's fragments, the bias, each wave's outputs
                        const long tiles = elem == 4 ? up(out, 32) : up(out, 64) * 2;
                        const long lds = tiles * p.steps * 1024 + tiles * 128 + p.threads / 64 * unit_bytes(elem);
                        if (p.lds != lds || lds > kMostLds || p.steps * 32 < in * elem || p.blocks > 65535 || p.chunk < 32 || p.chunk % 32 ||
                            (ragged ? p.blocks * p.chunk < rows : (p.blocks - 1) * (p.threads / 2) >= rows))
                            std::printf("forward %ld rows, %d to %d, elem %d, ragged %d: lds %d threads %d\n", rows, in, out, elem, ragged, p.lds, p.threads);
                    }
}

void long_rows() {
    for (int in = 1; in <= 1200; in++)
        for (int out = 1; out <= 100; out++)
            for (const long rows : {1L, 4095L, 32767L, 32768L, 100'001L, 40'000'000L})
                for (const bool ragged : {false, true}) {
                    const Long p = plan_long(rows, in, out, ragged ? 3 : 1, ragged);
                    if (!p.blocks) continue;
                    looked++;
                    // the weight's fragments, the bias, each wave's lines and outputs
                    const long lds = p.tiles * (p.lines * 4096L + 128) + p.threads / 64 * unit_bytes(4);
                    if (p.lds != lds || lds > kMostLds || p.lines * 32 < in || (p.lines - 1) * 32 >= in || p.tiles * 32 < out || p.tiles > 2 || in < 4 ||
                        p.blocks > 65535 || p.chunk < 32 || p.chunk % 32 || (ragged ? p.blocks * p.chunk < rows : (p.blocks - 1) * (p.threads / 2) >= rows))
                        std::printf("long %ld rows, %d to %d, ragged %d: lds %d\n", rows, in, out, ragged, p.lds);
                }
}

void narrow_backward() {
    for (const int elem : {2, 4})
        for (int in = 1; in <= 300; in++)
            for (int out = 1; out <= 300; out++)
                for (const long rows : {0L, 1L, 32L, 33L, 4096L, 40'000'000L})
                    for (const int groups : {1, 7, 32768})
                        for (const bool curved : {false, true}) {
                            const NarrowBwd p = plan_narrow_bwd(rows, in, out, groups, curved, elem);
                            if (!p.blocks) continue;
                            looked++;
                            const int terms = p.fine ? 2 : 1;
                            if (p.lds > kMostLds || up(out, 32) * terms > p.zt || up(in, 32) > p.xt || p.blocks > 65535 || p.blocks * p.chunk < rows ||
                                (rows && (p.blocks - 1) * block_rows(elem) >= rows) || p.bytes != (p.blocks + groups) * (1L * in * out + out) * 4)
                                std::printf("backward %ld rows, %d to %d, elem %d, groups %d: lds %d\n", rows, in, out, elem, groups, p.lds);
                        }
}

// What a tile's loads add to their beginnings in 32 bits, of rows of any width that a layer may have.
void offsets() {
    for (const int elem : {2, 4})
        for (int width = 0; width <= 24; width++)
            for (const int less : {0, 1}) {
                const long in = (1L << width) - less, line = up(in, 16 / elem) * 16;
                if (in < 1) continue;
                const int depth = kTileDepthBytes / elem;
                looked++;
                if (line > kMostLine) std::printf("rows of %ld, elem %d: lines of %ld bytes, over %ld\n", in, elem, line, kMostLine);
                if (plain_offset(kLoadLines - 1, kMostLine, 7) >> 32 || across_offset(depth - 1, kMostLine, kMostLine - 16) >> 32)
                    std::printf("elem %d: offsets past 32 bits\n", elem);
            }
}

}  // namespace

int main() {
    offsets();
    narrow();
    long_rows();
    narrow_backward();
    std::printf("looked at %ld\n", looked);
}
