// The check of a sequence's positions in front of every attention call (csrc/work_cut.h, rows_fit) against its definition in
// 64 bits, at the ends of the cache and of 32 bits; and that what the kernels form of positions it lets through -- the end of
// the rows, the tiles up to it, the end of the last tile -- stays in 32 bits for every width of a tile.
#include <cstdio>
#include <cstdlib>

#include "../../bruce-engine_b200/csrc/work_cut.h"

#define CHECK(c)                                                                   \
    do {                                                                           \
        if (!(c)) {                                                                \
            std::printf("FAILED %s:%d: %s (p0 %lld rows %d ring %d cap %lld)\n", __FILE__, __LINE__, #c, p0, rows, ring, cap); \
            std::exit(1);                                                          \
        }                                                                          \
    } while (0)

int main() {
    const long long MAX = 0x7fffffffLL, END = MAX - battn::POS_ROOM;
    const long long caps[] = {2, 128, 512, 634, 32768, 262144, MAX - 511, MAX - 257, MAX - 256, MAX - 127, MAX};
    for (int ring = 0; ring < 2; ++ring)
        for (long long cap : caps)
            for (int rows = 1; rows <= 512; ++rows) {
                const long long base[] = {-MAX - 1, -1, 0, cap - rows, cap, END - rows, MAX - rows, MAX};
                for (long long b : base)
                    for (long long p0 = b - 3; p0 <= b + 3; ++p0) {
                        if (p0 < -MAX - 1 || p0 > MAX) continue;
                        const bool fits = battn::rows_fit((int)p0, rows, ring != 0, (int)cap);
                        const long long end = p0 + rows;
                        CHECK(fits == (p0 >= 0 && end <= END && (ring || end <= cap)));
                        if (!fits) continue;
                        for (int tile = 64; tile <= 256; tile *= 2)
                            CHECK(end >= 1 && end + tile - 1 <= MAX && ((end - 1) / tile + 1) * tile <= MAX);
                    }
            }
    std::puts("OK");
    return 0;
}
