// Every address that the products' buffer loads of rows take, on the host, by the
// arithmetic of the kernels (ter_amd/csrc/int8_rows.h): a load is within the
// rows, or its vector offset, all that the hardware checks, is at or behind the size.
//
// int8_rows stream: rows by 16, 32 and 64 of a wave, units past the last among them.
// int8_rows tiles: rows by the tiles' 64 to 256, whole units of the last rows.
#include <cstdio>
#include <cstring>
#include <initializer_list>

#include "../../ter_amd/csrc/int8_rows.h"

using namespace terhip;

static long long bad = 0, outside = 0, inside = 0;

// 16 bytes at vector offset v of rows of `size` bytes.
static void load(unsigned v, long long size, unsigned checked, bool want, const char* what, int rows, int K, int u) {
    const bool in = (long long)v + 16 <= size, out = v >= checked;
    ++(out ? outside : inside);
    if ((in && !out) || (out && !want)) return;
    if (++bad < 10) printf("%s: rows %d K %d unit %d: offset %u of %lld (checked against %u)\n", what, rows, K, u, v, size, checked);
}

static void stream(int M, int K, int ldx) {
    const int units = (K + kI8Unit - 1) / kI8Unit;
    const long long size = (long long)(M - 1) * ldx + K;
    const unsigned checked = i8_rows_size(M, ldx, K);
    const int blocks = M <= 16 ? 1 : M <= 32 ? 2 : 4;
    // (16 waves and four units of each ahead: 63 units past the last at most)
    for (int u = 0; u < units + 64; ++u)
        for (int t = 0; t < 2; ++t)
            for (int m = 0; m < 16 * blocks; ++m)
                for (int g = 0; g < 4; ++g) {
                    const int k = u * kI8Unit + t * 64 + g * 16;
                    const unsigned v = i8_rows_at(i8_stream_lane(m, g, M, ldx), u, t);
                    load(v, size, checked, m < M && k < K, "stream", M, K, u);
                    if (m < M && k < K && v != (unsigned)(m * ldx + k)) ++bad;  // (its own 16 values)
                }
}

static void tiles(int M, int BM, int K, int ldx) {
    const int units = (K + kI8Unit - 1) / kI8Unit;
    for (int m0 = 0; m0 < M; m0 += BM) {
        const int rows = M - m0 < BM ? M - m0 : BM;
        const long long size = (long long)(rows - 1) * ldx + K;
        const unsigned checked = i8_rows_size(rows, ldx, K);
        for (int u = 0; u < units; ++u)
            for (int run = 0; run < BM / 8; ++run)
                for (int lane = 0; lane < 64; ++lane) {
                    // (the lane's place in LDS is chunk lane % 8 of the row)
                    const int row = run * 8 + lane / 8, chunk = (lane % 8) ^ i8_swizzle(row), k = u * kI8Unit + chunk * 16;
                    const unsigned v = i8_rows_at(i8_tile_lane(row, lane, ldx), u, 0);
                    load(v, size, checked, row < rows && k < K, "tiles", rows, K, u);
                    if (row < rows && k < K && v != (unsigned)(row * ldx + k)) ++bad;
                }
    }
}

int main(int argc, char** argv) {
    if (argc < 2) return 2;
    if (!strcmp(argv[1], "stream")) {
        for (int M : {1, 2, 15, 16, 17, 32, 33, 63, 64})
            for (int K = 16; K <= 9000; K += 16)
                for (int pad : {0, 16, 4096}) {
                    if (pad && M > 33 && K % 160) continue;
                    stream(M, K, K + pad);
                }
        for (int M : {1, 16, 64}) stream(M, 131056, 1 << 22);
    } else if (!strcmp(argv[1], "tiles")) {
        for (int BM : {64, 96, 128, 160, 192, 224, 256})
            for (int M : {17, 64, 65, 66, 97, 200, 256, 257})
                for (int K = 16; K <= 9000; K += K < 700 ? 16 : 1616 + 16)
                    for (int pad : {0, 16, 4096}) tiles(M, BM, K, K + pad);
        tiles(257, 256, 131056, 1 << 22);
    } else {
        return 2;
    }
    if (bad || !outside || !inside) {
        printf("%lld loads of %lld are wrong\n", bad, inside + outside);
        return 1;
    }
    puts("ok");
    return 0;
}
