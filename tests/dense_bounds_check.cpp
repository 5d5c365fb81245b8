// Walks every operand request of the dense linear's tiles on the host: what the range check lets through lies inside the operand, and the
// pieces of rows and columns that exist are let through.  Built and run by test_dense_bounds.py.
#include <cstdio>
#include <cstdlib>
#include <initializer_list>

#include "../primus_amd/csrc/mx_gemm_addr.h"

using namespace mxl::addr;
static long checked = 0;

static void request(const Desc& d, uint32_t voff, uint32_t soff, int64_t bytes, bool exists) {
    for (int c = 0; c < 4; ++c) {
        ++checked;
        const bool in = accepted(d, voff, soff, c);
        const int64_t a = d.base + (int64_t)voff + (int64_t)soff + 4 * c;
        if ((in && (a < 0 || a + 4 > bytes)) || (exists && !in)) {
            std::printf("bad request: offset %lld of %lld, exists %d\n", (long long)a, (long long)bytes, (int)exists);
            std::exit(1);
        }
    }
}

static void rows(int tile, int threads, int64_t total, int64_t k, int64_t row0) {
    const int64_t ld = k * 2, slots = (k + 63) / 64;
    const Desc d = tall_rows_desc(total, row0, ld);
    for (int64_t s = 0; s < slots + 3; ++s)
        for (int e = 0; e < tile * 128 / (threads * 16); ++e)
            for (int t = 0; t < threads; ++t) {
                const int row = (t >> 3) + threads / 8 * e, piece = (t & 7) ^ ((row >> 1) & 7);
                const bool live = s < slots;
                request(d, dense_rows_lane(t, e, threads, ld), live ? (uint32_t)(s * 128) : kDropped, total * ld, live && row0 + row < total && s * 128 + piece * 16 < ld);
            }
}

static void cols(int tile, int threads, int64_t k, int64_t n, int64_t col0) {
    const int64_t ld = n * 2, slots = (k + 63) / 64;
    const Desc d = tall_cols_desc(0, k, ld, col0 * 2);
    const int pieces = tile / 8;
    for (int64_t s = 0; s < slots + 3; ++s)
        for (int e = 0; e < tile * 128 / (threads * 16); ++e)
            for (int t = 0; t < threads; ++t) {
                const int row = t / pieces + threads / pieces * e, piece = (t % pieces) ^ ((row & 3) << (tile >= 128 ? 2 : 1));
                const bool live = s < slots;
                if (piece < 0 || piece >= pieces || row >= 64) std::exit(2);
                request(d, dense_cols_lane(t, e, threads, tile, ld), live ? (uint32_t)(s * 64 * ld) : kDropped, k * ld, live && s * 64 + row < k && col0 + piece * 8 < n);
            }
}

int main() {
    for (int64_t m : std::initializer_list<int64_t>{1, 17, 63, 64, 65, 255, 256, 300, 513})
        for (int64_t k : std::initializer_list<int64_t>{32, 64, 96, 160, 352}) {
            for (int64_t r = 0; r < m; r += 64) rows(64, 256, m, k, r);
            for (int64_t r = 0; r < m; r += 256) rows(256, 512, m, k, r);
            for (int64_t r = 0; r < m; r += 128) rows(128, 512, m, k, r);
        }
    for (int64_t n : std::initializer_list<int64_t>{32, 64, 96, 160, 352})
        for (int64_t k : std::initializer_list<int64_t>{32, 64, 96, 224}) {
            for (int64_t c = 0; c < n; c += 64) cols(64, 256, k, n, c);
            for (int64_t c = 0; c < n; c += 128) cols(128, 512, k, n, c);
        }
    // the weight gradient: contraction rows in any number, 256 columns of the first operand
    for (int64_t n : std::initializer_list<int64_t>{32, 96, 256, 288, 544})
        for (int64_t k : std::initializer_list<int64_t>{1, 17, 63, 64, 65, 130}) {
            for (int64_t c = 0; c < n; c += 64) cols(64, 256, k, n, c);
            for (int64_t c = 0; c < n; c += 128) cols(128, 512, k, n, c);
            for (int64_t c = 0; c < n; c += 256) cols(256, 512, k, n, c);
        }
    // the largest operands: one row, and a tile's last rows, of 2^21 elements; a matrix of almost 4 GiB
    rows(256, 512, 256, 1 << 21, 0);
    const int64_t n = 1 << 15, k = (1 << 16) - 32;
    for (int t = 0; t < 512; ++t)
        for (int e = 0; e < 2; ++e) {
            const Desc d = tall_cols_desc(0, k, n * 2, (n - 128) * 2);
            request(d, dense_cols_lane(t, e, 512, 128, n * 2), (uint32_t)((k / 64) * 64 * n * 2), k * n * 2, false);
            request(d, dense_cols_lane(t, e, 512, 128, n * 2), kDropped, k * n * 2, false);
        }
    std::printf("%ld requests inside their operands\n", checked);
    return 0;
}
