// Which kernel takes an 8-bit product and how it is cut. Host arithmetic alone,
// without a CUDA header.
#pragma once

namespace dz {

constexpr int Q8_PARTS = 8;        // blocks that split k at most

struct Q8Plan {
    int rows;    // of a tile: 8 or 16 in registers (q8matmul.cu), 32, 64 or 128 of a block, 256 of a pair (q8gemm.cu)
    int parts;   // blocks that share a tile's k
    double time; // estimated, in microseconds
};

// The kernel and the cut of the least estimated time. What the estimates take
// from measurements (one B200, device time, kernels in a row):
// - registers: 1.5 us, then the levels once for every 8 rows at 7.5 MB a
//   microsecond, or for every 16 at 5.6 where their activations fit shared memory
//   (2 x 2048 x 2048: 2.3 us, 1 x 4096 x 16384: 9.8, 16 x 4096 x 5120: 7.7);
// - blocks: 2.9, 3.6 or 6.8 us for 32, 64 or 128 rows each time the SMs are full
//   of them, two to an SM, 0.21 us for each step of 128 of k, alone on its SM or
//   0.33 (0.44) where two share one, 1 us and 0.1 for each part to join parts (32 x
//   2048 x 2048: 7.5 us whole, 5.0 in four parts; 32 x 4096 x 5120: 6.9 in four, 11.4
//   in eight, which are more blocks than there are places; 128 x 4096 x 16384: 14.7
//   with 64 rows, 15.0 with 128, 25.6 with 32);
// - pairs of SMs: 6 us, 0.28 us a step while few are at work and 0.335 when all
//   are (256 x 4096 x 16384: 17.6 us, 20.2 in blocks; 256 x 4096 x 5120: 15.9,
//   13.0 in blocks of 64 rows);
// - levels that L2 does not hold come at 6.3 MB a microsecond (1 x 4096 x 32000:
//   22.6 us in blocks, 24.0 in registers, whose loads wait longer).
inline Q8Plan q8_plan(long long m, long long k, long long n, long long sms, long long staging) {
    Q8Plan best{0, 1, 1e30};
    const double levels = (double)k * (double)n;
    const bool far = levels > 100e6;
    auto consider = [&](int rows, int parts, double time) {
        if (time < best.time) best = Q8Plan{rows, parts, time};
    };
    const long long steps = (k + 127) / 128;
    auto least = [&](double time, double rate) { return far && time < 1.8 + levels / rate ? 1.8 + levels / rate : time; };
    if (m <= 16) {
        const bool two = m > 8 && m * (steps * 128 + 64) <= staging;             // both groups of 8 rows at once
        consider(two ? 16 : 8, 1, least(1.5 + 0.03 * m + (two ? levels / 5.6e6 : (m > 8 ? 2 : 1) * levels / 7.5e6), 5.9e6));
    }
    const long long tiles = (n + 127) / 128;
    for (int rows = 32; rows <= 128; rows *= 2) {
        const double start = rows == 32 ? 2.9 : rows == 64 ? 3.6 : 6.8, shared = rows == 128 ? 0.44 : 0.33;
        for (int parts = 1; parts <= Q8_PARTS && (parts == 1 || 2 * parts <= steps); parts *= 2) {
            const long long blocks = tiles * ((m + rows - 1) / rows) * parts, full = blocks / (2 * sms), rest = blocks % (2 * sms);
            const double each = (double)((steps + parts - 1) / parts);
            const double few = 0.6 + 0.4 * (double)(rest - sms) / (double)sms;       // not all of the SMs have two
            const double step = full * shared + (rest == 0 ? 0.0 : rest <= sms ? 0.21 : 0.21 + (shared - 0.21) * few);
            const double starts = start * (double)(full + (rest ? 1 : 0));
            consider(rows, parts, least(starts + each * step + (parts > 1 ? 1.0 + 0.1 * parts : 0.0), 6.3e6));
        }
    }
    const long long pairs = ((n + 255) / 256) * ((m + 255) / 256), rounds = (pairs + sms / 2 - 1) / (sms / 2);
    consider(256, 1, least(6.0 + (double)rounds * steps * (4 * pairs <= sms ? 0.28 : 0.335), 6.3e6));
    return best;
}

}  // namespace dz
