// How a block of the one-token kernels (delta_step.cu) is laid out. Plain C++, so that every shape's offsets can be
// checked on the host.
#pragma once

#ifdef __CUDACC__
#define GB_HOST_DEVICE __host__ __device__
#else
#define GB_HOST_DEVICE
#endif

namespace gb {

// Threads of a block: x over the columns in fours, y over groups of `rows` rows, z over heads. Blocks of about 128
// threads: 256 is 2 to 20 % slower at 64 x 64.
struct StepShape {
    int x, y, z;
    GB_HOST_DEVICE constexpr StepShape(int K, int V, int rows) : x((V + 3) / 4), y((K + rows - 1) / rows), z(128 / (x * y)) {
        z = z < 1 ? 1 : z > 64 ? 64 : z;
    }
};

// A block's shared memory, in floats from a 16-byte boundary: the row groups' sums [z][y][2][cols] (with k, with q), which
// are read and written 16 bytes at a time and so come first (z K may be odd); k and q as pairs [z][K]; k.q [z][y]. cols: 4 x.
struct StepShared {
    int sums, pairs, dots, end;
    GB_HOST_DEVICE constexpr StepShared(int K, int cols, int y, int z)
        : sums(0), pairs(z * y * 2 * cols), dots(2 * z * (K + y * cols)), end(dots + z * y) {}
};

}  // namespace gb
