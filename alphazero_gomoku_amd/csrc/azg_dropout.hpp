// Dropout from a counter-based generator: y = [r +] keep(i) ? s x : 0, s = 65536 / (65536 - T), T = round(65536 p).
//
// keep(i) = (16 bits of element i) >= T.  The bits come from Philox4x32-10 (Salmon, Moraes, Dror, Shaw,
// "Parallel random numbers: as easy as 1, 2, 3", 2011): counter = (element number div 8, call number), key =
// seed; the four output words hold the eight elements' half-words, low half first.  The mask is therefore a
// function of (seed, call, element number) and is never stored: the backward pass is the same map on the
// gradient.  p is quantised to 1/65536 and s is the exact reciprocal of the quantised keep rate, so the
// expectation is x whatever p.  Sixteen bits an element (not 32) because the multiplies bound the narrow types.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace azgops {

struct DropoutArgs {
    const void *x, *res;             // [rows][cols], row strides below (elements); res may be null
    void *out;
    long long rows, cols, xs, rs, os;
    unsigned long long first, step;  // element number of (row, col) = first + row * step + col, modulo 2^64
    unsigned long long seed, offset;
    const long long *offset_dev;     // null, or added to offset when the kernel runs
    unsigned threshold;
    float scale;
};

__device__ inline void philox4x32_10(uint32_t (&c)[4], uint32_t k0, uint32_t k1)
{
#pragma unroll
    for (int r = 0; r < 10; r++) {
        const uint64_t a = (uint64_t)c[0] * 0xD2511F53u, b = (uint64_t)c[2] * 0xCD9E8D57u;
        const uint32_t n0 = (uint32_t)(b >> 32) ^ c[1] ^ k0, n2 = (uint32_t)(a >> 32) ^ c[3] ^ k1;
        c[0] = n0; c[1] = (uint32_t)b; c[2] = n2; c[3] = (uint32_t)a;
        k0 += 0x9E3779B9u; k1 += 0xBB67AE85u;
    }
}

// eight elements of any alignment: the hardware takes unaligned global accesses
template <typename T> struct __attribute__((packed)) Eight { T v[8]; };

// One thread per block of eight element numbers and row, so that one counter serves eight elements in one 16- or 32-byte
// access; blocks cut by the ends of a row go element by element.  Bound by memory: [16384, 4096] bfloat16 with a residual moves
// 403 MB in 67 us, 6.0 TB/s (a plain copy reaches 5.2 TB/s, half of it writes); [4099, 1111] half precision, whose rows start
// inside blocks, 18 MB in 6.4 us; the heads of a mini-batch ([512, 900] float32) 3 us, a launch.
template <typename T>
__global__ __launch_bounds__(256) void dropout_kernel(DropoutArgs a, long long blocks_per_row)
{
    unsigned long long off = a.offset;
    if (a.offset_dev) off += (unsigned long long)*a.offset_dev;
    const long long total = a.rows * blocks_per_row;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long long)gridDim.x * 256) {
        const long long row = a.rows == 1 ? 0 : i / blocks_per_row, j = i - row * blocks_per_row;
        const unsigned long long e0 = a.first + (unsigned long long)row * a.step;
        const unsigned long long blk = ((e0 >> 3) + (unsigned long long)j) & ((1ull << 61) - 1);   // (numbers are modulo 2^64)
        const long long col0 = (long long)(blk * 8 - e0);                   // column of the block's first element: -7 .. cols
        if (col0 >= a.cols) continue;
        uint32_t c[4] = {(uint32_t)blk, (uint32_t)(blk >> 32), (uint32_t)off, (uint32_t)(off >> 32)};
        philox4x32_10(c, (uint32_t)a.seed, (uint32_t)(a.seed >> 32));
        const T *x = static_cast<const T *>(a.x) + row * a.xs + col0;
        const T *r = a.res ? static_cast<const T *>(a.res) + row * a.rs + col0 : nullptr;
        T *o = static_cast<T *>(a.out) + row * a.os + col0;
        if (col0 >= 0 && col0 + 8 <= a.cols) {
            const Eight<T> xv = *reinterpret_cast<const Eight<T> *>(x);
            Eight<T> y;
            float f[8];
#pragma unroll
            for (int q = 0; q < 8; q++) {
                const uint32_t u = (q & 1) ? c[q >> 1] >> 16 : c[q >> 1] & 0xFFFFu;
                f[q] = u >= a.threshold ? (float)xv.v[q] * a.scale : 0.f;
            }
            if (r) {
                const Eight<T> rv = *reinterpret_cast<const Eight<T> *>(r);
#pragma unroll
                for (int q = 0; q < 8; q++) f[q] = (float)rv.v[q] + f[q];
            }
#pragma unroll
            for (int q = 0; q < 8; q++) y.v[q] = (T)f[q];
            *reinterpret_cast<Eight<T> *>(o) = y;
        } else {
#pragma unroll
            for (int q = 0; q < 8; q++) {
                if (col0 + q < 0 || col0 + q >= a.cols) continue;
                const uint32_t u = (q & 1) ? c[q >> 1] >> 16 : c[q >> 1] & 0xFFFFu;
                float f = u >= a.threshold ? (float)x[q] * a.scale : 0.f;
                if (r) f = (float)r[q] + f;
                o[q] = (T)f;
            }
        }
    }
}

}  // namespace azgops
