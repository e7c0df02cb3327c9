// otf_rng.h — the counter-based generator behind dropout (gfx950).
//
// Philox4x32-10 (J. Salmon, M. Moraes, R. Dror, D. Shaw, "Parallel random numbers: as easy
// as 1, 2, 3", SC 2011): ten rounds of two 32 x 32 -> 64 products over a 128-bit counter
// under a 64-bit key.  The counter of eight consecutive columns of a row is
// (row * ceil(cols / 8) + col / 8, offset) and the key is the seed, so a mask depends on the
// element's place alone: forward and backward, any launch shape and any vector width make
// the same one, and it is never stored.
#pragma once
#include "otf_device.h"

namespace otf {

struct DropKey {
    uint32_t k0, k1, o0, o1;
};

// rng: two int64, seed and offset (wave-uniform loads); null where nothing is dropped
__device__ __forceinline__ DropKey drop_key(const int64_t* rng) {
    if (!rng) return DropKey{};
    const uint64_t seed = (uint64_t)rng[0], off = (uint64_t)rng[1];
    return DropKey{(uint32_t)seed, (uint32_t)(seed >> 32), (uint32_t)off, (uint32_t)(off >> 32)};
}

__device__ __forceinline__ void philox4x32_10(uint64_t index, const DropKey& key, uint32_t (&out)[4]) {
    uint32_t c0 = (uint32_t)index, c1 = (uint32_t)(index >> 32), c2 = key.o0, c3 = key.o1;
    uint32_t k0 = key.k0, k1 = key.k1;
#pragma unroll
    for (int r = 0; r < 10; ++r) {
        const uint64_t p0 = (uint64_t)c0 * 0xD2511F53u, p1 = (uint64_t)c2 * 0xCD9E8D57u;
        c0 = (uint32_t)(p1 >> 32) ^ c1 ^ k0;
        c2 = (uint32_t)(p0 >> 32) ^ c3 ^ k1;
        c1 = (uint32_t)p1;
        c3 = (uint32_t)p0;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    out[0] = c0, out[1] = c1, out[2] = c2, out[3] = c3;
}

// Bit j: column j of eight is kept, its 16-bit field reaching `threshold`.  16 bits an element
// halve the generator's work against a 32-bit word each; the probability is the multiple of 2^-16
// nearest to the asked one, and the scale is that multiple's, so the expectation is exact.
// A threshold of 0 (uniform) keeps all without the generator.
__device__ __forceinline__ uint32_t keep8(uint64_t index, const DropKey& key, uint32_t threshold) {
    if (threshold == 0) return 0xffu;
    uint32_t w[4], m = 0;
    philox4x32_10(index, key, w);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const uint32_t field = (j & 1) ? w[j >> 1] >> 16 : w[j >> 1] & 0xffffu;
        m |= field >= threshold ? 1u << j : 0u;
    }
    return m;
}
// kept columns scaled, the others an exact 0 (a select: what is dropped may be inf or NaN)
__device__ __forceinline__ void drop8(float (&v)[8], uint32_t kept, float scale) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = (kept >> j) & 1 ? v[j] * scale : 0.0f;
}

// host: probability -> threshold (of 65536) and scale; p < 1 always keeps something
inline bool drop_params(double p, uint32_t& threshold, float& scale) {
    if (!(p >= 0.0 && p <= 1.0)) return false;
    double t = p >= 1.0 ? 65536.0 : (double)(int64_t)(p * 65536.0 + 0.5);
    if (p < 1.0 && t > 65535.0) t = 65535.0;
    threshold = (uint32_t)t;
    scale = t >= 65536.0 ? 0.0f : (float)(65536.0 / (65536.0 - t));
    return true;
}

// ---- launches ---------------------------------------------------------------------------
// Workgroups, more than 2^20 of them in rows of 2^20: HIP counts a dimension's threads in 32 bits,
// and launches what is left of a larger count without an error.
__device__ __forceinline__ int64_t block_id() { return (int64_t)blockIdx.y * gridDim.x + blockIdx.x; }
inline dim3 blocks(int64_t n) { return n <= 1 << 20 ? dim3((unsigned)n) : dim3(1u << 20, (unsigned)((n + (1 << 20) - 1) >> 20)); }

// ---- eight consecutive elements of a row, in float ------------------------------------
// Rows may start at any element: the vector is aligned to its element only (global memory
// takes unaligned 16-byte accesses on this target), so odd widths and strides keep wide
// loads; only the last chunk of a row goes element by element.
template <typename T> struct Chunk8 {
    using type = T __attribute__((ext_vector_type(8), aligned(sizeof(T))));
};

// as stored, zeros past `valid`
template <typename T> __device__ __forceinline__ typename Chunk8<T>::type load8_raw(const T* p, int valid) {
    typename Chunk8<T>::type q{};
    if (valid >= 8) {
        q = *reinterpret_cast<const typename Chunk8<T>::type*>(p);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j < valid) q[j] = p[j];
    }
    return q;
}

template <typename T>
__device__ __forceinline__ void load8(const T* p, int valid, float (&v)[8]) {
    if (valid >= 8) {
        const typename Chunk8<T>::type q = *reinterpret_cast<const typename Chunk8<T>::type*>(p);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = (float)q[j];
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = j < valid ? (float)p[j] : 0.0f;
    }
}

template <typename T>
__device__ __forceinline__ void store8(T* p, int valid, const float (&v)[8]) {
    if (valid >= 8) {
        typename Chunk8<T>::type q;
#pragma unroll
        for (int j = 0; j < 8; ++j) q[j] = (T)v[j];
        *reinterpret_cast<typename Chunk8<T>::type*>(p) = q;
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j < valid) p[j] = (T)v[j];
    }
}

}  // namespace otf
