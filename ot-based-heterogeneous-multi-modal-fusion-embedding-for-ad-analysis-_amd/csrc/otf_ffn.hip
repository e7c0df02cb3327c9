// otf_ffn.hip — the gated feed-forward block, forward and backward, on the matrix cores.
//
//   forward    h = act(x Wg^T) * (x Wu^T)        one kernel: both products share x, gate and up
//              y = h Wd^T                        of a feature meet in one lane's registers
//   backward   dh = dy Wd;  dg = dh u act'(g), du = dh act(g)    epilogue of the dh product
//              dx = dg Wg + du Wu                one product over 2 f, two segments of K
//              dWg = dg^T x, dWu = du^T x, dWd = dy^T h
//
// Every product is C[m, n] = sum_k A(m, k) B(n, k) with each operand either K-contiguous
// (layout K: rows are m or n) or row-contiguous (layout T: rows are k).  Both go global -> LDS
// by 16-byte buffer loads that write LDS directly; what lies past an operand's end comes back
// as zero from the buffer descriptor's range check, so ragged edges cost no branch.  Layout T
// is transposed on the way from LDS to registers (ds_read_b64_tr_b16).
//
// All sums are float32 in the accumulators.  h, dg and du are rounded to the operands' type, which
// the products that read them need (up to 8 rows with their low parts beside them); g and u are kept in float32 for the backward pass, where their
// rounding would meet dg's and du's own (gradients of 16-bit operands then err by 1.4 times their
// final rounding instead of 1.8; at 8192 x 4096 x 11264 the wider buffers cost 2 % of a step).
#include "otf_rng.h"

namespace otf {
namespace {

typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
typedef __attribute__((ext_vector_type(8))) __bf16 b16x8;
typedef __attribute__((ext_vector_type(4))) short s16x4;
typedef __attribute__((address_space(3))) char lds_char;

[[maybe_unused]] constexpr int kRsrcFlags = 0x00020000;   // raw buffer of 32-bit data
constexpr int kTileBytes = 128;          // depth of a K-tile: 64 16-bit or 32 float32 values

// ---- one 16 x 16 block over 64 bytes of K ---------------------------------------------
// A fragment is 16 bytes a lane: row lane % 16, K chunk lane / 16.  For float32 the four
// values feed four 16x16x4 steps; both operands name the same k for a lane and step, which is
// all the sum needs.
template <typename T> struct Frag;
template <> struct Frag<_Float16> {
    using type = f16x8;
    static __device__ __forceinline__ f32x4 mma(type a, type b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    }
};
template <> struct Frag<__bf16> {
    using type = b16x8;
    static __device__ __forceinline__ f32x4 mma(type a, type b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    }
};
template <> struct Frag<float> {
    using type = f32x4;
    static __device__ __forceinline__ f32x4 mma(type a, type b, f32x4 c) {
#pragma unroll
        for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], b[j], c, 0, 0, 0);
        return c;
    }
};

// ---- activations ------------------------------------------------------------------------
enum { kSilu = 0, kGelu = 1 };
// one exponential and one reciprocal instruction, each within an ulp or two of float32
__device__ __forceinline__ float sigmoid(float g) {
    return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.44269504088896341f * g));
}
// The normal distribution function c(g) and e = exp(-g^2 / 2).  float32 operands: erfc.  16-bit ones:
// erfc(x) = t Q(t) exp(-x^2), t = 1 / (1 + 0.46 x), with Q the polynomial of degree 7 of the least
// relative error to exp(x^2) erfc(x) / t on 0 < t <= 1 (fitted by weighted least squares; 6.8e-7), so that the tail
// of act(g) keeps its digits: with the exponential's argument 2e-6 of the value at g = -5, 2e-5 at -13.  It
// shares the exponential with the derivative (erfc took 6 us of the 34 of a gate and up product at
// 777 x 1000 x 2730).
template <typename T> __device__ __forceinline__ void normal_cdf(float g, float& c, float& e) {
    const float x = 0.70710678118654752f * fabsf(g);
    e = __builtin_amdgcn_exp2f(-1.44269504088896341f * x * x);
    float q;
    if constexpr (sizeof(T) == 4) {
        q = erfcf(x);
    } else {
        const float t = __builtin_amdgcn_rcpf(1.0f + 0.46f * x);
        q = 0.16919090f + t * (-0.22662924f + t * 0.067714341f);
        q = 0.23118190f + t * (0.18684773f + t * (0.052610725f + t * q));
        q = t * (0.25952706f + t * (0.25955728f + t * q)) * e;
    }
    c = g < 0.0f ? 0.5f * q : 1.0f - 0.5f * q;
}
template <typename T> __device__ __forceinline__ float act_value(int act, float g) {
    if (act == kSilu) return g * sigmoid(g);
    float c, e;
    normal_cdf<T>(g, c, e);
    return g * c;
}
template <typename T> __device__ __forceinline__ void act_both(int act, float g, float& a, float& da) {
    if (act == kSilu) {
        const float s = sigmoid(g);
        a = g * s;
        da = s * (1.0f + g * (1.0f - s));
    } else {
        float c, e;
        normal_cdf<T>(g, c, e);
        a = g * c;
        da = c + g * 0.39894228040143268f * e;
    }
}

// ---- operands -----------------------------------------------------------------------------
// One tile of R rows (m or n) by a K-tile, R * 128 bytes of LDS.
//   layout K: two halves of 64 bytes of K, each [R][64 B], the four 16-byte chunks of a row
//             permuted by the row, so 16 rows' fragments of one chunk fall on different banks
//   layout T: [k][R values], the 16-byte chunks of a row permuted by k so that the rows that
//             one LDS read spans fall on different banks
struct Operand {
    const char* p[2];   // second segment of K, or the second half of the tile (gated)
    int64_t ld;         // bytes
    int mn;             // valid rows (K) / columns (T)
    int k;              // valid k
};

__device__ __forceinline__ int swz_k(int row) { return (0x78 >> (2 * ((row >> 2) & 3))) & 3; }
template <typename T, int R> __device__ __forceinline__ int swz_t(int k) {
    if constexpr (sizeof(T) == 2) {
        if constexpr (R >= 128) return 2 * ((k & 3) | (((k >> 3) & 1) << 2));
        if constexpr (R == 64) return 2 * (((k >> 1) & 1) | (((k >> 3) & 1) << 1));
        if constexpr (R == 32) return 2 * ((k >> 3) & 1);
        return 0;
    } else {
        if constexpr (R >= 64) return 4 * ((k >> 2) & 3);
        if constexpr (R == 32) return 4 * ((k >> 2) & 1);
        return 0;
    }
}

template <typename T, bool TR, int R, int NT> struct Tile {
    static constexpr int BYTES = R * kTileBytes, CHUNKS = BYTES / 16, PER = CHUNKS / NT;
    static_assert(CHUNKS % NT == 0, "every wave issues the same loads");
    static constexpr int BK = kTileBytes / (int)sizeof(T);
    static constexpr int CPR = R * (int)sizeof(T) / 16;   // layout T: chunks of a k row
    uint32_t off[PER];
    int kb[PER];   // layout K: byte of K of the lane's chunk

    __device__ __forceinline__ void init(int64_t ld) {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int c = i * NT + (int)threadIdx.x;
            if constexpr (TR) {
                const int k = c / CPR, chunk = (c % CPR) ^ swz_t<T, R>(k);
                off[i] = (uint32_t)(k * ld) + chunk * 16;
                kb[i] = 0;
            } else {
                const int half = c / (R * 4), row = (c % (R * 4)) >> 2, chunk = (c & 3) ^ swz_k(row);
                kb[i] = half * 64 + chunk * 16;
                off[i] = (uint32_t)(row * ld) + kb[i];
            }
        }
    }
    // A K-tile into LDS at `dst`: `bytes` from `base` on are readable and a lane past them gets
    // zeros.  MASK: so does one past the first `left` bytes of K (layout K, whose rows are followed
    // by the next ones).
    template <bool MASK> __device__ __forceinline__ void put(const char* base, uint32_t bytes, int left, char* dst) const {
#ifdef __HIP_DEVICE_COMPILE__   // the buffer builtins: the host pass drops the launch stubs of kernels that reach them
        const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        const auto r = __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, (int)bytes, kRsrcFlags);
#pragma unroll
        for (int i = 0; i < PER; ++i)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(
                r, (__attribute__((address_space(3))) void*)(dst + (i * NT + wave * 64) * 16), 16,
                MASK && kb[i] >= left ? 0xfffffff0u : off[i], 0, 0, 0);
#endif
    }
    // fragment of the 16 rows from r0, K half s
    static __device__ __forceinline__ typename Frag<T>::type frag(const char* tile, int r0, int s, int lane) {
        if constexpr (!TR) {
            const int row = r0 + (lane & 15);
            return *reinterpret_cast<const typename Frag<T>::type*>(tile + s * (R * 64) + row * 64 +
                                                                    (((lane >> 4) ^ swz_k(row)) << 4));
        } else {
            static_assert(sizeof(T) == 4, "16-bit: read_tr");
            typename Frag<T>::type f;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int k = s * 16 + (lane >> 4) * 4 + j, c = r0 + (lane & 15);
                f[j] = *reinterpret_cast<const float*>(tile + k * (R * 4) + (((c >> 2) ^ swz_t<T, R>(k)) << 4) + (c & 3) * 4);
            }
            return f;
        }
    }
};

// ---- results ------------------------------------------------------------------------------
enum { kStore = 0, kGatedForward = 1, kGatedBackward = 2 };
struct GemmArgs {
    Operand a, b;
    int M, N;            // extent of the result; gated forward: N = features
    int segments;        // of K (each a.k deep)
    int splits;          // of the K-tiles, kStore: with more than one, c[0] is a float32 slab of C each
    int tiles_m, tiles_n;
    void* c[2];          // result; second: the rows past tiles of the first (batch), see batch
    int64_t ldc;         // elements
    int batch;           // 2: a.p[1] -> c[1] as a second product of the same shape
    int act;
    float* g;            // gated: saved gate and up products (backward: in; forward: out or null)
    float* u;
    int features;        // gated: valid columns; zeros are written past them up to N
    void* h;             // gated forward: h; backward: dg
    void* h2;            // gated backward: du
    int64_t ldh;         // elements, of g, u, h, h2
    int low;             // 16-row tiles: A's rows (kStore) or the hidden results' from here on are
                         // low parts; 0: none
};

template <typename T>
__device__ __forceinline__ void store4(T* p, int valid, bool vec, f32x4 v) {
    if (vec && valid >= 4) {
        using V = T __attribute__((ext_vector_type(4)));
        V q;
#pragma unroll
        for (int j = 0; j < 4; ++j) q[j] = (T)v[j];
        *reinterpret_cast<V*>(p) = q;
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (j < valid) p[j] = (T)v[j];
    }
}
template <typename T> __device__ __forceinline__ f32x4 load4(const T* p) {
    using V = T __attribute__((ext_vector_type(4)));
    const V q = *reinterpret_cast<const V*>(p);
    return f32x4{(float)q[0], (float)q[1], (float)q[2], (float)q[3]};
}

__device__ __forceinline__ bool finite(float v) { return fabsf(v) < __builtin_inff(); }
// A hidden value in 32 bits but for the last: the value's rounding to T, and `low` elements on what
// that left out (nothing of an overflow).  low = 0: the rounding alone.
template <typename T> __device__ __forceinline__ void store_hidden(T* p, int64_t low, f32x4 v) {
    store4(p, 4, true, v);
    if constexpr (sizeof(T) == 2) {
        if (low) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float high = (float)(T)v[j];
                v[j] = finite(high) ? v[j] - high : 0.0f;
            }
            store4(p + low, 4, true, v);
        }
    }
}

// four consecutive columns n.. of row m: acc0 of the tile's first half, acc1 of its second
// (at n2; gated forward: the up product of the same columns)
template <typename T, int EPI>
__device__ __forceinline__ void finish4(const GemmArgs& a, int z, int split, int m, int n, int n2, f32x4 acc0, f32x4 acc1) {
    if (m >= a.M) return;
    if constexpr (EPI == kStore) {
        if (a.splits > 1) {   // ldc: a multiple of 4 past N
            float* c = (float*)a.c[0] + (((int64_t)split * a.batch + z) * a.M + m) * a.ldc;
            if (n < a.N) *reinterpret_cast<f32x4*>(c + n) = acc0;
            if (n2 < a.N) *reinterpret_cast<f32x4*>(c + n2) = acc1;
            return;
        }
        T* c = (T*)a.c[z] + (int64_t)m * a.ldc;
        const bool vec = (a.ldc & 3) == 0 && ((uintptr_t)a.c[z] & (4 * sizeof(T) - 1)) == 0;
        store4(c + n, a.N - n, vec, acc0);
        store4(c + n2, a.N - n2, vec, acc1);
    } else if constexpr (EPI == kGatedForward) {
        if (n >= a.N) return;   // N, ldh whole K-tiles
        const int64_t o = (int64_t)m * a.ldh + n;
        f32x4 h;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (n + j >= a.features) acc0[j] = acc1[j] = 0.0f;
            h[j] = act_value<T>(a.act, acc0[j]) * acc1[j];
        }
        store_hidden((T*)a.h + o, a.low * a.ldh, h);
        if (a.g) {
            store4(a.g + o, 4, true, acc0);
            store4(a.u + o, 4, true, acc1);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int nn = i ? n2 : n;
            if (nn >= a.N) continue;
            const int64_t o = (int64_t)m * a.ldh + nn;
            const f32x4 g = load4(a.g + o), u = load4(a.u + o), dh = i ? acc1 : acc0;
            f32x4 dg, du;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float v, dv;
                act_both<T>(a.act, g[j], v, dv);
                dg[j] = nn + j < a.features ? dh[j] * u[j] * dv : 0.0f;
                du[j] = nn + j < a.features ? dh[j] * v : 0.0f;
            }
            store_hidden((T*)a.h + o, a.low * a.ldh, dg);
            store_hidden((T*)a.h2 + o, a.low * a.ldh, du);
        }
    }
}

// Workgroup -> tile.  Consecutive ids go to the 8 XCDs in turn; each XCD gets a run of
// consecutive tiles, walked in groups of 8 row tiles, so its L2 holds the operands they share.
__device__ __forceinline__ void tile_of(int id, int count, int tiles_m, int tiles_n, int& tm, int& tn) {
    const int q = count / 8, r = count % 8, x = id % 8;
    const int t = (x < r ? x * (q + 1) : r * (q + 1) + (x - r) * q) + id / 8;
    const int per = 8 * tiles_n, g = t / per, first = g * 8, rows = min(tiles_m - first, 8), in = t - g * per;
    tm = first + in % rows;
    tn = in / rows;
}

// A tile's place in its operand, moved on by a K-tile with each load, so that a load costs a few
// scalar instructions.  Readable bytes: layout K, the valid rows whole (the K-tile may start anywhere
// in them; a row past them starts past that range); layout T, the K-tile's rows, fewer in a
// segment's last one.  Past the end of K nothing is readable: a load brings zeros.
template <typename T, bool TR, int R> struct Cursor {
    static constexpr int BK = kTileBytes / (int)sizeof(T);
    const char *p, *second;
    int64_t step;
    uint32_t bytes, bytes_last;
    int nk, total, kbytes, left;
    // K-tiles from k0 on of `segments` runs of nk: the first from p0, the second from p1
    __device__ __forceinline__ void init(const Operand& o, const char* p0, const char* p1, int mn, int nk_, int total_, int k0) {
        nk = nk_, total = total_;
        const int64_t rows = min(mn, R);
        step = TR ? BK * o.ld : kTileBytes;
        const int last = o.k - (nk - 1) * BK;
        if (TR) {
            bytes = mn > 0 ? (uint32_t)((BK - 1) * o.ld + rows * (int)sizeof(T)) : 0u;
            bytes_last = mn > 0 && last > 0 ? (uint32_t)((last - 1) * o.ld + rows * (int)sizeof(T)) : 0u;
        } else {
            bytes = bytes_last = mn > 0 ? (uint32_t)((rows - 1) * o.ld + (int64_t)o.k * (int)sizeof(T)) : 0u;
        }
        const int skip = k0 >= nk ? k0 - nk : k0;
        p = (k0 >= nk ? p1 : p0) + skip * step;
        second = p1;
        kbytes = o.k * (int)sizeof(T);
        left = kbytes - skip * kTileBytes;
    }
    template <bool MASK, typename TILE> __device__ __forceinline__ void load(const TILE& tile, int kt, char* dst) {
        uint32_t n = kt >= total ? 0u : bytes;
        if (TR && (kt == nk - 1 || kt == total - 1)) n = bytes_last;
        tile.template put<MASK && !TR>(p, n, left, dst);
        p = kt == nk - 1 ? second : p + step;
        if (MASK && !TR) left = kt == nk - 1 ? kbytes : left - kTileBytes;
    }
};

// A transposed LDS read.  The pointer is restrict-qualified: with no alias information on the read
// the compiler waits for every LDS-writing load in flight before it; the order that matters here is
// kept by this file's own waits and barriers.
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
__device__ __forceinline__ s16x4 read_tr4(lds_s16x4* __restrict__ p) { return __builtin_amdgcn_ds_read_tr16_b64_v4i16(p); }
// N fragments of layout T over a whole K-tile: f[block][half of K][four k], from this lane's
// addresses of the blocks' first k, rows of ROW bytes (the permutation of a row's chunks is the
// same four rows on and half a K-tile on)
template <int N, int ROW> __device__ __forceinline__ void read_tr(const uint32_t (&p)[N], uint32_t offset, s16x4 (&f)[N][2][2]) {
#pragma unroll
    for (int t = 0; t < N; ++t)
#pragma unroll
        for (int q = 0; q < 4; ++q)
            f[t][q >> 1][q & 1] = read_tr4((lds_s16x4*)(uintptr_t)(p[t] + offset + (q >> 1) * 32 * ROW + (q & 1) * 4 * ROW));
}
template <int N> __device__ __forceinline__ void wait_loads() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }

// N fragments of a tile, both halves of K, in either layout
template <typename T, int N> union Frags {
    s16x4 h[N][2][2];
    typename Frag<T>::type f[N][2];
    __device__ __forceinline__ Frags() {}
};
// this lane's LDS address of the block of 16 columns from r0 in a layout T tile of R columns
template <typename T, int R> __device__ __forceinline__ uint32_t tr_address(const char* tile, int r0, int lane) {
    const int i = lane & 15, k = (lane >> 4) * 8 + (i >> 2);
    return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const char*)tile + k * (R * 2) +
           (((r0 / 8 + ((i & 3) >> 1)) ^ swz_t<T, R>(k)) << 4) + (i & 1) * 8;
}

// A lane's sums with those of the rows `low` further on in its 16 (the low parts').  A sum that is not
// finite stands alone, as with more rows: an infinite factor meets both parts, and times the low one
// is an infinity of its sign or, where it is 0, NaN.
__device__ __forceinline__ f32x4 with_low_rows(f32x4 v, int low) {
    f32x4 r;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float l = __shfl(v[j], ((int)threadIdx.x & 48) | (((int)threadIdx.x + low) & 15));
        r[j] = finite(v[j]) ? v[j] + l : v[j];
    }
    return r;
}

// ---- the tiled product -----------------------------------------------------------------
// TM x TN tile (B in two halves of TN / 2), WGM x WGN waves.  S buffers of one K-tile: S - 1 are on
// their way while the MFMAs of one run, one barrier a K-tile.  These tiles serve products that do
// not fill the chip with large ones, whose K loop is bound by the latency of a load.
// gemm_tile: tile `id` of product z, slab `split`; smem: S (TM + TN) K-tiles' rows.
template <typename T, bool TRA, bool TRB, int TM, int TN, int WGM, int WGN, int S, int EPI>
__device__ __forceinline__ void gemm_tile(const GemmArgs& a, int id, int z, int split, char* smem) {
    constexpr int NT = 64 * WGM * WGN, TH = TN / 2, RA = TM / WGM / 16, RB = TH / WGN / 16;
    using TA = Tile<T, TRA, TM, NT>;
    using TB = Tile<T, TRB, TH, NT>;
    constexpr int BUF = TA::BYTES + 2 * TB::BYTES;
    constexpr int LOADS = TA::PER + 2 * TB::PER;   // a wave's, a K-tile
    static_assert(BUF == (TM + TN) * kTileBytes, "what the callers set aside");
    const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6, wm = wid / WGN, wn = wid % WGN;

    const int tiles = a.tiles_m * a.tiles_n;
    int tm, tn;
    tile_of(id, tiles, a.tiles_m, a.tiles_n, tm, tn);
    const int m0 = tm * TM, n0 = EPI == kGatedForward ? tn * TH : tn * TN;

    TA ta;
    TB tb;
    ta.init(a.a.ld);
    tb.init(a.b.ld);
    const int64_t am = TRA ? (int64_t)m0 * (int)sizeof(T) : (int64_t)m0 * a.a.ld;
    const int64_t bn = TRB ? (int64_t)n0 * (int)sizeof(T) : (int64_t)n0 * a.b.ld;
    const int64_t bh = TRB ? (int64_t)TH * (int)sizeof(T) : (int64_t)TH * a.b.ld;

    const int nk = (a.a.k + TA::BK - 1) / TA::BK, total = nk * a.segments;
    const int k0 = (int)((int64_t)total * split / a.splits), k1 = (int)((int64_t)total * (split + 1) / a.splits);
    const char *a0 = a.a.p[a.batch > 1 ? z : 0] + am, *a1 = a.a.p[1] + am;   // a batch has one segment
    const char *b0 = a.b.p[0] + bn, *b1 = a.b.p[1] + bn;
    Cursor<T, TRA, TM> ca;
    ca.init(a.a, a0, a1, a.a.mn - m0, nk, total, k0);
    Cursor<T, TRB, TH> cb[2];
    if constexpr (EPI == kGatedForward) {
        cb[0].init(a.b, b0, b0, a.b.mn - n0, nk, total, k0);
        cb[1].init(a.b, b1, b1, a.b.mn - n0, nk, total, k0);
    } else {
        cb[0].init(a.b, b0, b1, a.b.mn - n0, nk, total, k0);
        cb[1].init(a.b, b0 + bh, b1 + bh, a.b.mn - n0 - TH, nk, total, k0);
    }
    auto stage = [&](int kt, int buf) {
        char* dst = smem + buf * BUF;
        ca.template load<true>(ta, kt, dst);
        cb[0].template load<true>(tb, kt, dst + TA::BYTES);
        cb[1].template load<true>(tb, kt, dst + TA::BYTES + TB::BYTES);
    };

    // float32 operands: a sum for each half of the K-tiles, added at the end.  The rounding of a sum
    // grows with the root of its length, and theirs is not hidden under a 16-bit result's.
    constexpr int SUMS = sizeof(T) == 4 ? 2 : 1;
    f32x4 acc[SUMS][2][RB][RA];
#pragma unroll
    for (int c = 0; c < SUMS; ++c)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int j = 0; j < RB; ++j)
#pragma unroll
                for (int i = 0; i < RA; ++i) acc[c][h][j][i] = f32x4{0.f, 0.f, 0.f, 0.f};

    uint32_t xa[RA], xb[RB];   // layout T: addresses in the first buffer
#pragma unroll
    for (int i = 0; i < RA; ++i) xa[i] = tr_address<T, TM>(smem, (wm * RA + i) * 16, lane);
#pragma unroll
    for (int j = 0; j < RB; ++j) xb[j] = tr_address<T, TH>(smem + TA::BYTES, (wn * RB + j) * 16, lane);

    // past the end of K (k1: past this split's) the loads bring what nothing reads; the counts hold
#pragma unroll
    for (int i = 0; i < S - 1; ++i) stage(k0 + i, i);
    int buf = 0;
    for (int kt = k0; kt < k1; ++kt) {
        wait_loads<(S - 2) * LOADS>();
        __builtin_amdgcn_s_barrier();   // K-tile kt is there for every wave, and kt - 1 read by all
        asm volatile("" ::: "memory");
        const int next = buf == 0 ? S - 1 : buf - 1;
        const char* sa = smem + buf * BUF;
        const char* sb = sa + TA::BYTES;
        Frags<T, RA> fa;
        Frags<T, RB> fb[2];
        if constexpr (TRA && sizeof(T) == 2) {
            read_tr<RA, TM * 2>(xa, buf * BUF, fa.h);
        } else {
#pragma unroll
            for (int i = 0; i < RA; ++i)
#pragma unroll
                for (int s = 0; s < 2; ++s) fa.f[i][s] = TA::frag(sa, (wm * RA + i) * 16, s, lane);
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            if constexpr (TRB && sizeof(T) == 2) {
                read_tr<RB, TH * 2>(xb, buf * BUF + h * TB::BYTES, fb[h].h);
            } else {
#pragma unroll
                for (int j = 0; j < RB; ++j)
#pragma unroll
                    for (int s = 0; s < 2; ++s) fb[h].f[j][s] = TB::frag(sb + h * TB::BYTES, (wn * RB + j) * 16, s, lane);
            }
        }
        asm volatile("" ::: "memory");
        stage(kt + S - 1, next);
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int j = 0; j < RB; ++j)
#pragma unroll
                    for (int i = 0; i < RA; ++i)
                        acc[s % SUMS][h][j][i] = Frag<T>::mma(fb[h].f[j][s], fa.f[i][s], acc[s % SUMS][h][j][i]);
        // the reads have returned (the MFMAs used them) before this wave reaches the next barrier
        buf = buf + 1 == S ? 0 : buf + 1;
    }
    wait_loads<0>();
    // B is the first operand of the MFMAs, so a lane holds four consecutive n of one m
#pragma unroll
    for (int i = 0; i < RA; ++i)
#pragma unroll
        for (int j = 0; j < RB; ++j) {
            const int m = m0 + (wm * RA + i) * 16 + (lane & 15), n = n0 + (wn * RB + j) * 16 + (lane >> 4) * 4;
            f32x4 r0 = acc[0][0][j][i], r1 = acc[0][1][j][i];
            if constexpr (SUMS == 2) r0 += acc[1][0][j][i], r1 += acc[1][1][j][i];
            if constexpr (TM == 16 && EPI == kStore && sizeof(T) == 2) {
                if (a.low) r0 = with_low_rows(r0, a.low), r1 = with_low_rows(r1, a.low);
            }
            finish4<T, EPI>(a, z, split, m, n, n + TH, r0, r1);
        }
}

template <typename T, bool TRA, bool TRB, int TM, int TN, int WGM, int WGN, int S, int EPI>
__global__ __launch_bounds__(64 * WGM * WGN, TM == 64 ? 3 : 2) void ffn_gemm_kernel(GemmArgs a) {
    __shared__ __attribute__((aligned(16))) char smem[S * (TM + TN) * kTileBytes];
    gemm_tile<T, TRA, TRB, TM, TN, WGM, WGN, S, EPI>(a, blockIdx.x, blockIdx.y % a.batch, blockIdx.y / a.batch, smem);
}

// ---- the tiled product, 256 x 256 -----------------------------------------------------------
// 16-bit operands, whole K-tiles where an operand is K-contiguous, eight waves in 2 (m) x 4 (n),
// each 2 x 64 rows by 2 x 32 columns: 128 accumulator registers a lane.  Each operand's tile is two half-tiles of 16 KB; two K-tiles of
// four half-tiles fill 128 KB of LDS.  A K-tile runs as four phases, one quadrant of the result
// each (A0 B0, A0 B1, A1 B1, A1 B0; B's halves the other way round in every second K-tile), so a
// phase reads only the fragments that the registers do not hold, 8, 4, 8 and 4 of them.  Each
// phase puts one half-tile in flight, up to two K-tiles ahead.  The two wave groups (m) run one
// barrier apart, so on every SIMD one wave's MFMAs cover the other's LDS reads and loads.
constexpr int kTile256Bytes = 2 * 4 * 128 * kTileBytes;
// tile `id` of product z, slab `split`
template <typename T, bool TRA, bool TRB, int EPI>
__device__ __forceinline__ void gemm256_tile(const GemmArgs& a, int id, int z, int split, char* smem) {
    static_assert(sizeof(T) == 2, "16-bit operands");
    constexpr int HT = 128 * kTileBytes, BUF = 4 * HT;   // half-tiles A0, A1, B0, B1
    using TA = Tile<T, TRA, 128, 512>;
    using TB = Tile<T, TRB, 128, 512>;
    const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6, wm = wid >> 2, wn = wid & 3;

    const int tiles = a.tiles_m * a.tiles_n;
    int tm, tn;
    tile_of(id, tiles, a.tiles_m, a.tiles_n, tm, tn);
    const int m0 = tm * 256, n0 = EPI == kGatedForward ? tn * 128 : tn * 256;

    TA ta;
    TB tb;
    ta.init(a.a.ld);
    tb.init(a.b.ld);
    const int nk = (a.a.k + TA::BK - 1) / TA::BK, total = nk * a.segments;
    const int k0 = (int)((int64_t)total * split / a.splits), k1 = (int)((int64_t)total * (split + 1) / a.splits);
    const int za = a.batch > 1 ? z : 0;   // a batch has one segment
    const int64_t am = TRA ? (int64_t)m0 * 2 : (int64_t)m0 * a.a.ld, ah = TRA ? 256 : 128 * a.a.ld;
    const int64_t bn = TRB ? (int64_t)n0 * 2 : (int64_t)n0 * a.b.ld, bh = TRB ? 256 : 128 * a.b.ld;
    const char *a0 = a.a.p[za] + am, *a1 = a.a.p[1] + am, *b0 = a.b.p[0] + bn, *b1 = a.b.p[1] + bn;
    Cursor<T, TRA, 128> ca[2];
    ca[0].init(a.a, a0, a1, a.a.mn - m0, nk, total, k0);
    ca[1].init(a.a, a0 + ah, a1 + ah, a.a.mn - m0 - 128, nk, total, k0);
    Cursor<T, TRB, 128> cb[2];
    if constexpr (EPI == kGatedForward) {
        cb[0].init(a.b, b0, b0, a.b.mn - n0, nk, total, k0);
        cb[1].init(a.b, b1, b1, a.b.mn - n0, nk, total, k0);
    } else {
        cb[0].init(a.b, b0, b1, a.b.mn - n0, nk, total, k0);
        cb[1].init(a.b, b0 + bh, b1 + bh, a.b.mn - n0 - 128, nk, total, k0);
    }
    auto stage_a = [&](int h, int kt, int buf) { ca[h].template load<false>(ta, kt, smem + buf * BUF + h * HT); };
    auto stage_b = [&](int h, int kt, int buf) { cb[h].template load<false>(tb, kt, smem + buf * BUF + (2 + h) * HT); };

    uint32_t xa[4], xb[2];   // layout T: addresses in the first buffer
#pragma unroll
    for (int t = 0; t < 4; ++t) xa[t] = tr_address<T, 128>(smem, wm * 64 + t * 16, lane);
#pragma unroll
    for (int u = 0; u < 2; ++u) xb[u] = tr_address<T, 128>(smem, wn * 32 + u * 16, lane);
    Frags<T, 4> fa;
    Frags<T, 2> fb[2];
    auto read_a = [&](int buf, auto half) {
        constexpr int H = decltype(half)::value;
        if constexpr (TRA) {
            read_tr<4, 256>(xa, buf * BUF + H * HT, fa.h);
        } else {
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int s = 0; s < 2; ++s) fa.f[t][s] = TA::frag(smem + buf * BUF + H * HT, wm * 64 + t * 16, s, lane);
        }
    };
    auto read_b = [&](int buf, auto half) {
        constexpr int H = decltype(half)::value;
        if constexpr (TRB) {
            read_tr<2, 256>(xb, buf * BUF + (2 + H) * HT, fb[H].h);
        } else {
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int s = 0; s < 2; ++s) fb[H].f[u][s] = TB::frag(smem + buf * BUF + (2 + H) * HT, wn * 32 + u * 16, s, lane);
        }
    };
    f32x4 acc[2][2][4][2];
#pragma unroll
    for (int i = 0; i < 32; ++i) acc[i >> 4][(i >> 3) & 1][(i >> 1) & 3][i & 1] = f32x4{0.f, 0.f, 0.f, 0.f};
    auto quadrant = [&](auto ha, auto hb) {
        constexpr int A = decltype(ha)::value, B = decltype(hb)::value;
        __builtin_amdgcn_s_barrier();
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int u = 0; u < 2; ++u) acc[A][B][t][u] = Frag<T>::mma(fb[B].f[u][s], fa.f[t][s], acc[A][B][t][u]);
        __builtin_amdgcn_s_setprio(0);
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    using I0 = std::integral_constant<int, 0>;
    using I1 = std::integral_constant<int, 1>;

    // K-tile kt of parity P takes B's half P first.  A half-tile is restaged, for the K-tile after
    // the next, two phases after its last read: the other group's reads of the phase before may
    // still be under way.  Every phase issues one half-tile and lets five stay in flight.  Past
    // the end of K the loads bring zeros that nothing reads, so the counts hold to the last phase.
    auto k_tile = [&](int kt, auto parity) {
        constexpr int P = decltype(parity)::value;
        using First = std::integral_constant<int, P>;
        using Second = std::integral_constant<int, 1 - P>;
        read_a(P, I0{});
        stage_a(1, kt + 1, 1 - P);
        wait_loads<10>();
        quadrant(I0{}, First{});
        read_b(P, Second{});
        stage_b(P, kt + 2, P);
        wait_loads<10>();
        quadrant(I0{}, Second{});
        read_a(P, I1{});
        stage_a(0, kt + 2, P);
        wait_loads<10>();
        quadrant(I1{}, Second{});
        read_b(1 - P, Second{});   // the next K-tile's first half, into the registers this one is done with
        stage_b(1 - P, kt + 2, P);
        wait_loads<10>();
        quadrant(I1{}, First{});
    };
    stage_b(0, k0, 0);
    stage_a(0, k0, 0);
    stage_b(1, k0, 0);
    stage_a(1, k0, 0);
    stage_b(1, k0 + 1, 1);
    stage_a(0, k0 + 1, 1);
    stage_b(0, k0 + 1, 1);
    wait_loads<10>();   // B0 and A0
    __builtin_amdgcn_s_barrier();
    const int group = __builtin_amdgcn_readfirstlane(wm);
    if (group == 1) __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    read_b(0, I0{});
    // group 1 reads here what group 0 restages after one more barrier, a phase sooner than in later
    // K-tiles: its reads have returned before that barrier
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    for (int kt = k0; kt < k1; kt += 2) {
        k_tile(kt, I0{});
        if (kt + 1 < k1) k_tile(kt + 1, I1{});
    }
    if (group == 0) __builtin_amdgcn_s_barrier();   // both groups pass the same number of barriers
    wait_loads<0>();
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int m = m0 + h * 128 + wm * 64 + t * 16 + (lane & 15), n = n0 + wn * 32 + u * 16 + (lane >> 4) * 4;
                finish4<T, EPI>(a, z, split, m, n, n + 128, acc[h][0][t][u], acc[h][1][t][u]);
            }
}

template <typename T, bool TRA, bool TRB, int EPI>
__global__ __launch_bounds__(512) void ffn_gemm256_kernel(GemmArgs a) {
    __shared__ __attribute__((aligned(16))) char smem[kTile256Bytes];
    gemm256_tile<T, TRA, TRB, EPI>(a, blockIdx.x, blockIdx.y % a.batch, blockIdx.y / a.batch, smem);
}

// ---- two products in one launch -------------------------------------------------------------
// Products that need nothing of each other, a's workgroups before b's: b's fill the CUs that a's
// last round leaves and those that are done early, and a launch is saved (777 x 1000 x 2730 trained
// 141 -> 126 us, 100 x 512 x 1408 42 -> 36).  Tiles of both side by side would share an L2 with the
// other's operands: 8192 x 4096 x 11264, dWd and dh 1590-1630 us, an XCD of each kind in turn 1500,
// one after the other 1370-1400, as two launches 1580.  Ids are counted in eights, so all keep their
// XCDs.  B is row-contiguous in every product of backward.
template <typename T, int SIDE, bool TRA, int EPI>
__device__ __forceinline__ void pair_tile(const GemmArgs& g, int id, char* smem) {
    const int tiles = g.tiles_m * g.tiles_n, each = (tiles + 7) / 8 * 8, y = id / each;
    id -= y * each;
    if (id >= tiles) return;
    if constexpr (SIDE == 256)
        gemm256_tile<T, TRA, true, EPI>(g, id, y % g.batch, y / g.batch, smem);
    else
        gemm_tile<T, TRA, true, SIDE, SIDE, 2, 2, SIDE == 64 ? 3 : 2, EPI>(g, id, y % g.batch, y / g.batch, smem);
}
template <typename T, int SIDE, bool TRA1, int EPI1, bool TRA2, int EPI2>
__global__ __launch_bounds__(SIDE == 256 ? 512 : 256, SIDE == 64 ? 3 : 2) void ffn_gemm_pair_kernel(GemmArgs a, GemmArgs b, int first) {
    __shared__ __attribute__((aligned(16))) char smem[(SIDE == 64 ? 3 : 2) * 2 * SIDE * kTileBytes];
    const int id = blockIdx.x;
    if (id < first)
        pair_tile<T, SIDE, TRA1, EPI1>(a, id, smem);
    else
        pair_tile<T, SIDE, TRA2, EPI2>(b, id - first, smem);
}

// slabs [splits][batch][M][ldp] added in order and rounded once
template <typename T>
__global__ __launch_bounds__(256) void ffn_join_kernel(const float* __restrict__ slab, int splits, int batch, int64_t M,
                                                       int N, int64_t ldp, T* c0, T* c1, int64_t ldc) {
    const int64_t per = ldp / 4, i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= M * batch * per) return;
    const int64_t zm = i / per, n = (i - zm * per) * 4, z = zm / M, m = zm - z * M;
    if (n >= N) return;
    f32x4 s = *reinterpret_cast<const f32x4*>(slab + zm * ldp + n);
#pragma unroll 8   // the additions are in order, the loads need not wait for each other
    for (int k = 1; k < splits; ++k) s += *reinterpret_cast<const f32x4*>(slab + ((int64_t)k * batch * M + zm) * ldp + n);
    T* c = (z ? c1 : c0) + m * ldc;
    const bool vec = (ldc & 3) == 0 && ((uintptr_t)(z ? c1 : c0) & (4 * sizeof(T) - 1)) == 0;
    store4(c + n, (int)(N - n < 4 ? N - n : 4), vec, s);
}

// ---- few rows ------------------------------------------------------------------------------
// Up to 16 rows of x: the weights are read once, straight into registers, and bound the time.
// A workgroup takes 16 features (GATED: of both weights); its NW waves take 128-byte pieces of
// K in turn and meet in LDS.  Rows of x past the last are zero fragments.  low: GATED, where the
// low parts of the results go; else the low parts of x follow its rows (low = rows), in MFMA rows
// that would be zeros.
template <typename T, bool GATED, int NW>
__global__ __launch_bounds__(64 * NW) void ffn_few_kernel(const T* __restrict__ x, int64_t ldx, int rows,
                                                          const T* __restrict__ w0, const T* __restrict__ w1,
                                                          int64_t ldw, int K, int N, int act, T* __restrict__ out,
                                                          int64_t ldo, float* __restrict__ sg, float* __restrict__ su,
                                                          int low) {
    constexpr int NB = GATED ? 2 : 1, PIECE = 128 / (int)sizeof(T), CH = 16 / (int)sizeof(T);
    constexpr int UNROLL = GATED ? 2 : 4;
    __shared__ f32x4 part[NW][NB][64];
    const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6, r = lane & 15, kc = lane >> 4;
    const int n0 = blockIdx.x * 16;
    const int64_t wrow = n0 + r < N ? n0 + r : N - 1;   // past the end: read the last row, drop the result
    const T* pw[2] = {w0 + wrow * ldw, GATED ? w1 + wrow * ldw : nullptr};
    const bool live = r < rows, read = r < rows + (GATED ? 0 : low);
    const T* px = x + (int64_t)(read ? r : 0) * ldx;
    using F = typename Frag<T>::type;
    using U = T __attribute__((ext_vector_type(16 / sizeof(T)), aligned(sizeof(T))));
    auto chunk = [&](const T* p, int k) -> F {
        F f{};
        if (k + CH <= K) {
            const U q = *reinterpret_cast<const U*>(p + k);
#pragma unroll
            for (int j = 0; j < CH; ++j) f[j] = q[j];
        } else {
#pragma unroll
            for (int j = 0; j < CH; ++j)
                if (k + j < K) f[j] = p[k + j];
        }
        return f;
    };
    f32x4 acc[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) acc[b] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int k0 = wid * PIECE; k0 < K; k0 += NW * PIECE * UNROLL) {
        F fw[UNROLL][2][NB], fx[UNROLL][2];
#pragma unroll
        for (int u = 0; u < UNROLL; ++u)
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                const int k = k0 + u * NW * PIECE + (s * 4 + kc) * CH;
#pragma unroll
                for (int b = 0; b < NB; ++b) fw[u][s][b] = chunk(pw[b], k);
                fx[u][s] = read ? chunk(px, k) : F{};
            }
#pragma unroll
        for (int u = 0; u < UNROLL; ++u)
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int b = 0; b < NB; ++b) acc[b] = Frag<T>::mma(fw[u][s][b], fx[u][s], acc[b]);
    }
#pragma unroll
    for (int b = 0; b < NB; ++b) part[wid][b][lane] = acc[b];
    __syncthreads();
    if (wid) return;
    f32x4 s[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        s[b] = part[0][b][lane];
#pragma unroll
        for (int w = 1; w < NW; ++w) s[b] += part[w][b][lane];
    }
    if constexpr (!GATED && sizeof(T) == 2) {
        if (low) s[0] = with_low_rows(s[0], low);
    }
    if (!live) return;
    const int n = n0 + kc * 4;
    if constexpr (GATED) {   // ldo whole K-tiles, columns up to it written (zeros past N)
        f32x4 h;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (n + j >= N) s[0][j] = s[1][j] = 0.0f;
            h[j] = act_value<T>(act, s[0][j]) * s[1][j];
        }
        if (n >= ldo) return;
        const int64_t o = (int64_t)r * ldo + n;
        store_hidden(out + o, low * ldo, h);
        if (sg) {
            store4(sg + o, 4, true, s[0]);
            store4(su + o, 4, true, s[1]);
        }
    } else {
        const bool vec = (ldo & 3) == 0 && ((uintptr_t)out & (4 * sizeof(T) - 1)) == 0;
        store4(out + (int64_t)r * ldo + n, N - n, vec, s[0]);
    }
}

// ---- weight gradients of few rows -------------------------------------------------------------
// C[r, c] = sum_n A[n, r] B[n, c] over up to NR rows, up to three such sums in one launch: bound by
// the writing of C (bf16, 4096 x 11264, 1 row: the three take 45 us where tiles take 120).  A
// thread holds its 8 columns of B's rows in registers and walks `walk` rows of C, 16 or, where that
// leaves CUs idle, 4; A's values come from LDS.
struct OuterJob {
    const void *a, *b;
    void* c;
    int64_t lda, ldb, ldc;
    int64_t low_a, low_b;   // elements to the low parts, 0: none
    int R, C;
    int across;     // threads across the columns, a power of two from 32 to 256
    int wide;       // workgroups across the columns
    int64_t first;  // the job's first workgroup
};
struct OuterArgs {
    OuterJob job[3];
    int count, rows, walk;
};
template <typename T, int NR> __global__ __launch_bounds__(256) void ffn_outer_kernel(OuterArgs o) {
    __shared__ float sa[NR * 128];
    int k = 0;
    while (k + 1 < o.count && blockIdx.x >= o.job[k + 1].first) ++k;
    const OuterJob& j = o.job[k];
    const int block = (int)(blockIdx.x - j.first), deep = 256 / j.across, RB = o.walk * deep;
    const int tx = threadIdx.x % j.across, ty = threadIdx.x / j.across;
    const int r0 = (block / j.wide) * RB, col = ((block % j.wide) * j.across + tx) * 8;
    for (int i = threadIdx.x; i < NR * RB; i += 256) {
        const int n = i / RB, r = r0 + i % RB;
        float a = 0.0f;
        if (n < o.rows && r < j.R) {
            const T* p = (const T*)j.a + n * j.lda + r;
            a = (float)p[0];
            if (j.low_a) a += (float)p[j.low_a];
        }
        sa[i] = a;
    }
    __syncthreads();
    const int valid = j.C - col;
    if (valid <= 0) return;
    float b[NR][8];
#pragma unroll
    for (int n = 0; n < NR; ++n) {
        if (n < o.rows) {
            const T* p = (const T*)j.b + n * j.ldb + col;
            load8(p, valid, b[n]);
            if (j.low_b) {
                float l[8];
                load8(p + j.low_b, valid, l);
#pragma unroll
                for (int q = 0; q < 8; ++q) b[n][q] += l[q];
            }
        } else {
#pragma unroll
            for (int q = 0; q < 8; ++q) b[n][q] = 0.0f;
        }
    }
    for (int i = 0; i < o.walk; ++i) {
        const int in = i * deep + ty, r = r0 + in;
        if (r >= j.R) break;
        float v[8];
#pragma unroll
        for (int q = 0; q < 8; ++q) v[q] = 0.0f;
#pragma unroll
        for (int n = 0; n < NR; ++n) {
            const float a = sa[n * RB + in];
#pragma unroll
            for (int q = 0; q < 8; ++q) v[q] += a * b[n][q];
        }
        store8((T*)j.c + (int64_t)r * j.ldc + col, valid, v);
    }
}

// The same sums of 5 to 16 rows of 16-bit operands by MFMA, one step of 16 terms (with the low
// parts: up to 8 rows and as many more), so that they too are bound by the writing: bf16, 4096 x 11264,
// 8 rows 65 -> 56 us, 16 rows 102 -> 56; 1 row, without the MFMA, 45 instead of 59.
// A wave takes 128 columns (64: 59 us) and walks `walk` blocks of 16 rows of C.  A fragment's row i
// of column block x stands for column (x / 2) 32 + (i / 4) 8 + (x % 2) 4 + i % 4, so that a lane ends with
// runs of 8 columns of a row, four lanes' beside each other.
template <typename T> struct Outer;
template <> struct Outer<_Float16> {
    typedef __attribute__((ext_vector_type(4))) _Float16 type;
    static __device__ __forceinline__ f32x4 mma(type a, type b) {
        return __builtin_amdgcn_mfma_f32_16x16x16f16(a, b, f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
    }
};
template <> struct Outer<__bf16> {
    typedef __attribute__((ext_vector_type(4))) __bf16 type;
    static __device__ __forceinline__ f32x4 mma(type a, type b) {
        return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(s16x4, a), __builtin_bit_cast(s16x4, b),
                                                         f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
    }
};
template <typename T> __global__ __launch_bounds__(256) void ffn_outer_mfma_kernel(OuterArgs o) {
    int k = 0;
    while (k + 1 < o.count && blockIdx.x >= o.job[k + 1].first) ++k;
    const OuterJob& j = o.job[k];
    const int block = (int)(blockIdx.x - j.first), lane = threadIdx.x & 63, q = lane >> 4, i = lane & 15;
    const int r0 = (block / j.wide) * o.walk * 16, c0 = (block % j.wide) * 512 + (threadIdx.x >> 6) * 128;
    if (c0 >= j.C) return;
    const int terms = j.low_a || j.low_b ? 2 * o.rows : o.rows;
    // this lane's four terms of operand p at column `at` of `width`; a term past the rows: the low part
    auto four = [&](const T* p, int64_t ld, int64_t low, int at, int width) {
        typename Outer<T>::type v;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int n = q * 4 + e;
            const bool second = n >= o.rows;
            v[e] = n < terms && at < width ? p[(second ? n - o.rows : n) * ld + (second ? low : 0) + at] : (T)0.0f;
        }
        return v;
    };
    typename Outer<T>::type b[8];
#pragma unroll
    for (int x = 0; x < 8; ++x) b[x] = four((const T*)j.b, j.ldb, j.low_b, c0 + (x >> 1) * 32 + (i >> 2) * 8 + (x & 1) * 4 + (i & 3), j.C);
    const int col = c0 + q * 8, last = min(j.R, r0 + o.walk * 16);
    typename Outer<T>::type a = four((const T*)j.a, j.lda, j.low_a, r0 + i, j.R);
    // a fragment without its low terms
    auto high = [&](typename Outer<T>::type v) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (q * 4 + e >= o.rows) v[e] = (T)0.0f;
        return v;
    };
    for (int r = r0; r < last; r += 16) {
        const typename Outer<T>::type now = a;
        a = four((const T*)j.a, j.lda, j.low_a, r + 16 + i, last);
        float v[4][8];
        float bad = 0.0f;   // NaN where one of this lane's sums is not finite
#pragma unroll
        for (int x = 0; x < 8; ++x) {
            const f32x4 s = Outer<T>::mma(b[x], now);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                v[x >> 1][(x & 1) * 4 + e] = s[e];
                bad = __builtin_fmaf(s[e], 0.0f, bad);
            }
        }
        // with_low_rows' rule: a sum that is not finite is that of the high parts alone
        if (terms > o.rows && __any(bad != bad)) {
#pragma unroll
            for (int x = 0; x < 8; ++x) {
                const f32x4 s = Outer<T>::mma(high(b[x]), high(now));
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float& w = v[x >> 1][(x & 1) * 4 + e];
                    w = finite(w) ? w : s[e];
                }
            }
        }
        if (r + i >= last) continue;
        T* c = (T*)j.c + (int64_t)(r + i) * j.ldc + col;
#pragma unroll
        for (int h = 0; h < 4; ++h)
            if (j.C - col > h * 32) store8(c + h * 32, j.C - col - h * 32, v[h]);
    }
}

// ---- copies for unaligned operands ---------------------------------------------------------
// Rows copied to a leading dimension that is a multiple of 8, zeros past the last column.
struct PackItem {
    const void* src;
    void* dst;
    int64_t lds, ldd, rows, cols, first;   // first: index of the item's first chunk of 8
};
struct PackArgs {
    PackItem item[5];
    int count;
    int64_t total;
};
template <typename T> __global__ __launch_bounds__(256) void ffn_pack_kernel(PackArgs a) {
    const int64_t i = block_id() * 256 + threadIdx.x;
    if (i >= a.total) return;
    int k = 0;
    while (k + 1 < a.count && i >= a.item[k + 1].first) ++k;
    const PackItem& it = a.item[k];
    const int64_t per = it.ldd / 8, j = i - it.first, row = j / per, col = (j - row * per) * 8;
    float v[8];
    const int64_t left = it.cols - col;
    load8((const T*)it.src + row * it.lds + col, (int)(left < 8 ? left : 8), v);
    store8((T*)it.dst + row * it.ldd + col, 8, v);
}
template <typename T> __global__ __launch_bounds__(256) void ffn_zero_kernel(T* p, int64_t rows, int64_t cols, int64_t ld) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < rows * cols; i += (int64_t)gridDim.x * 256)
        p[i / cols * ld + i % cols] = (T)0.0f;
}

// ------------------------------------------------------------------------------------- host
int64_t up8(int64_t x) { return (x + 7) / 8 * 8; }
int64_t up_ktile(int64_t x, int es) { return (x + kTileBytes / es - 1) / (kTileBytes / es) * (kTileBytes / es); }
size_t up256(size_t x) { return (x + 255) / 256 * 256; }
size_t esize(int32_t t) { return t == OTF_F32 ? 4 : 2; }

struct Carver {
    char* base;
    size_t used = 0;
    void* take(size_t bytes) {
        void* p = base ? base + used : nullptr;
        used += up256(bytes);
        return p;
    }
};

// A product: operand layouts, extents, and what becomes of the result
struct Product {
    bool tra, trb;
    int epi;
    GemmArgs a;
};

constexpr int kCus = 256;   // MI355X; only tile choice depends on it

// Tile side and slabs of K, by the least estimated time.  A CU holds one tile of 256, two of 128,
// three of 64 or five of 16 by 64; a K-tile then takes it c microseconds (less where it holds
// fewer), a tile's start and results e, and slabs are written at 4 and joined at 6.4 TB/s.  Fitted
// to bf16 products of 64 to 4096 rows by 512 to 4096 and 1408 to 11264 columns, each run with all
// three sides:
//   gate and up 1024 x 2048 x 5632   62 / 91 / 85 us with 256 / 128 / 64   (176, 704, 2816 tiles)
//               64 x 4096 x 11264    85 / 93 / 58                          (88, 176, 352)
//   dh          1024 x 2048 x 5632   78 / 50 / 60                          (88, 352, 1408)
//   dx          1024 x 2048 x 5632   87 / 65 / 101, the first two with 16 and 4 slabs
//   dWg and dWu 777 x 1024 x 2752    36 / 20 / 28
struct Plan {
    int side, splits;
};
int per_cu(int side) { return side == 256 ? 1 : side == 128 ? 2 : side == 64 ? 3 : 5; }
int64_t tiles_of(const Product& p, int side) {
    const int64_t across = side == 16 ? 64 : side, width = p.epi == kGatedForward ? across / 2 : across;
    return (p.a.M + side - 1) / side * ((p.a.N + width - 1) / width) * p.a.batch;
}
int64_t ktiles_of(const Product& p, int elem) {
    const int depth = kTileBytes / elem;
    return (int64_t)((p.a.a.k + depth - 1) / depth) * p.a.segments;
}
bool can_take(const Product& p, int elem, int side) {
    if (side == 16) return !p.tra && p.a.M <= 16;
    if (p.a.low) return false;
    return side != 256 || (elem == 2 && (p.tra || p.a.a.k % 64 == 0) && (p.trb || p.a.b.k % 64 == 0));
}
// a tile of this many K-tiles where the launch fills `full` of the chip's slots
double tile_us(int side, int elem, int64_t ktiles, double full) {
    const double c = elem == 2 ? (side == 256 ? 1.35 : side == 128 ? 1.1 : side == 64 ? 0.75 : 0.6) : (side == 128 ? 4.2 : side == 64 ? 1.9 : 0.8);
    const double e = side == 256 ? 14.0 : side == 128 ? 11.0 : 5.0;
    return (double)ktiles * c * (side == 256 ? 1.0 : 0.5 + 0.5 * (full < 1.0 ? full : 1.0)) + e;
}
double join_us(const Product& p, int splits) {
    return splits > 1 ? 4.0 + (double)splits * p.a.batch * p.a.M * p.a.N * 4.0 * (1 / 6.4e6 + 1 / 4.0e6) : 0.0;
}
Plan plan_product(const Product& p, int elem, double* us = nullptr) {
    const int64_t ktiles = ktiles_of(p, elem);
    Plan best{64, 1};
    double least = 1e30;
    for (int side : {256, 128, 64, 16}) {   // 16: 16 rows by 64 columns
        if (!can_take(p, elem, side)) continue;
        const int64_t tiles = tiles_of(p, side), slots = (int64_t)kCus * per_cu(side);
        for (int splits = 1; splits <= 32; splits *= 2) {
            if (splits > 1 && (p.epi != kStore || tiles * splits > slots || ktiles / splits < 4)) break;
            const double full = (double)(tiles * splits) / slots;
            const double rounds = full < 1.0 ? 1.0 : side <= 64 ? full : (double)((tiles + slots - 1) / slots);
            const double t = rounds * tile_us(side, elem, (ktiles + splits - 1) / splits, full) + join_us(p, splits);
            if (t < least) least = t, best = Plan{side, splits};
        }
    }
    if (us) *us = least;
    return best;
}

// na tiles of ta, then nb of tb, each where a slot is free first
double two_runs_us(int64_t slots, int64_t na, double ta, int64_t nb, double tb) {
    const int64_t full = na / slots, late = na % slots;   // `late` slots take one more of a's
    const double start = (double)full * ta;
    int64_t k0 = 0, k1 = 0;   // b's that an early and a late slot take
    while ((slots - late) * k0 + late * k1 < nb)
        if (late == 0 || start + (double)(k0 + 1) * tb <= start + ta + (double)(k1 + 1) * tb) ++k0;
        else ++k1;
    const double early = start + (double)k0 * tb, last = late ? start + ta + (double)k1 * tb : 0.0;
    return early > last ? early : last;
}

// Two products in one launch of one tile, where that is estimated to be faster than a launch each: the
// second's tiles go where the first's leave room, and about 4 us of a launch's start and end are saved
// (at 1 % of large ones: dx and dW of 8192 x 4096 x 11264, whose rounds are the same, 2445 us both ways).
struct Pair {
    int side;   // 0: a launch each
    int splits; // of the first product
};
Pair plan_pair(const Product& a, const Product& b, int elem) {
    double ua, ub;
    plan_product(a, elem, &ua);
    plan_product(b, elem, &ub);
    double least = 0.99 * (ua + ub) + 4.0;
    Pair best{0, 1};
    for (int side : {256, 128, 64}) {
        if (!can_take(a, elem, side) || !can_take(b, elem, side)) continue;
        const int64_t ka = ktiles_of(a, elem), kb = ktiles_of(b, elem), slots = (int64_t)kCus * per_cu(side), nb = tiles_of(b, side);
        for (int splits = 1; splits <= 32; splits *= 2) {
            const int64_t na = tiles_of(a, side) * splits;
            if (splits > 1 && (na > slots || ka / splits < 4)) break;
            const double full = (double)(na + nb) / slots;
            const double ta = tile_us(side, elem, (ka + splits - 1) / splits, full), tb = tile_us(side, elem, kb, full);
            double t = ta > tb ? ta : tb;
            if (full > 1.0) {   // small tiles have no rounds: a slot is free soon
                const double run = side == 64 ? ((double)na * ta + (double)nb * tb) / slots : two_runs_us(slots, na, ta, nb, tb);
                t = run > t ? run : t;
            }
            t += join_us(a, splits);
            if (t < least) least = t, best = Pair{side, splits};
        }
    }
    return best;
}
size_t slab_bytes(const Product& p, int splits) {
    return splits > 1 ? (size_t)splits * p.a.batch * p.a.M * (size_t)up8(p.a.N) * 4 : 0;
}

template <typename T, bool TRA, bool TRB, int EPI>
hipError_t launch_tiles(GemmArgs a, const Plan& q, hipStream_t s) {
    // both operands run over the same K-tiles: the cursors shorten only the last one's rows
    constexpr int depth = kTileBytes / (int)sizeof(T);
    if ((a.a.k + depth - 1) / depth != (a.b.k + depth - 1) / depth) return hipErrorInvalidValue;
    a.splits = q.splits;
    a.tiles_m = (a.M + q.side - 1) / q.side;
    const int across = q.side == 16 ? 64 : q.side, cols = EPI == kGatedForward ? across / 2 : across;
    a.tiles_n = (a.N + cols - 1) / cols;
    const dim3 grid((unsigned)(a.tiles_m * a.tiles_n), (unsigned)(a.batch * q.splits));
    if (q.side == 256) {
        if constexpr (sizeof(T) == 2)
            ffn_gemm256_kernel<T, TRA, TRB, EPI><<<grid, 512, 0, s>>>(a);
        else
            return hipErrorInvalidValue;
    } else if (q.side == 128) {
        // a third buffer where a CU has only one tile: 4096 x 1024 x 4096, down product, 82 -> 56 us.  With
        // a T operand it gains nothing, and two tiles of two buffers are faster where there are more.
        if constexpr (!TRA && !TRB) {
            if ((int64_t)grid.x * grid.y <= kCus) {
                ffn_gemm_kernel<T, TRA, TRB, 128, 128, 2, 2, 3, EPI><<<grid, 256, 0, s>>>(a);
                return hipGetLastError();
            }
        }
        ffn_gemm_kernel<T, TRA, TRB, 128, 128, 2, 2, 2, EPI><<<grid, 256, 0, s>>>(a);
    } else if (q.side == 16) {   // up to 16 rows: a taller tile's MFMAs would be spent on rows that are not there
        if constexpr (!TRA && (TRB || sizeof(T) == 2))   // float32's forward takes the few-rows kernel
            ffn_gemm_kernel<T, TRA, TRB, 16, 64, 1, 2, 3, EPI><<<grid, 128, 0, s>>>(a);
        else
            return hipErrorInvalidValue;
    } else {
        ffn_gemm_kernel<T, TRA, TRB, 64, 64, 2, 2, 3, EPI><<<grid, 256, 0, s>>>(a);
    }
    return hipGetLastError();
}

// the product with its result in the slabs of `q` where it has some, and what joins them
GemmArgs slabs(const Product& p, int splits, float* slab) {
    GemmArgs a = p.a;
    a.splits = splits;
    if (splits > 1) a.c[0] = slab, a.ldc = up8(a.N);
    return a;
}
template <typename T> hipError_t join(const Product& p, int splits, const float* slab, hipStream_t s) {
    if (splits == 1) return hipSuccess;
    const GemmArgs& a = p.a;
    const int64_t ldc = up8(a.N), work = (int64_t)a.M * a.batch * (ldc / 4);
    ffn_join_kernel<T><<<(unsigned)((work + 255) / 256), 256, 0, s>>>(slab, splits, a.batch, a.M, a.N, ldc, (T*)a.c[0],
                                                                     (T*)a.c[1], a.ldc);
    return hipGetLastError();
}

template <typename T, bool TRA, bool TRB>
hipError_t run_store(const Product& p, float* slab, hipStream_t s) {
    const Plan q = plan_product(p, (int)sizeof(T));
    const hipError_t e = launch_tiles<T, TRA, TRB, kStore>(slabs(p, q.splits, slab), q, s);
    return e != hipSuccess ? e : join<T>(p, q.splits, slab, s);
}

template <typename T, bool TRA1, bool TRA2, int EPI2>
hipError_t run_pair(const Product& p, const Product& second, const Pair& q, float* slab, hipStream_t s) {
    constexpr int depth = kTileBytes / (int)sizeof(T);
    GemmArgs a = slabs(p, q.splits, slab), b = second.a;
    int64_t blocks[2];
    for (GemmArgs* g : {&a, &b}) {
        if ((g->a.k + depth - 1) / depth != (g->b.k + depth - 1) / depth) return hipErrorInvalidValue;
        g->tiles_m = (g->M + q.side - 1) / q.side, g->tiles_n = (g->N + q.side - 1) / q.side;
        blocks[g == &b] = ((int64_t)g->tiles_m * g->tiles_n + 7) / 8 * 8 * g->batch * g->splits;
    }
    const unsigned grid = (unsigned)(blocks[0] + blocks[1]);
    const int first = (int)blocks[0];
    if (q.side == 256) {
        if constexpr (sizeof(T) == 2)
            ffn_gemm_pair_kernel<T, 256, TRA1, kStore, TRA2, EPI2><<<grid, 512, 0, s>>>(a, b, first);
        else
            return hipErrorInvalidValue;
    } else if (q.side == 128) {
        ffn_gemm_pair_kernel<T, 128, TRA1, kStore, TRA2, EPI2><<<grid, 256, 0, s>>>(a, b, first);
    } else {
        ffn_gemm_pair_kernel<T, 64, TRA1, kStore, TRA2, EPI2><<<grid, 256, 0, s>>>(a, b, first);
    }
    const hipError_t e = hipGetLastError();
    return e != hipSuccess ? e : join<T>(p, q.splits, slab, s);
}

// Up to 8 rows of 16-bit operands: the hidden values (h, dg, du) keep their low parts, as many more
// rows that a 16-row tile has room for, so that only the results are rounded (y of one token 1.0
// instead of 1.4 times its rounding off).  More rows would cost MFMAs and passes over the hidden
// values.
int low_rows_of(int64_t rows, int es) { return es == 2 && rows <= 8 ? (int)rows : 0; }
// The block's buffers and products.  Built twice: for the sizes (null pointers) and to run.
struct Block {
    const otf_ffn_args* o;
    int es;
    int64_t n, d, f, fk;    // fk: f in whole K-tiles, the hidden buffers' leading dimension, zeros past f
    int low;                // rows of low parts after a hidden buffer's
    int64_t nh;             // its rows with them
    bool whole;             // operands copied to whole K-tiles (large products of ragged widths)
    Operand x{}, wg{}, wu{}, wd{}, dy{};   // k: columns there are, zeros past the caller's
    PackArgs pack{};
    Carver ws{};

    Block(const otf_ffn_args* args, int elem, void* workspace) : o(args), es(elem) {
        n = o->rows, d = o->d, f = o->f, fk = up_ktile(f, es);
        low = low_rows_of(n, es), nh = n + low;
        // ragged widths: a copy costs two passes over the operands, and pays where the products are large
        whole = es == 2 && ((n + 255) / 256) * ((f + 127) / 128) >= kCus;
        ws.base = (char*)workspace;
    }

    // by_k: the columns are K in some product
    bool aligned(const void* p, int64_t ld, int64_t cols, bool by_k) const {
        return cols % (whole && by_k ? 64 : 8) == 0 && ld % 8 == 0 && (uintptr_t)p % 16 == 0;
    }
    void place(Operand& v, const void* p, int64_t ld, int64_t rows, int64_t cols, bool copy) {
        v.p[0] = v.p[1] = (const char*)p;
        v.ld = ld * es;
        v.k = (int)cols;
        if (copy) {
            const int64_t ldd = up_ktile(cols, es);
            void* dst = ws.take((size_t)(rows * ldd * es));
            pack.item[pack.count++] = PackItem{p, dst, ld, ldd, rows, cols, pack.total};
            pack.total += rows * (ldd / 8);
            v.p[0] = v.p[1] = (const char*)dst;
            v.ld = ldd * es;
            v.k = (int)ldd;
        }
    }
    // gate and up: one leading dimension, so both are copied or none
    void weights_in(bool by_k) {
        const bool copy = !aligned(o->w_gate, o->ldw_in, d, by_k) || !aligned(o->w_up, o->ldw_in, d, by_k);
        place(wg, o->w_gate, o->ldw_in, f, d, copy);
        place(wu, o->w_up, o->ldw_in, f, d, copy);
    }
    void operand(Operand& v, const void* p, int64_t ld, int64_t rows, int64_t cols, bool by_k) {
        place(v, p, ld, rows, cols, !aligned(p, ld, cols, by_k));
    }
    template <typename T> hipError_t run_pack(hipStream_t s) {
        if (!pack.count) return hipSuccess;
        ffn_pack_kernel<T><<<blocks((pack.total + 255) / 256), 256, 0, s>>>(pack);
        return hipGetLastError();
    }
};

// an input as layout K (its columns are k, `k` of them) or T (its rows are k)
Operand by_rows(const Operand& v, int64_t rows, int64_t k) {
    Operand r = v;
    r.mn = (int)rows;
    r.k = (int)k;
    return r;
}
Operand by_columns(const Operand& v, int64_t rows) {
    Operand r = v;
    r.mn = v.k;
    r.k = (int)rows;
    return r;
}
Operand buffer_operand(const void* p, int64_t ld, int es, int64_t mn, int64_t k) {
    return Operand{{(const char*)p, (const char*)p}, ld * es, (int)mn, (int)k};
}
GemmArgs product_args(const Operand& a, const Operand& b, int64_t M, int64_t N, void* c, int64_t ldc) {
    GemmArgs g{};
    g.a = a, g.b = b, g.M = (int)M, g.N = (int)N, g.segments = 1, g.splits = 1, g.batch = 1;
    g.c[0] = c, g.ldc = ldc;
    return g;
}

// The few-rows kernel takes one MFMA tile of rows.  With more of them its reads of x grow beside
// the weights': bf16, d = 4096, f = 11264, 16 rows 71 us against 57 for the tiles, 1 row 53; d = 1024,
// f = 4096, 16 rows 16.0 against 18.6.  float32 tiles are slower everywhere up to 16 rows.
bool few_rows(int64_t rows, int64_t d, int64_t f, int es) {
    return rows <= 16 && (es == 4 || rows * d * f <= (int64_t)1 << 26);
}

constexpr int64_t kMaxRows = INT32_MAX / 8, kMaxWidth = 1 << 20, kMaxElements = (int64_t)1 << 34;
bool is_type(int32_t t) { return t == OTF_F32 || t == OTF_F16 || t == OTF_BF16; }

int check_ffn(const otf_ffn_args* o) {
    if (!o) return OTF_EINVAL;
    if (!is_type(o->dtype)) return OTF_EINVAL;
    if (o->activation != OTF_ACT_SILU && o->activation != OTF_ACT_GELU) return OTF_EINVAL;
    if (o->rows < 0 || o->d <= 0 || o->f <= 0) return OTF_EINVAL;
    // 32-bit element counts of a row tile and of the K extents
    if (o->rows > kMaxRows || o->d > kMaxWidth || o->f > kMaxWidth) return OTF_EUNSUPPORTED;
    // and 32-bit thread counts of the products' launches (the copies of operands, up to five in one, count theirs in two dimensions)
    const int64_t wide = o->d > o->f ? o->d : o->f;
    if (o->d * o->f > kMaxElements || o->rows * wide > kMaxElements) return OTF_EUNSUPPORTED;
    return OTF_OK;
}
// leading dimensions: 256 rows within a 31-bit byte offset
bool bad_ld(int64_t ld, int64_t cols) { return ld < cols || ld > (1 << 20); }
bool misaligned(const void* p, int32_t dtype) { return (uintptr_t)p % esize(dtype) != 0; }

struct Saved {
    float *g, *u;
    char* h;
};
Saved carve_saved(void* p, int64_t n, int64_t fk) {
    if (!p) return Saved{};   // a size query
    char* b = (char*)p;
    const size_t wide = up256((size_t)(n * fk) * 4);
    return Saved{(float*)b, (float*)(b + wide), b + 2 * wide};
}
size_t saved_bytes(int64_t n, int64_t fk, int es) {
    return 2 * up256((size_t)(n * fk) * 4) + up256((size_t)((n + low_rows_of(n, es)) * fk * es));
}

// forward: the workspace it needs in *need; runs where `have` is given, the bytes that there are
template <typename T> int forward(const otf_ffn_args* o, void* workspace, size_t* need, const size_t* have, hipStream_t s) {
    Block b(o, (int)sizeof(T), workspace);
    Saved sv{};
    if (o->saved)
        sv = carve_saved(o->saved, b.n, b.fk);
    else
        sv.h = (char*)b.ws.take((size_t)(b.nh * b.fk * b.es));
    if (few_rows(b.n, b.d, b.f, b.es)) {
        *need = b.ws.used;
        if (!have) return OTF_OK;
        if (*need && (!workspace || *have < *need)) return OTF_EINVAL;
        const unsigned g1 = (unsigned)((b.fk + 15) / 16), g2 = (unsigned)((b.d + 15) / 16);
        ffn_few_kernel<T, true, 4><<<g1, 256, 0, s>>>((const T*)o->x, o->ldx, (int)b.n, (const T*)o->w_gate,
                                                       (const T*)o->w_up, o->ldw_in, (int)b.d, (int)b.f, o->activation,
                                                       (T*)sv.h, b.fk, sv.g, sv.u, b.low);
        OTF_HIP(hipGetLastError());
        ffn_few_kernel<T, false, 8><<<g2, 512, 0, s>>>((const T*)sv.h, b.fk, (int)b.n, (const T*)o->w_down, nullptr,
                                                        o->ldw_down, (int)b.f, (int)b.d, 0, (T*)o->y, o->ldy, nullptr,
                                                        nullptr, b.low);
        return check_hip(hipGetLastError());
    }
    b.operand(b.x, o->x, o->ldx, b.n, b.d, true);
    b.weights_in(true);
    b.operand(b.wd, o->w_down, o->ldw_down, b.d, b.f, true);
    const int kin = b.x.k < b.wg.k ? b.x.k : b.wg.k;   // what is copied ends in zeros
    Product in{false, false, kGatedForward, product_args(by_rows(b.x, b.n, kin), by_rows(b.wg, b.f, kin), b.n, b.fk, nullptr, 0)};
    in.a.b.p[1] = b.wu.p[0];
    in.a.act = o->activation, in.a.features = (int)b.f, in.a.g = sv.g, in.a.u = sv.u, in.a.h = sv.h, in.a.ldh = b.fk, in.a.low = b.low;
    Product down{false, false, kStore, product_args(buffer_operand(sv.h, b.fk, b.es, b.nh, b.wd.k), by_rows(b.wd, b.d, b.wd.k), b.n, b.d, o->y, o->ldy)};
    down.a.low = b.low;
    float* slab = (float*)b.ws.take(slab_bytes(down, plan_product(down, b.es).splits));
    *need = b.ws.used;
    if (!have) return OTF_OK;
    if (*need && (!workspace || *have < *need)) return OTF_EINVAL;
    OTF_HIP(b.run_pack<T>(s));
    OTF_HIP((launch_tiles<T, false, false, kGatedForward>(in.a, plan_product(in, b.es), s)));
    OTF_HIP((run_store<T, false, false>(down, slab, s)));
    return OTF_OK;
}

constexpr int kOuterRows = 16;

// dWg, dWu and dWd, those that are wanted, of up to kOuterRows rows
template <typename T>
hipError_t run_outer(const Block& b, const char* dg, const char* du, const char* h, hipStream_t s) {
    const otf_ffn_args* o = b.o;
    OuterArgs args{};
    args.rows = (int)b.n;
    const bool mfma = sizeof(T) == 2 && b.n > 4;
    // a thousand workgroups of 16 rows by 256 threads, or by MFMA of 128 rows by 512 columns: else shorter walks
    args.walk = mfma ? (b.d * b.f >= (int64_t)1 << 24 ? 8 : 4) : b.d * b.f >= (int64_t)1 << 23 ? 16 : 4;
    int64_t blocks = 0;
    auto add = [&](const void* a, int64_t lda, int64_t low_a, int64_t R, const void* bb, int64_t ldb, int64_t low_b, int64_t C, void* c, int64_t ldc) {
        int across = 32;
        while (across < 256 && across * 8 < C) across *= 2;
        const int64_t wide = mfma ? (C + 511) / 512 : (C + across * 8 - 1) / (across * 8);
        const int64_t deep = args.walk * (mfma ? 16 : 256 / across);
        args.job[args.count++] = OuterJob{a, bb, c, lda, ldb, ldc, low_a, low_b, (int)R, (int)C, across, (int)wide, blocks};
        blocks += wide * ((R + deep - 1) / deep);
    };
    if (o->dw_gate) {
        add(dg, b.fk, b.low * b.fk, b.f, o->x, o->ldx, 0, b.d, o->dw_gate, o->lddw_in);
        add(du, b.fk, b.low * b.fk, b.f, o->x, o->ldx, 0, b.d, o->dw_up, o->lddw_in);
    }
    if (o->dw_down) add(o->dy, o->lddy, 0, b.d, h, b.fk, b.low * b.fk, b.f, o->dw_down, o->lddw_down);
    if (!args.count) return hipSuccess;
    if constexpr (sizeof(T) == 2) {
        if (mfma)
            ffn_outer_mfma_kernel<T><<<(unsigned)blocks, 256, 0, s>>>(args);
        else
            ffn_outer_kernel<T, 4><<<(unsigned)blocks, 256, 0, s>>>(args);
    } else {
        if (b.n <= 4)
            ffn_outer_kernel<T, 4><<<(unsigned)blocks, 256, 0, s>>>(args);
        else if (b.n <= 8)
            ffn_outer_kernel<T, 8><<<(unsigned)blocks, 256, 0, s>>>(args);
        else
            ffn_outer_kernel<T, kOuterRows><<<(unsigned)blocks, 256, 0, s>>>(args);
    }
    return hipGetLastError();
}

template <typename T> int backward(const otf_ffn_args* o, void* workspace, size_t* need, const size_t* have, hipStream_t s) {
    Block b(o, (int)sizeof(T), workspace);
    const Saved sv = carve_saved(o->saved, b.n, b.fk);
    const bool win = o->dw_gate != nullptr, wdown = o->dw_down != nullptr, wx = o->dx != nullptr;
    char* dg = (char*)b.ws.take((size_t)(b.nh * b.fk * b.es));
    char* du = (char*)b.ws.take((size_t)(b.nh * b.fk * b.es));
    b.operand(b.dy, o->dy, o->lddy, b.n, b.d, true);
    if (wx || win) b.operand(b.wd, o->w_down, o->ldw_down, b.d, b.f, false);
    if (wx) b.weights_in(false);
    const bool outer = b.n <= kOuterRows;   // the weights' gradients without tiles
    if (win && !outer) b.operand(b.x, o->x, o->ldx, b.n, b.d, false);
    // dh = dy Wd: K = d, the rows of Wd
    Product mid{false, true, kGatedBackward, product_args(by_rows(b.dy, b.n, b.dy.k), by_columns(b.wd, b.d), b.n, b.fk, nullptr, 0)};
    mid.a.act = o->activation, mid.a.features = (int)b.f, mid.a.g = sv.g, mid.a.u = sv.u, mid.a.h = dg, mid.a.h2 = du, mid.a.ldh = b.fk, mid.a.low = b.low;
    // dx = dg Wg + du Wu: two segments of K = f, the rows of the weights
    Product px{false, true, kStore, product_args(buffer_operand(dg, b.fk, b.es, b.nh, b.fk), by_columns(b.wg, b.f), b.n, b.d, o->dx, o->lddx)};
    px.a.a.p[1] = du, px.a.b.p[1] = b.wu.p[0], px.a.segments = 2, px.a.low = b.low;
    // dWg, dWu = dg^T x, du^T x: a batch of two, K = rows
    Product pi{true, true, kStore, product_args(buffer_operand(dg, b.fk, b.es, b.fk, b.n), by_columns(b.x, b.n), b.f, b.d, o->dw_gate, o->lddw_in)};
    pi.a.a.p[1] = du, pi.a.c[1] = o->dw_up, pi.a.batch = 2;
    // dWd = dy^T h
    Product pd{true, true, kStore, product_args(by_columns(b.dy, b.n), buffer_operand(sv.h, b.fk, b.es, b.fk, b.n), b.d, b.f, o->dw_down, o->lddw_down)};
    // what needs nothing of each other shares a launch: dWd and dh, then dx and dWg, dWu
    const bool dh = wx || win;
    const Pair with_dh = dh && wdown && !outer ? plan_pair(pd, mid, b.es) : Pair{0, 1};
    const Pair with_in = wx && win && !outer ? plan_pair(px, pi, b.es) : Pair{0, 1};
    size_t slab = 0;   // one after another on the stream: they share it
    auto more = [&](const Product& p, const Pair& q) {
        const size_t k = slab_bytes(p, q.side ? q.splits : plan_product(p, b.es).splits);
        slab = k > slab ? k : slab;
    };
    if (wx) more(px, with_in);
    if (win && !outer && !with_in.side) more(pi, Pair{0, 1});
    if (wdown && !outer) more(pd, with_dh);
    float* part = (float*)b.ws.take(slab);
    *need = b.ws.used;
    if (!have) return OTF_OK;
    if (*need && (!workspace || *have < *need)) return OTF_EINVAL;
    OTF_HIP(b.run_pack<T>(s));
    if (with_dh.side)
        OTF_HIP((run_pair<T, true, false, kGatedBackward>(pd, mid, with_dh, part, s)));
    else if (dh)
        OTF_HIP((launch_tiles<T, false, true, kGatedBackward>(mid.a, plan_product(mid, b.es), s)));
    if (with_in.side)
        OTF_HIP((run_pair<T, false, true, kStore>(px, pi, with_in, part, s)));
    else if (wx)
        OTF_HIP((run_store<T, false, true>(px, part, s)));
    if (outer) {
        OTF_HIP((run_outer<T>(b, dg, du, sv.h, s)));
        return OTF_OK;
    }
    if (win && !with_in.side) OTF_HIP((run_store<T, true, true>(pi, part, s)));
    if (wdown && !with_dh.side) OTF_HIP((run_store<T, true, true>(pd, part, s)));
    return OTF_OK;
}

template <typename T> hipError_t zero_rows(void* p, int64_t rows, int64_t cols, int64_t ld, hipStream_t s) {
    const int64_t n = (rows * cols + 255) / 256;
    ffn_zero_kernel<T><<<(unsigned)(n < 65536 ? n : 65536), 256, 0, s>>>((T*)p, rows, cols, ld);
    return hipGetLastError();
}

int forward_any(const otf_ffn_args* o, void* ws, size_t* need, const size_t* have, hipStream_t s) {
    if (o->dtype == OTF_F32) return forward<float>(o, ws, need, have, s);
    if (o->dtype == OTF_F16) return forward<_Float16>(o, ws, need, have, s);
    return forward<__bf16>(o, ws, need, have, s);
}
int backward_any(const otf_ffn_args* o, void* ws, size_t* need, const size_t* have, hipStream_t s) {
    if (o->dtype == OTF_F32) return backward<float>(o, ws, need, have, s);
    if (o->dtype == OTF_F16) return backward<_Float16>(o, ws, need, have, s);
    return backward<__bf16>(o, ws, need, have, s);
}

}  // namespace
}  // namespace otf

using namespace otf;

extern "C" {

size_t otf_gated_ffn_saved_size(int64_t rows, int64_t f, int32_t dtype) {
    if (rows <= 0 || f <= 0 || !is_type(dtype)) return 0;
    if (rows > kMaxRows || f > kMaxWidth || rows * f > kMaxElements) return 0;   // no call takes them
    return saved_bytes(rows, up_ktile(f, (int)esize(dtype)), (int)esize(dtype));
}

size_t otf_gated_ffn_workspace_size(const otf_ffn_args* o) {
    size_t need = 0;
    if (check_ffn(o) != OTF_OK || o->rows == 0) return 0;
    forward_any(o, nullptr, &need, nullptr, nullptr);
    return need;
}

size_t otf_gated_ffn_backward_workspace_size(const otf_ffn_args* o) {
    size_t need = 0;
    if (check_ffn(o) != OTF_OK || o->rows == 0) return 0;
    backward_any(o, nullptr, &need, nullptr, nullptr);
    return need;
}

int otf_gated_ffn(const otf_ffn_args* o, void* workspace, size_t workspace_bytes, otf_stream_t stream) {
    const int rc = check_ffn(o);
    if (rc != OTF_OK || o->rows == 0) return rc;
    if (!o->x || !o->w_gate || !o->w_up || !o->w_down || !o->y) return OTF_EINVAL;
    if (bad_ld(o->ldx, o->d) || bad_ld(o->ldw_in, o->d) || bad_ld(o->ldw_down, o->f) || o->ldy < o->d) return OTF_EINVAL;
    for (const void* p : {o->x, o->w_gate, o->w_up, o->w_down, (const void*)o->y})
        if (misaligned(p, o->dtype)) return OTF_EINVAL;
    if ((uintptr_t)o->saved % 16 || (uintptr_t)workspace % 16) return OTF_EINVAL;
    size_t need = 0;
    return forward_any(o, workspace, &need, &workspace_bytes, (hipStream_t)stream);
}

int otf_gated_ffn_backward(const otf_ffn_args* o, void* workspace, size_t workspace_bytes, otf_stream_t stream) {
    const int rc = check_ffn(o);
    if (rc != OTF_OK) return rc;
    if ((o->dw_gate == nullptr) != (o->dw_up == nullptr)) return OTF_EINVAL;
    hipStream_t s = (hipStream_t)stream;
    if (o->dw_gate && (o->lddw_in < o->d || misaligned(o->dw_gate, o->dtype) || misaligned(o->dw_up, o->dtype))) return OTF_EINVAL;
    if (o->dw_down && (o->lddw_down < o->f || misaligned(o->dw_down, o->dtype))) return OTF_EINVAL;
    if (o->rows == 0) {   // no row: the sums are zero
        auto zero = [&](void* p, int64_t r, int64_t c, int64_t ld) {
            if (!p) return hipSuccess;
            return o->dtype == OTF_F32 ? zero_rows<float>(p, r, c, ld, s) : zero_rows<_Float16>(p, r, c, ld, s);
        };
        OTF_HIP(zero(o->dw_gate, o->f, o->d, o->lddw_in));
        OTF_HIP(zero(o->dw_up, o->f, o->d, o->lddw_in));
        OTF_HIP(zero(o->dw_down, o->d, o->f, o->lddw_down));
        return OTF_OK;
    }
    if (!o->dy || !o->saved || !o->w_down || bad_ld(o->lddy, o->d) || bad_ld(o->ldw_down, o->f)) return OTF_EINVAL;
    if (o->dx && (!o->w_gate || !o->w_up || bad_ld(o->ldw_in, o->d) || o->lddx < o->d)) return OTF_EINVAL;
    if (o->dw_gate && (!o->x || bad_ld(o->ldx, o->d))) return OTF_EINVAL;
    for (const void* p : {o->dy, o->x, o->w_gate, o->w_up, o->w_down, (const void*)o->dx})
        if (misaligned(p, o->dtype)) return OTF_EINVAL;
    if ((uintptr_t)o->saved % 16 || (uintptr_t)workspace % 16) return OTF_EINVAL;
    size_t need = 0;
    return backward_any(o, workspace, &need, &workspace_bytes, s);
}

}  // extern "C"
