// otf_norm.hip — dropout, layer norm and the residual sum with both, forward and backward.
//
// All of it is bound by HBM: each operand is read once and each result written once, rows
// are held in registers between the statistics and the output, and the dropout mask is made
// again from its counter instead of being stored (otf_rng.h).
//
//   dropout                y = [residual +] keep * x / (1 - p)
//   layer norm             y = (x - mean) rstd w + b, statistics of a row in float32, the
//                          variance from the centred values (a second pass over registers:
//                          E[x^2] - mean^2 would cancel for rows with a large mean)
//   its backward           c = dy w;  dx = rstd (c - mean(c) - xhat mean(c xhat));
//                          dw = sum_rows dy xhat;  db = sum_rows dy
//   residual norm          z = residual + dropout(x), y = LN(z) of the float32 sum; backward adds
//                          the gradient that reaches z directly.  It reads z where z is stored
//                          in float32 and makes the sum again from x and residual where z was
//                          rounded to 16 bits: dw sums dy xhat over the rows, which a rounded
//                          row would put off by 2e-3 (2 more bytes an element, of 10)
//
// dw and db: every workgroup keeps float32 partials of its rows in registers and writes them
// once; a second launch adds the partials in a fixed order (no atomics: the same bits every
// call).
#include "otf_rng.h"

namespace otf {
namespace {

// widest rows held in registers: 1024 threads x 4 chunks of 8; backward, which also holds the
// parameter gradients' sums, 512 threads x 4
constexpr int kMaxHeldCols = 32768, kMaxHeldColsBackward = 16384;
// Up to here the parameter gradients share the backward launch: 5 us less of a call that the host
// bounds.  The sum over rows is then one workgroup's: 64 x 1024 float32 replayed from a graph 16 us both
// ways, 128 x 4096 21 us against 18, 256 x 1024 28 against 16.
constexpr int kFewRows = 64;

struct NormArgs {
    const void* x;       // forward: input; backward: the normalised input (x or z), or with res x
    int64_t ldx;
    const void* res;     // residual
    int64_t ldr;
    const void* dz;      // backward (may be null)
    int64_t lddz;
    const void* dy;      // backward
    int64_t lddy;
    void* y;             // forward: y; backward: dx
    int64_t ldy;
    void* z;             // forward: z; backward: dresidual
    int64_t ldz;
    const void* w;
    const void* b;
    int wf32;            // weight and bias are float32 (else the input's type)
    float* mean;
    float* rstd;
    float* partial;      // backward: [grid][2][cols]
    void* dw;            // backward, one workgroup: written directly
    void* db;
    int64_t rows;
    int cols;
    float eps;
    const int64_t* rng;
    uint32_t threshold;
    float scale;
};

__device__ __forceinline__ int chunk_valid(int cols, int col) { return cols - col < 8 ? cols - col : 8; }

template <typename T>
__device__ __forceinline__ void load_param8(const void* p, int wf32, int col, int valid, float (&v)[8]) {
    if (wf32)
        load8((const float*)p + col, valid, v);
    else
        load8((const T*)p + col, valid, v);
}

// x over lanes whose ids differ below bit TPR (a row's lanes), or from it on (the rows of a wave)
template <int TPR> __device__ __forceinline__ float row_lanes_sum(float x) {
    if constexpr (TPR > 1) x += wave_xor<float, 1>(x);
    if constexpr (TPR > 2) x += wave_xor<float, 2>(x);
    if constexpr (TPR > 4) x += wave_xor<float, 4>(x);
    if constexpr (TPR > 8) x += wave_xor<float, 8>(x);
    if constexpr (TPR > 16) x += wave_xor<float, 16>(x);
    if constexpr (TPR > 32) x += wave_xor<float, 32>(x);
    return x;
}

// Sum of NV values over the TPR threads of a row.  Up to 64: within a wave, no LDS.  Else one
// barrier: `red` holds two generations of [wave][NV], and a wave can be at most one
// reduction ahead of another.
template <int TPR, int NV>
__device__ __forceinline__ void row_sums(float (&s)[NV], float* red, int& gen) {
#pragma unroll
    for (int i = 0; i < NV; ++i) s[i] = TPR >= 64 ? wave_sum(s[i]) : row_lanes_sum<TPR>(s[i]);
    if constexpr (TPR > 64) {
        constexpr int NW = TPR / 64;
        float* slot = red + gen * NW * NV;
        const int wid = threadIdx.x >> 6;
        if ((threadIdx.x & 63) == 0)
#pragma unroll
            for (int i = 0; i < NV; ++i) slot[wid * NV + i] = s[i];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            float t = 0.0f;
#pragma unroll
            for (int w = 0; w < NW; ++w) t += slot[w * NV + i];
            s[i] = t;
        }
        gen ^= 1;
    }
}

// ------------------------------------------------------------------------------- dropout
// One thread a group of 8 columns.  FLAT: the tensor is one run of whole groups (no row
// arithmetic).
template <typename T, bool RES, bool FLAT>
__global__ __launch_bounds__(256) void dropout_kernel(const T* __restrict__ x, int64_t ldx,
                                                      const T* __restrict__ res, int64_t ldr, T* __restrict__ y,
                                                      int64_t ldy, uint64_t total, uint32_t groups, int cols,
                                                      const int64_t* __restrict__ rng, uint32_t threshold,
                                                      float scale) {
    const uint64_t g = (uint64_t)block_id() * 256 + threadIdx.x;
    if (g >= total) return;
    int64_t ox, orr, oy;
    int valid = 8;
    if constexpr (FLAT) {
        ox = orr = oy = (int64_t)g * 8;
    } else {
        const uint64_t row = (total >> 32) ? g / groups : (uint64_t)((uint32_t)g / groups);
        const int col = (int)(g - row * groups) * 8;
        valid = chunk_valid(cols, col);
        ox = (int64_t)row * ldx + col;
        orr = (int64_t)row * ldr + col;
        oy = (int64_t)row * ldy + col;
    }
    float v[8];
    load8(x + ox, valid, v);
    float r[8];
    if constexpr (RES) load8(res + orr, valid, r);
    drop8(v, keep8(g, drop_key(rng), threshold), scale);
    if constexpr (RES)
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] += r[j];
    store8(y + oy, valid, v);
}

// ---------------------------------------------------------------------------- layer norm
// TPR threads a row, CH chunks of 8 columns a thread (chunk c of thread t: column
// (c TPR + t) 8); a workgroup of max(TPR, 256) threads.
template <typename T, typename TR, bool DROP, int TPR, int CH>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void norm_forward_kernel(NormArgs a) {
    constexpr int NT = TPR > 256 ? TPR : 256, RPB = NT / TPR;
    __shared__ float red[TPR > 64 ? 2 * (TPR / 64) : 1];
    int gen = 0;
    const int t = threadIdx.x % TPR;
    const int64_t row = block_id() * RPB + threadIdx.x / TPR;
    if (row >= a.rows) return;   // all of a row's threads; RPB > 1 only where they share a wave
    const int cols = a.cols;
    const T* x = (const T*)a.x + row * a.ldx;
    float v[CH][8];
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int col = (c * TPR + t) * 8;
        load8(x + col, cols - col, v[c]);
    }
    if constexpr (DROP) {
        const TR* res = (const TR*)a.res + row * a.ldr;
        TR* z = (TR*)a.z + row * a.ldz;
        const DropKey key = drop_key(a.rng);
        const uint64_t first = (uint64_t)row * (uint32_t)((cols + 7) / 8);
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int col = (c * TPR + t) * 8;
            if (col >= cols) continue;
            float r[8];
            load8(res + col, cols - col, r);
            drop8(v[c], keep8(first + (uint32_t)(col / 8), key, a.threshold), a.scale);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[c][j] = col + j < cols ? v[c][j] + r[j] : 0.0f;
            store8(z + col, cols - col, v[c]);
        }
    }
    float s[1] = {0.0f};
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int j = 0; j < 8; ++j) s[0] += v[c][j];
    row_sums<TPR, 1>(s, red, gen);
    const float mean = s[0] / (float)cols;
    s[0] = 0.0f;
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float d = (c * TPR + t) * 8 + j < cols ? v[c][j] - mean : 0.0f;
            s[0] += d * d;
        }
    row_sums<TPR, 1>(s, red, gen);
    const float rstd = rsqrtf(s[0] / (float)cols + a.eps);
    if (t == 0 && a.mean) {
        a.mean[row] = mean;
        a.rstd[row] = rstd;
    }
    T* y = (T*)a.y + row * a.ldy;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int col = (c * TPR + t) * 8;
        if (col >= cols) continue;
        float w[8], b[8];
        if (a.w) load_param8<T>(a.w, a.wf32, col, cols - col, w);
        if (a.b) load_param8<T>(a.b, a.wf32, col, cols - col, b);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            float o = (v[c][j] - mean) * rstd;
            if (a.w) o *= w[j];
            if (a.b) o += b[j];
            v[c][j] = o;
        }
        store8(y + col, cols - col, v[c]);
    }
}

// Rows wider than kMaxHeldCols: one workgroup a row, the row read three times (its second
// and third reading come from L2 / the memory-side cache).
template <typename T, typename TR, bool DROP>
__global__ __launch_bounds__(1024) void norm_forward_long_kernel(NormArgs a) {
    __shared__ float red[2 * 16];
    int gen = 0;
    const int64_t row = block_id();
    if (row >= a.rows) return;
    const int cols = a.cols;
    const T* x = (const T*)a.x + row * a.ldx;
    TR* z = DROP ? (TR*)a.z + row * a.ldz : nullptr;
    float s[1] = {0.0f};
    auto sum_of = [&](int64_t col, int valid, float (&v)[8]) {   // the row's values, in float32
        load8(x + col, valid, v);
        if constexpr (DROP) {
            float r[8];
            load8((const TR*)a.res + row * a.ldr + col, valid, r);
            const uint64_t index = (uint64_t)row * (uint32_t)((cols - 1) / 8 + 1) + (uint64_t)(col / 8);
            drop8(v, keep8(index, drop_key(a.rng), a.threshold), a.scale);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = j < valid ? v[j] + r[j] : 0.0f;
        }
    };
    for (int64_t col = threadIdx.x * 8; col < cols; col += 8192) {
        const int valid = (int)(cols - col < 8 ? cols - col : 8);
        float v[8];
        sum_of(col, valid, v);
        if constexpr (DROP) store8(z + col, valid, v);
#pragma unroll
        for (int j = 0; j < 8; ++j) s[0] += v[j];
    }
    row_sums<1024, 1>(s, red, gen);
    const float mean = s[0] / (float)cols;
    s[0] = 0.0f;
    auto again = [&](int64_t col, int valid, float (&v)[8]) {   // this thread's own z where it holds the sum
        if constexpr (DROP && sizeof(TR) == 4)
            load8((const TR*)z + col, valid, v);
        else
            sum_of(col, valid, v);
    };
    for (int64_t col = threadIdx.x * 8; col < cols; col += 8192) {
        const int valid = (int)(cols - col < 8 ? cols - col : 8);
        float v[8];
        again(col, valid, v);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float d = j < valid ? v[j] - mean : 0.0f;
            s[0] += d * d;
        }
    }
    row_sums<1024, 1>(s, red, gen);
    const float rstd = rsqrtf(s[0] / (float)cols + a.eps);
    if (threadIdx.x == 0 && a.mean) {
        a.mean[row] = mean;
        a.rstd[row] = rstd;
    }
    for (int64_t col = threadIdx.x * 8; col < cols; col += 8192) {
        const int valid = (int)(cols - col < 8 ? cols - col : 8);
        float v[8], w[8], b[8];
        again(col, valid, v);
        if (a.w) load_param8<T>(a.w, a.wf32, (int)col, valid, w);
        if (a.b) load_param8<T>(a.b, a.wf32, (int)col, valid, b);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            float o = (v[j] - mean) * rstd;
            if (a.w) o *= w[j];
            if (a.b) o += b[j];
            v[j] = o;
        }
        store8((T*)a.y + row * a.ldy + col, valid, v);
    }
}

// One parameter gradient's partial sums
__device__ __forceinline__ void store_partial(const NormArgs& a, int which, int col, const float (&s)[8]) {
    store8(a.partial + ((int64_t)blockIdx.x * 2 + which) * a.cols + col, chunk_valid(a.cols, col), s);
}

// Workgroup blockIdx.x of `groups`, its rows groups RPB apart.  WG: parameter gradients wanted.  TR: the type of residual and z (= T
// without the residual sum); a 16-bit one makes the sum again from x and residual.
template <typename T, typename TR, bool DROP, bool WG, int NT, int TPR, int CH>
__device__ __forceinline__ void norm_backward_rows(const NormArgs& a, int groups) {
    constexpr int RPB = NT / TPR;
    __shared__ float red[TPR > 64 ? 4 * (TPR / 64) : 1];
    __shared__ float comb[WG && RPB > 1 ? (NT / 64 - 1) * 64 * 8 : 1];
    int gen = 0;
    const int t = threadIdx.x % TPR, part = threadIdx.x / TPR;
    const int cols = a.cols;
    float w[CH][8], gw[CH][8], gb[CH][8];
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int col = (c * TPR + t) * 8;
#pragma unroll
        for (int j = 0; j < 8; ++j) w[c][j] = 1.0f, gw[c][j] = 0.0f, gb[c][j] = 0.0f;
        if (a.w && col < cols) load_param8<T>(a.w, a.wf32, col, cols - col, w[c]);
    }
    const float inv = 1.0f / (float)cols;
    DropKey key{};
    if constexpr (DROP) key = drop_key(a.rng);
    // where the registers allow, the next row is on its way while this one is reduced and stored:
    // a workgroup has one row at a time, and its loads' latency would stand between rows
    // (16384 x 4096 bf16: 131 us without)
    constexpr bool AGAIN = DROP && sizeof(TR) == 2;
    constexpr bool AHEAD = NT == 256 && CH * (sizeof(T) + sizeof(TR) + (AGAIN ? 2 : 0)) <= 16;
    typename Chunk8<TR>::type rx[CH], rr[CH];
    typename Chunk8<T>::type rg[CH];
    float row_mean = 0.0f, row_rstd = 0.0f;
    auto fetch = [&](int64_t row) {
        const TR* x = (const TR*)a.x + row * a.ldx;
        const T* dy = (const T*)a.dy + row * a.lddy;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int col = (c * TPR + t) * 8;
            rx[c] = load8_raw(x + col, cols - col);
            rg[c] = load8_raw(dy + col, cols - col);
            if constexpr (AGAIN) rr[c] = load8_raw((const TR*)a.res + row * a.ldr + col, cols - col);
        }
        row_mean = a.mean[row];
        row_rstd = a.rstd[row];
    };
    const int64_t first = (int64_t)blockIdx.x * RPB + part, step = (int64_t)groups * RPB;
    if (AHEAD && first < a.rows) fetch(first);
    for (int64_t row = first; row < a.rows; row += step) {
        if (!AHEAD) fetch(row);
        float v[CH][8], g[CH][8];
        uint32_t kept[CH];
#pragma unroll
        for (int c = 0; c < CH; ++c) {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[c][j] = (float)rx[c][j], g[c][j] = (float)rg[c][j];
            if constexpr (DROP)
                kept[c] = keep8((uint64_t)row * (uint32_t)((cols + 7) / 8) + (uint32_t)(c * TPR + t), key, a.threshold);
            if constexpr (AGAIN) {
                drop8(v[c], kept[c], a.scale);
#pragma unroll
                for (int j = 0; j < 8; ++j) v[c][j] += (float)rr[c][j];
            }
        }
        const float mean = row_mean, rstd = row_rstd;
        if (AHEAD && row + step < a.rows) fetch(row + step);
        float s[2] = {0.0f, 0.0f};
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int col = (c * TPR + t) * 8;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float xh = col + j < cols ? (v[c][j] - mean) * rstd : 0.0f;
                v[c][j] = xh;
                if constexpr (WG) {
                    gw[c][j] += g[c][j] * xh;
                    gb[c][j] += g[c][j];
                }
                g[c][j] *= w[c][j];
                s[0] += g[c][j];
                s[1] += g[c][j] * xh;
            }
        }
        row_sums<TPR, 2>(s, red, gen);
        const float m1 = s[0] * inv, m2 = s[1] * inv;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int col = (c * TPR + t) * 8;
            if (col >= cols) continue;
#pragma unroll
            for (int j = 0; j < 8; ++j) g[c][j] = rstd * (g[c][j] - m1 - v[c][j] * m2);
            if constexpr (DROP) {
                if (a.dz) {
                    float r[8];
                    load8((const TR*)a.dz + row * a.lddz + col, cols - col, r);
#pragma unroll
                    for (int j = 0; j < 8; ++j) g[c][j] += r[j];
                }
                store8((TR*)a.z + row * a.ldz + col, cols - col, g[c]);
                drop8(g[c], kept[c], a.scale);
            }
            store8((T*)a.y + row * a.ldy + col, cols - col, g[c]);
        }
    }
    if constexpr (WG) {
        if constexpr (RPB == 1) {
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                const int col = (c * TPR + t) * 8;
                if (col >= cols) continue;
                store_partial(a, 0, col, gw[c]);
                store_partial(a, 1, col, gb[c]);
            }
        } else {   // a wave's rows joined by exchanges, the waves through LDS, a chunk of one gradient at a time
            constexpr int NW = NT / 64;
            const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
#pragma unroll
            for (int i = 0; i < 2 * CH; ++i) {
                float(&s)[8] = (i & 1) ? gb[i >> 1] : gw[i >> 1];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    if constexpr (TPR <= 8) s[j] += wave_xor<float, 8>(s[j]);
                    if constexpr (TPR <= 16) s[j] += wave_xor<float, 16>(s[j]);
                    if constexpr (TPR <= 32) s[j] += wave_xor<float, 32>(s[j]);
                }
                __syncthreads();
                if (wid > 0)
#pragma unroll
                    for (int j = 0; j < 8; ++j) comb[((wid - 1) * 8 + j) * 64 + lane] = s[j];
                __syncthreads();
                const int col = ((i >> 1) * TPR + t) * 8;
                if (wid == 0 && lane < TPR && col < cols) {
                    for (int p = 0; p < NW - 1; ++p)
#pragma unroll
                        for (int j = 0; j < 8; ++j) s[j] += comb[(p * 8 + j) * 64 + lane];
                    store_partial(a, i & 1, col, s);
                }
            }
        }
    }
}

// x -> residual + dropout(x) of one chunk
template <typename TR>
__device__ __forceinline__ void add_residual(const NormArgs& a, int64_t row, int64_t col, int valid, uint32_t kept,
                                             float (&v)[8]) {
    float r[8];
    load8((const TR*)a.res + row * a.ldr + col, valid, r);
    drop8(v, kept, a.scale);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] += r[j];
}

// Rows wider than kMaxHeldColsBackward: dx (and dresidual) by one workgroup a row.
template <typename T, typename TR, bool DROP>
__global__ __launch_bounds__(1024) void norm_backward_long_kernel(NormArgs a) {
    __shared__ float red[2 * 16 * 2];
    int gen = 0;
    const int64_t row = block_id();
    if (row >= a.rows) return;
    const int cols = a.cols;
    const TR* x = (const TR*)a.x + row * a.ldx;
    const T* dy = (const T*)a.dy + row * a.lddy;
    const float mean = a.mean[row], rstd = a.rstd[row];
    float m1 = 0.0f, m2 = 0.0f;
    for (int pass = 0; pass < 2; ++pass) {
        float s[2] = {0.0f, 0.0f};
        for (int64_t col = threadIdx.x * 8; col < cols; col += 8192) {
            const int valid = (int)(cols - col < 8 ? cols - col : 8);
            float v[8], g[8], w[8];
            uint32_t kept = 0;
            load8(x + col, valid, v);
            load8(dy + col, valid, g);
            if constexpr (DROP)
                kept = keep8((uint64_t)row * (uint32_t)((cols - 1) / 8 + 1) + (uint64_t)(col / 8), drop_key(a.rng), a.threshold);
            if constexpr (DROP && sizeof(TR) == 2) add_residual<TR>(a, row, col, valid, kept, v);
            if (a.w) load_param8<T>(a.w, a.wf32, (int)col, valid, w);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                v[j] = j < valid ? (v[j] - mean) * rstd : 0.0f;
                if (a.w) g[j] *= w[j];
                s[0] += g[j];
                s[1] += g[j] * v[j];
            }
            if (pass == 1) {
#pragma unroll
                for (int j = 0; j < 8; ++j) g[j] = rstd * (g[j] - m1 - v[j] * m2);
                if constexpr (DROP) {
                    if (a.dz) {
                        float r[8];
                        load8((const TR*)a.dz + row * a.lddz + col, valid, r);
#pragma unroll
                        for (int j = 0; j < 8; ++j) g[j] += r[j];
                    }
                    store8((TR*)a.z + row * a.ldz + col, valid, g);
                    drop8(g, kept, a.scale);
                }
                store8((T*)a.y + row * a.ldy + col, valid, g);
            }
        }
        if (pass == 0) {
            row_sums<1024, 2>(s, red, gen);
            m1 = s[0] / (float)cols;
            m2 = s[1] / (float)cols;
        }
    }
}

// Parameter gradients by columns: 64 chunks of 8 by the workgroup's NW waves, the rows dealt to
// `parts` workgroups and their waves in turn; one partial a workgroup, or (parts = 1) the result.
template <typename T, typename TR, bool DROP, int NW>
__device__ __forceinline__ void norm_param_columns(const NormArgs& a, int block, int which, int parts) {
    __shared__ float comb[(NW - 1) * 64 * 16];
    const int t = threadIdx.x & 63, part = threadIdx.x >> 6;
    const int64_t col = ((int64_t)block * 64 + t) * 8;
    const int valid = col < a.cols ? (int)(a.cols - col < 8 ? a.cols - col : 8) : 0;
    float s[2][8];
#pragma unroll
    for (int j = 0; j < 8; ++j) s[0][j] = 0.0f, s[1][j] = 0.0f;
    if (valid > 0)
        for (int64_t row = (int64_t)which * NW + part; row < a.rows; row += (int64_t)parts * NW) {
            const float mean = a.mean[row], rstd = a.rstd[row];
            float v[8], g[8];
            load8((const TR*)a.x + row * a.ldx + col, valid, v);
            load8((const T*)a.dy + row * a.lddy + col, valid, g);
            if constexpr (DROP && sizeof(TR) == 2)
                add_residual<TR>(a, row, col, valid,
                                 keep8((uint64_t)row * (uint32_t)((a.cols - 1) / 8 + 1) + (uint64_t)(col / 8), drop_key(a.rng), a.threshold), v);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                s[0][j] += g[j] * ((v[j] - mean) * rstd);
                s[1][j] += g[j];
            }
        }
    if (part > 0)
#pragma unroll
        for (int i = 0; i < 16; ++i) comb[((part - 1) * 16 + i) * 64 + t] = s[i >> 3][i & 7];
    __syncthreads();
    if (part > 0 || valid <= 0) return;
    for (int p = 0; p < NW - 1; ++p)
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i >> 3][i & 7] += comb[(p * 16 + i) * 64 + t];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        void* out = i ? a.db : a.dw;
        if (parts > 1)
            store8(a.partial + ((int64_t)which * 2 + i) * a.cols + col, valid, s[i]);
        else if (out && a.wf32)
            store8((float*)out + col, valid, s[i]);
        else if (out)
            store8((T*)out + col, valid, s[i]);
    }
}

template <typename T, typename TR, bool DROP, bool WG, int NT, int TPR, int CH>
__global__ __launch_bounds__(NT) void norm_backward_kernel(NormArgs a) {
    norm_backward_rows<T, TR, DROP, WG, NT, TPR, CH>(a, gridDim.x);
}

// Few rows: the workgroups past `groups` take the parameter gradients, which need a row's statistics
// but not its sums.  x and dy are read twice, from L2, and a second launch and its partials are
// saved (8 x 2048 float32 with the autograd around it: 80 -> 75 us).
template <typename T, typename TR, bool DROP, int NT, int TPR, int CH>
__global__ __launch_bounds__(NT) void norm_backward_few_kernel(NormArgs a, int groups) {
    if ((int)blockIdx.x < groups)
        norm_backward_rows<T, TR, DROP, false, NT, TPR, CH>(a, groups);
    else
        norm_param_columns<T, TR, DROP, NT / 64>(a, blockIdx.x - groups, 0, 1);
}

// Rows wider than kMaxHeldColsBackward
template <typename T, typename TR, bool DROP>
__global__ __launch_bounds__(256) void norm_param_long_kernel(NormArgs a) {
    norm_param_columns<T, TR, DROP, 4>(a, blockIdx.x, blockIdx.y, gridDim.y);
}

// partial [groups][2][cols] -> dw (blockIdx.z = 0), db (1).  64 columns a workgroup, its 16
// waves every 16th partial each, joined in wave order.
template <typename TW>
__global__ __launch_bounds__(1024) void norm_param_kernel(const float* __restrict__ partial, int groups, int cols,
                                                          TW* dw, TW* db) {
    __shared__ float comb[16 * 64];
    TW* out = blockIdx.z ? db : dw;
    if (!out) return;
    const int t = threadIdx.x & 63, wid = threadIdx.x >> 6;
    const int64_t col = block_id() * 64 + t;
    float s = 0.0f;
    if (col < cols) {
        const float* p = partial + (int64_t)blockIdx.z * cols + col;
#pragma unroll 4
        for (int g = wid; g < groups; g += 16) s += p[(int64_t)g * 2 * cols];
    }
    comb[wid * 64 + t] = s;
    __syncthreads();
    if (wid == 0 && col < cols) {
#pragma unroll
        for (int k = 1; k < 16; ++k) s += comb[k * 64 + t];
        out[col] = (TW)s;
    }
}

// ------------------------------------------------------------------------------ dispatch
template <typename TW> hipError_t norm_param(const float* partial, int groups, int cols, void* dw, void* db, hipStream_t s) {
    dim3 g = blocks(((int64_t)cols + 63) / 64);
    g.z = 2;
    norm_param_kernel<TW><<<g, 1024, 0, s>>>(partial, groups, cols, (TW*)dw, (TW*)db);
    return hipGetLastError();
}

template <typename T, typename TR, bool DROP>
hipError_t norm_forward(const NormArgs& a, hipStream_t s) {
#define OTF_NF(TPR, CH) norm_forward_kernel<T, TR, DROP, TPR, CH><<<grid, TPR > 256 ? TPR : 256, 0, s>>>(a)
    const int c = a.cols;
    // narrow rows share a wave: with 64 lanes a row of 64 columns, 7 of 8 lanes would idle
    const int per = c <= 64 ? 32 : c <= 128 ? 16 : c <= 256 ? 8 : c <= 2048 ? 4 : 1;
    const dim3 grid = blocks((a.rows + per - 1) / per);
    if (c <= 64)
        OTF_NF(8, 1);
    else if (c <= 128)
        OTF_NF(16, 1);
    else if (c <= 256)
        OTF_NF(32, 1);
    else if (c <= 512)
        OTF_NF(64, 1);
    else if (c <= 1024)
        OTF_NF(64, 2);
    else if (c <= 2048)
        OTF_NF(64, 4);
    else if (c <= 4096)
        OTF_NF(256, 2);
    else if (c <= 8192)
        OTF_NF(256, 4);
    else if (c <= 16384)
        OTF_NF(1024, 2);
    else if (c <= kMaxHeldCols)
        OTF_NF(1024, 4);
    else
        norm_forward_long_kernel<T, TR, DROP><<<grid, 1024, 0, s>>>(a);
#undef OTF_NF
    return hipGetLastError();
}

// Workgroups of the backward pass, each of which leaves one partial of dw and db.  Up to 2048
// columns a workgroup's row is short and its latency bounds: 1024 of them (4099 x 1531 float16: 27
// -> 25 us), until the partials' traffic counts (16384 x 2048 float32: 88 us, 82 with 512).
int norm_backward_groups(int64_t rows, int64_t cols) {
    const bool held = cols <= kMaxHeldColsBackward;
    const int64_t per = !held ? 64 : cols <= 64 ? 32 : cols <= 128 ? 16 : cols <= 256 ? 8 : cols <= 1024 ? 4 : 1;
    const int64_t most = !held ? 32 : cols > 8192 ? 256 : cols > 1024 && cols <= 2048 && rows < 8192 ? 1024 : 512;
    const int64_t want = (rows + per - 1) / per;
    return (int)(want < most ? want : most);
}

template <typename T, typename TR, bool DROP, bool WG>
hipError_t norm_backward_wg(const NormArgs& a, hipStream_t s) {
    const int c = a.cols, grid = norm_backward_groups(a.rows, c);
    const bool held = c <= kMaxHeldColsBackward;
    const bool few = WG && held && a.rows <= kFewRows;
    const int columns = (c - 1) / 512 + 1;
#define OTF_NB(NT, TPR, CH)                                                                                      \
    if (few)                                                                                                     \
        norm_backward_few_kernel<T, TR, DROP, NT, TPR, CH><<<grid + columns, NT, 0, s>>>(a, grid);               \
    else                                                                                                         \
        norm_backward_kernel<T, TR, DROP, WG, NT, TPR, CH><<<grid, NT, 0, s>>>(a)
    if (c <= 64) {
        OTF_NB(256, 8, 1);
    } else if (c <= 128) {
        OTF_NB(256, 16, 1);
    } else if (c <= 256) {
        OTF_NB(256, 32, 1);
    } else if (c <= 512) {
        OTF_NB(256, 64, 1);
    } else if (c <= 1024) {
        OTF_NB(256, 64, 2);
    } else if (c <= 2048) {
        OTF_NB(256, 256, 1);
    } else if (c <= 4096) {
        OTF_NB(256, 256, 2);
    } else if (c <= 8192) {
        OTF_NB(256, 256, 4);
    } else if (held) {
        OTF_NB(512, 512, 4);
    } else {
        norm_backward_long_kernel<T, TR, DROP><<<blocks(a.rows), 1024, 0, s>>>(a);
        if (WG) norm_param_long_kernel<T, TR, DROP><<<dim3((unsigned)((c - 1) / 512 + 1), (unsigned)grid), 256, 0, s>>>(a);
    }
#undef OTF_NB
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || !WG || few || grid == 1) return e;
    return a.wf32 ? norm_param<float>(a.partial, grid, c, a.dw, a.db, s) : norm_param<T>(a.partial, grid, c, a.dw, a.db, s);
}

template <typename T, typename TR, bool DROP>
hipError_t norm_backward(const NormArgs& a, hipStream_t s) {
    return a.dw || a.db ? norm_backward_wg<T, TR, DROP, true>(a, s) : norm_backward_wg<T, TR, DROP, false>(a, s);
}

template <typename T>
hipError_t dropout_launch(const void* x, int64_t ldx, const void* res, int64_t ldr, void* y, int64_t ldy,
                          int64_t rows, int64_t cols, uint32_t threshold, float scale, const int64_t* rng,
                          hipStream_t s) {
    const uint32_t groups = (uint32_t)((cols + 7) / 8);
    const uint64_t total = (uint64_t)rows * groups;
    const bool flat = cols % 8 == 0 && ldx == cols && ldy == cols && (!res || ldr == cols);
    const dim3 grid = blocks((int64_t)((total + 255) / 256));
#define OTF_DK(RES, FLAT)                                                                                     \
    dropout_kernel<T, RES, FLAT><<<grid, 256, 0, s>>>((const T*)x, ldx, (const T*)res, ldr, (T*)y, ldy, total, \
                                                      groups, (int)cols, rng, threshold, scale)
    if (res) {
        if (flat)
            OTF_DK(true, true);
        else
            OTF_DK(true, false);
    } else {
        if (flat)
            OTF_DK(false, true);
        else
            OTF_DK(false, false);
    }
#undef OTF_DK
    return hipGetLastError();
}

bool type16_or_32(int32_t t) { return t == OTF_F32 || t == OTF_F16 || t == OTF_BF16; }
size_t elem_size(int32_t t) { return t == OTF_F32 ? 4 : 2; }
bool elem_aligned(const void* p, int32_t t) { return (uintptr_t)p % elem_size(t) == 0; }

bool too_large(int64_t rows, int64_t cols) { return rows > INT32_MAX || cols > INT32_MAX - 8192; }   // the kernels' index types

// what every call here checks: sizes, types, parameters
int check_norm(int64_t rows, int64_t cols, int32_t dtype, int32_t rdtype, int32_t wdtype) {
    if (rows < 0 || cols <= 0) return OTF_EINVAL;
    if (!type16_or_32(dtype)) return OTF_EINVAL;
    if (rdtype != dtype && rdtype != OTF_F32) return OTF_EINVAL;
    if (wdtype != dtype && wdtype != OTF_F32) return OTF_EINVAL;
    if (too_large(rows, cols)) return OTF_EUNSUPPORTED;
    return OTF_OK;
}

template <bool DROP, typename F> int by_type(int32_t dtype, int32_t rdtype, F f) {
    hipError_t e;
    if (dtype == OTF_F32)
        e = f((float*)0, (float*)0);
    else if (dtype == OTF_F16)
        e = (DROP && rdtype == OTF_F32) ? f((_Float16*)0, (float*)0) : f((_Float16*)0, (_Float16*)0);
    else
        e = (DROP && rdtype == OTF_F32) ? f((__bf16*)0, (float*)0) : f((__bf16*)0, (__bf16*)0);
    return check_hip(e);
}

}  // namespace
}  // namespace otf

using namespace otf;

extern "C" {

int otf_dropout(const void* x, int64_t ldx, const void* residual, int64_t ldr, void* y, int64_t ldy, int64_t rows,
                int64_t cols, int32_t dtype, double p, const int64_t* rng, otf_stream_t stream) {
    uint32_t threshold;
    float scale;
    if (rows < 0 || cols < 0 || !type16_or_32(dtype) || !drop_params(p, threshold, scale)) return OTF_EINVAL;
    if (rows == 0 || cols == 0) return OTF_OK;
    if (!x || !y || (threshold && !rng) || ldx < cols || ldy < cols || (residual && ldr < cols)) return OTF_EINVAL;
    if (!elem_aligned(x, dtype) || !elem_aligned(y, dtype) || !elem_aligned(residual, dtype)) return OTF_EINVAL;
    if ((uintptr_t)rng % 8) return OTF_EINVAL;
    if (cols > INT32_MAX - 8 || rows > INT64_MAX / ((cols + 7) / 8)) return OTF_EUNSUPPORTED;
    if (rows * ((cols + 7) / 8) > (int64_t)1 << 42) return OTF_EUNSUPPORTED;   // of 8 elements each
    return by_type<false>(dtype, dtype, [&](auto* t, auto*) {
        using T = std::remove_pointer_t<decltype(t)>;
        return dropout_launch<T>(x, ldx, residual, ldr, y, ldy, rows, cols, threshold, scale, rng, (hipStream_t)stream);
    });
}

int otf_layer_norm(const void* x, int64_t ldx, int32_t dtype, const void* weight, const void* bias, int32_t wdtype,
                   double eps, int64_t rows, int64_t cols, void* y, int64_t ldy, float* mean, float* rstd,
                   otf_stream_t stream) {
    const int rc = check_norm(rows, cols, dtype, dtype, wdtype);
    if (rc != OTF_OK) return rc;
    if (!(eps >= 0.0) || (mean == nullptr) != (rstd == nullptr)) return OTF_EINVAL;
    if (rows == 0) return OTF_OK;
    if (!x || !y || ldx < cols || ldy < cols) return OTF_EINVAL;
    if (!elem_aligned(x, dtype) || !elem_aligned(y, dtype) || !elem_aligned(weight, wdtype) ||
        !elem_aligned(bias, wdtype) || !elem_aligned(mean, OTF_F32) || !elem_aligned(rstd, OTF_F32))
        return OTF_EINVAL;
    NormArgs a{};
    a.x = x, a.ldx = ldx, a.y = y, a.ldy = ldy, a.w = weight, a.b = bias, a.wf32 = wdtype == OTF_F32;
    a.mean = mean, a.rstd = rstd, a.rows = rows, a.cols = (int)cols, a.eps = (float)eps;
    return by_type<false>(dtype, dtype, [&](auto* t, auto*) {
        using T = std::remove_pointer_t<decltype(t)>;
        return norm_forward<T, T, false>(a, (hipStream_t)stream);
    });
}

int otf_dropout_add_layer_norm(const void* x, int64_t ldx, int32_t dtype, const void* residual, int64_t ldr,
                               int32_t rdtype, const void* weight, const void* bias, int32_t wdtype, double eps,
                               double p, const int64_t* rng, int64_t rows, int64_t cols, void* y, int64_t ldy,
                               void* z, int64_t ldz, float* mean, float* rstd, otf_stream_t stream) {
    const int rc = check_norm(rows, cols, dtype, rdtype, wdtype);
    if (rc != OTF_OK) return rc;
    NormArgs a{};
    if (!(eps >= 0.0) || (mean == nullptr) != (rstd == nullptr) || !drop_params(p, a.threshold, a.scale))
        return OTF_EINVAL;
    if (rows == 0) return OTF_OK;
    if (!x || !residual || !y || !z || (a.threshold && !rng)) return OTF_EINVAL;
    if (ldx < cols || ldr < cols || ldy < cols || ldz < cols) return OTF_EINVAL;
    if (!elem_aligned(x, dtype) || !elem_aligned(y, dtype) || !elem_aligned(residual, rdtype) ||
        !elem_aligned(z, rdtype) || !elem_aligned(weight, wdtype) || !elem_aligned(bias, wdtype) ||
        !elem_aligned(mean, OTF_F32) || !elem_aligned(rstd, OTF_F32) || (uintptr_t)rng % 8)
        return OTF_EINVAL;
    a.x = x, a.ldx = ldx, a.res = residual, a.ldr = ldr, a.y = y, a.ldy = ldy, a.z = z, a.ldz = ldz;
    a.w = weight, a.b = bias, a.wf32 = wdtype == OTF_F32, a.mean = mean, a.rstd = rstd, a.rng = rng;
    a.rows = rows, a.cols = (int)cols, a.eps = (float)eps;
    return by_type<true>(dtype, rdtype, [&](auto* t, auto* r) {
        using T = std::remove_pointer_t<decltype(t)>;
        using TR = std::remove_pointer_t<decltype(r)>;
        return norm_forward<T, TR, true>(a, (hipStream_t)stream);
    });
}

size_t otf_layer_norm_backward_workspace_size(int64_t rows, int64_t cols) {
    if (rows <= 0 || cols <= 0 || too_large(rows, cols)) return 0;
    if (cols <= kMaxHeldColsBackward && rows <= kFewRows) return 0;
    const int g = norm_backward_groups(rows, cols);
    return g > 1 ? (size_t)g * 2 * (size_t)cols * sizeof(float) : 0;
}

// shared by the two backward entry points
static int norm_backward_call(NormArgs& a, bool drop, int32_t dtype, int32_t rdtype, int32_t wdtype, int64_t rows,
                              int64_t cols, void* workspace, size_t workspace_bytes, otf_stream_t stream) {
    const int rc = check_norm(rows, cols, dtype, rdtype, wdtype);
    if (rc != OTF_OK) return rc;
    a.rows = rows, a.cols = (int)cols, a.wf32 = wdtype == OTF_F32, a.partial = (float*)workspace;
    hipStream_t s = (hipStream_t)stream;
    if (!elem_aligned(a.dw, wdtype) || !elem_aligned(a.db, wdtype) || !elem_aligned(a.w, wdtype)) return OTF_EINVAL;
    if (rows == 0) {   // no row: the sums are zero
        if (!a.dw && !a.db) return OTF_OK;
        // 0 is 0 in both 16-bit types
        return check_hip(a.wf32 ? norm_param<float>(nullptr, 0, (int)cols, a.dw, a.db, s) : norm_param<_Float16>(nullptr, 0, (int)cols, a.dw, a.db, s));
    }
    if (!a.x || !a.dy || !a.y || !a.mean || !a.rstd || a.ldx < cols || a.lddy < cols || a.ldy < cols) return OTF_EINVAL;
    if (!elem_aligned(a.x, rdtype) || !elem_aligned(a.dy, dtype) || !elem_aligned(a.y, dtype) ||
        !elem_aligned(a.z, rdtype) || !elem_aligned(a.mean, OTF_F32) ||
        !elem_aligned(a.rstd, OTF_F32))
        return OTF_EINVAL;
    const size_t need = (a.dw || a.db) ? otf_layer_norm_backward_workspace_size(rows, cols) : 0;
    if (need && (!workspace || workspace_bytes < need || (uintptr_t)workspace % 16)) return OTF_EINVAL;
    if (drop)
        return by_type<true>(dtype, rdtype, [&](auto* t, auto* r) {
            using T = std::remove_pointer_t<decltype(t)>;
            using TR = std::remove_pointer_t<decltype(r)>;
            return norm_backward<T, TR, true>(a, s);
        });
    return by_type<false>(dtype, dtype, [&](auto* t, auto*) {
        using T = std::remove_pointer_t<decltype(t)>;
        return norm_backward<T, T, false>(a, s);
    });
}

int otf_layer_norm_backward(const void* dy, int64_t lddy, const void* x, int64_t ldx, int32_t dtype,
                            const void* weight, int32_t wdtype, const float* mean, const float* rstd, int64_t rows,
                            int64_t cols, void* dx, int64_t lddx, void* dweight, void* dbias, void* workspace,
                            size_t workspace_bytes, otf_stream_t stream) {
    NormArgs a{};
    a.dy = dy, a.lddy = lddy, a.x = x, a.ldx = ldx, a.w = weight, a.mean = const_cast<float*>(mean);
    a.rstd = const_cast<float*>(rstd), a.y = dx, a.ldy = lddx, a.dw = dweight, a.db = dbias;
    return norm_backward_call(a, false, dtype, dtype, wdtype, rows, cols, workspace, workspace_bytes, stream);
}

int otf_dropout_add_layer_norm_backward(const void* dy, int64_t lddy, const void* dz, int64_t lddz, const void* z,
                                        int64_t ldz, const void* x, int64_t ldx, const void* residual, int64_t ldr,
                                        int32_t dtype, int32_t rdtype, const void* weight, int32_t wdtype,
                                        const float* mean, const float* rstd, double p, const int64_t* rng,
                                        int64_t rows, int64_t cols, void* dx, int64_t lddx, void* dresidual,
                                        int64_t lddr, void* dweight, void* dbias, void* workspace,
                                        size_t workspace_bytes, otf_stream_t stream) {
    NormArgs a{};
    if (!drop_params(p, a.threshold, a.scale)) return OTF_EINVAL;
    const bool again = rdtype != OTF_F32;
    if (rows > 0) {
        if ((a.threshold && !rng) || (uintptr_t)rng % 8 || !dresidual || lddr < cols || (dz && lddz < cols)) return OTF_EINVAL;
        if (again && (!residual || ldr < cols || !elem_aligned(residual, rdtype))) return OTF_EINVAL;
        if (!elem_aligned(dz, rdtype)) return OTF_EINVAL;
    }
    a.dy = dy, a.lddy = lddy, a.dz = dz, a.lddz = lddz, a.w = weight;
    a.x = again ? x : z, a.ldx = again ? ldx : ldz, a.res = residual, a.ldr = ldr;
    a.mean = const_cast<float*>(mean), a.rstd = const_cast<float*>(rstd), a.rng = rng;
    a.y = dx, a.ldy = lddx, a.z = dresidual, a.ldz = lddr, a.dw = dweight, a.db = dbias;
    return norm_backward_call(a, true, dtype, rdtype, wdtype, rows, cols, workspace, workspace_bytes, stream);
}

}  // extern "C"
