// Matrix product in 8-bit integers with a scale for each token and each output channel (az_quantize_rows, az_int8_linear).
//
//   q_mk = rint(127 x_mk / max_k |x_mk|) (ties to even), s_m = max_k |x_mk| / 127
//   y_mn = s_m w_n sum_k q_mk Q_nk + b_n        (the sum in 32-bit integers: exact, whatever its order)
//
// Many tokens: the tile loop of az_gemm.cuh, bound by the matrix instructions. Few tokens (up to 64): bound by the bytes of Q, which
// stream from memory to registers once.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <string>

#include "../../include/azamd.h"
#include "az_gemm.cuh"
#include "az_types.cuh"

namespace az {
int fail(int code, const std::string& msg);

namespace {

int64_t round_up(int64_t a, int64_t b) { return (a + b - 1) / b * b; }

// ------------------------------------------------------------------------------------------------ quantisation
struct QuantArgs {
    const void* x;
    int64_t pitch;      // elements
    int32_t cols;
    int64_t rows;
    int8_t* q;
    int64_t q_pitch;    // bytes; behind the last column zeros up to the pitch rounded down to 16
    float* scale;
};

// One workgroup per row: the maximum, then the quotients (the second read of the row comes from L1 / L2).
// The nearest whole number of the real quotient 127 x / max: the product with the reciprocal is off by less than 127 * 2^-23, so
// only where it comes within 1e-4 of a half does a division in 64 bits (127 x exact there) decide.
template <int DT>
__global__ __launch_bounds__(256) void k_quantize(QuantArgs a) {
    __shared__ float tops[4];
    const int64_t row = blockIdx.x;
    const int64_t base = row * a.pitch;
    constexpr int V = DT == DT_F32 ? 4 : 8;
    const bool wide = (((uintptr_t)a.x & 15) == 0) && (a.pitch % V == 0);
    float top = 0.0f;
    auto see = [&](float v) {
        v = fabsf(v);
        top = v > top || v != v ? v : top;      // a NaN stays
    };
    auto load = [&](int c, float (&v)[16]) {    // 16 columns from c on
        if (wide && c + 16 <= a.cols) {
            if constexpr (DT == DT_F32) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float4 f = *(const float4*)((const float*)a.x + base + c + 4 * e);
                    v[4 * e] = f.x, v[4 * e + 1] = f.y, v[4 * e + 2] = f.z, v[4 * e + 3] = f.w;
                }
            } else {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const uint4 f = *(const uint4*)((const uint16_t*)a.x + base + c + 8 * e);
                    const uint32_t u[4] = {f.x, f.y, f.z, f.w};
#pragma unroll
                    for (int k = 0; k < 4; ++k) v[8 * e + 2 * k] = from_bits<DT>((uint16_t)u[k]), v[8 * e + 2 * k + 1] = from_bits<DT>((uint16_t)(u[k] >> 16));
                }
            }
        } else {
#pragma unroll
            for (int e = 0; e < 16; ++e) v[e] = c + e < a.cols ? load_scalar<DT>(a.x, base + c + e) : 0.0f;
        }
    };
    float v[16];
    for (int c = threadIdx.x * 16; c < a.cols; c += 4096) {
        load(c, v);
#pragma unroll
        for (int e = 0; e < 16; ++e) see(v[e]);
    }
#pragma unroll
    for (int o = 1; o < 64; o *= 2) see(__shfl_xor(top, o));
    if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 4; ++w) see(tops[w]);
    const bool finite = top < INFINITY;          // false for NaN
    if (threadIdx.x == 0) a.scale[row] = finite ? top / 127.0f : NAN;
    const float inv = top >= 1e-30f ? 127.0f / top : 0.0f;
    const int64_t q_cols = a.q_pitch / 16 * 16;
    const bool whole = (((uintptr_t)a.q | (uintptr_t)a.q_pitch) & 15) == 0;
    for (int c = threadIdx.x * 16; c < a.cols; c += 4096) {
        load(c, v);
        int8_t q[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const float y = v[e] * inv, n = rintf(y);
            int r = (int)n;
            if (!(fabsf(y - n) < 0.4999f) || inv == 0.0f) r = finite && top > 0.0f ? (int)rint(127.0 * (double)v[e] / (double)top) : 0;
            q[e] = (int8_t)r;
        }
        if (whole && c + 16 <= q_cols) *(uint4*)(a.q + row * a.q_pitch + c) = *(const uint4*)q;
        else
            for (int e = 0; e < 16; ++e)
                if (c + e < a.cols) a.q[row * a.q_pitch + c + e] = q[e];
    }
}

// Rows of bytes into rows of whole 16 bytes, for weights whose rows start anywhere.
__global__ __launch_bounds__(256) void k_align(const int8_t* src, int64_t src_pitch, int64_t rows, int cols, int8_t* dst, int64_t pitch) {
    const int64_t pieces = pitch >> 4, at = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (at >= rows * pieces) return;
    const int64_t r = at / pieces;
    const int c = (int)(at - r * pieces) * 16;
    int8_t v[16];
    if (c + 16 <= cols) __builtin_memcpy(v, src + r * src_pitch + c, 16);
    else
        for (int e = 0; e < 16; ++e) v[e] = c + e < cols ? src[r * src_pitch + c + e] : (int8_t)0;
    *(uint4*)(dst + at * 16) = *(const uint4*)v;
}

// ------------------------------------------------------------------------------------------------ products
struct Scales {
    const float *x, *w;     // per token, per channel
    const void* bias;       // of the output's type, or null
    int32_t bias_dtype;
    void* y;                // [tokens][channels]
    int32_t tokens, channels;
};

__device__ __forceinline__ float bias_at(const Scales& s, int64_t m) {
    if (!s.bias) return 0.0f;
    return s.bias_dtype == DT_F32 ? load_scalar<DT_F32>(s.bias, m) : s.bias_dtype == DT_BF16 ? load_scalar<DT_BF16>(s.bias, m) : load_scalar<DT_F16>(s.bias, m);
}

// Four neighbouring channels of a token.
template <int DT>
__device__ __forceinline__ void finish4(const Scales& s, int64_t n, int64_t m, const i32x4& sum) {
    if (n >= s.tokens) return;
    const float sx = s.x[n];
    float v[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const int64_t c = m + r < s.channels ? m + r : s.channels - 1;
        v[r] = (float)sum[r] * sx * s.w[c] + bias_at(s, c);
    }
    const int64_t at = n * s.channels + m;
    if ((s.channels & 3) == 0) {
        if (m < s.channels) store4<DT>(s.y, at, v[0], v[1], v[2], v[3]);
    } else {
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (m + r < s.channels) store_scalar<DT>(s.y, at + r, v[r]);
    }
}

struct TileArgs {
    MmOperand w, x;
    Scales s;
    int32_t kbytes, tiles_p, tiles_q, splits, per;   // k in `splits` pieces of `per` steps; with more than one, sums go to part
    i32x4* part;                                     // [splits][tiles][THREADS][FP * FQ] as the lanes hold them
};

template <class T, int DT>
__global__ __launch_bounds__(T::THREADS) void k_int8_tile(TileArgs a) {
    __shared__ __align__(16) char lds[T::LDS];
    const int tiles = a.tiles_p * a.tiles_q;
    const int piece = blockIdx.x / tiles;
    int tp, tq;
    mm_place(blockIdx.x - piece * tiles, a.tiles_p, a.tiles_q, tp, tq);
    const int64_t p0 = (int64_t)tp * T::BP, q0 = (int64_t)tq * T::BQ;
    typename T::acc_t acc[T::FP][T::FQ];
    const int steps = (a.kbytes + 127) >> 7, first = piece * a.per, last = first + a.per < steps ? first + a.per : steps;
    mm_tile<T>(a.w, a.x, p0, q0, a.kbytes, first, last, false, lds, acc);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wp = wave / T::WQ, wq = wave % T::WQ;
    if (a.splits > 1) {
        i32x4* o = a.part + (((int64_t)piece * tiles + tp * a.tiles_q + tq) * (T::FP * T::FQ)) * T::THREADS + threadIdx.x;
#pragma unroll
        for (int i = 0; i < T::FP; ++i)
#pragma unroll
            for (int j = 0; j < T::FQ; ++j) o[(i * T::FQ + j) * T::THREADS] = acc[i][j];
        return;
    }
    float sx[T::FQ];
#pragma unroll
    for (int j = 0; j < T::FQ; ++j) {
        const int64_t n = q0 + wq * T::TQ + j * 16 + (lane & 15);
        sx[j] = a.s.x[n < a.s.tokens ? n : a.s.tokens - 1];
    }
    f32x4 v[T::FP][T::FQ];
#pragma unroll
    for (int i = 0; i < T::FP; ++i) {
        float w[4], b[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int64_t m = p0 + wp * T::TP + i * 16 + (lane >> 4) * 4 + r, c = m < a.s.channels ? m : a.s.channels - 1;
            w[r] = a.s.w[c];
            b[r] = bias_at(a.s, c);
        }
#pragma unroll
        for (int j = 0; j < T::FQ; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) v[i][j][r] = (float)acc[i][j][r] * sx[j] * w[r] + b[r];
    }
    if constexpr (DT == DT_F32) {       // 16 bytes per lane already
#pragma unroll
        for (int j = 0; j < T::FQ; ++j) {
            const int64_t n = q0 + wq * T::TQ + j * 16 + (lane & 15);
            if (n >= a.s.tokens) continue;
#pragma unroll
            for (int i = 0; i < T::FP; ++i) {
                const int64_t m = p0 + wp * T::TP + i * 16 + (lane >> 4) * 4;
                float* o = (float*)a.s.y + n * a.s.channels + m;
                if ((a.s.channels & 3) == 0) {
                    if (m < a.s.channels) *(f32x4*)o = v[i][j];
                } else {
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (m + r < a.s.channels) o[r] = v[i][j][r];
                }
            }
        }
    } else {
        mm_stage<T>(lds, [&](int i, int j) { return pack4<DT>(v[i][j][0], v[i][j][1], v[i][j][2], v[i][j][3]); });
        __syncthreads();
        mm_unstage<T, T::BQ, T::BP>(lds, (char*)a.s.y + (q0 * a.s.channels + p0) * 2, (int64_t)a.s.channels * 2, a.s.tokens - q0, (a.s.channels - p0) * 2,
                                    (a.s.channels & 7) == 0);
    }
}

// Joins the pieces of k: thread t of block (tile, fragment) adds what thread t of each piece's workgroup left.
template <class T, int DT>
__global__ __launch_bounds__(T::THREADS) void k_int8_join(TileArgs a) {
    const int tiles = a.tiles_p * a.tiles_q, tile = blockIdx.x / (T::FP * T::FQ), f = blockIdx.x % (T::FP * T::FQ);
    const int tp = tile / a.tiles_q, tq = tile % a.tiles_q, i = f / T::FQ, j = f % T::FQ;
    i32x4 sum = {};
    for (int p = 0; p < a.splits; ++p) sum += a.part[(((int64_t)p * tiles + tile) * (T::FP * T::FQ) + f) * T::THREADS + threadIdx.x];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wp = wave / T::WQ, wq = wave % T::WQ;
    finish4<DT>(a.s, (int64_t)tq * T::BQ + wq * T::TQ + j * 16 + (lane & 15), (int64_t)tp * T::BP + wp * T::TP + i * 16 + (lane >> 4) * 4, sum);
}

struct FewArgs {
    const int8_t *w, *x;
    int64_t w_pitch, x_pitch;
    int32_t cols;
    Scales s;
};

__device__ __forceinline__ i32x4 bytes16(const int8_t* row, int k, int cols) {
    i32x4 v = {0, 0, 0, 0};
    if (k + 16 <= cols) __builtin_memcpy(&v, row + k, 16);
    else if (k < cols) {
        uint32_t u[4] = {0, 0, 0, 0};
#pragma unroll
        for (int e = 0; e < 16; ++e)
            if (k + e < cols) u[e >> 2] |= (uint32_t)(uint8_t)row[k + e] << (8 * (e & 3));
        v = i32x4{(int)u[0], (int)u[1], (int)u[2], (int)u[3]};
    }
    return v;
}

// Up to 16 * MT tokens: a workgroup takes 16 channels, its waves take k in turns of 64 bytes, straight from memory to the matrix
// instruction's registers (lane: channel lane & 15, 16 bytes of k). Nothing is read twice but the tokens.
template <int DT, int MT>
__global__ __launch_bounds__(1024) void k_int8_few(FewArgs a) {
    __shared__ i32x4 joint[16][MT][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
    const int64_t m0 = (int64_t)blockIdx.x * 16;
    const int64_t m = m0 + (lane & 15) < a.s.channels ? m0 + (lane & 15) : a.s.channels - 1;
    const int8_t* wr = a.w + m * a.w_pitch;
    i32x4 acc[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) acc[t] = i32x4{};
    for (int k0 = wave * 64; k0 < a.cols; k0 += waves * 64) {
        const int k = k0 + (lane >> 4) * 16;
        const i32x4 w = bytes16(wr, k, a.cols);
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            const int n = t * 16 + (lane & 15);
            const i32x4 x = n < a.s.tokens ? bytes16(a.x + n * a.x_pitch, k, a.cols) : i32x4{};
            acc[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w, x, acc[t], 0, 0, 0);
        }
    }
#pragma unroll
    for (int t = 0; t < MT; ++t) joint[wave][t][lane] = acc[t];
    __syncthreads();
    for (int t = wave; t < MT; t += waves) {
        i32x4 sum = {};
        for (int v = 0; v < waves; ++v) sum += joint[v][t][lane];
        finish4<DT>(a.s, t * 16 + (lane & 15), m0 + (lane >> 4) * 4, sum);
    }
}

// ------------------------------------------------------------------------------------------------ host side
typedef MmTile<256, 256, 2, 4, MM_I8> Big;
typedef MmTile<128, 128, 2, 2, MM_I8> Mid;
typedef MmTile<64, 64, 2, 2, MM_I8> Small;

struct Plan {
    bool few, align_w, align_x;
    int edge = 64, splits = 1, per = 0;
    int64_t kpitch;
    int64_t q = -1, scale = -1, w = -1, x = -1, part = -1, bytes = 0;
    int64_t take(int64_t n) {
        const int64_t at = bytes;
        bytes += round_up(n, 256);
        return at;
    }
};

Plan plan_of(const az_int8_args& a) {
    Plan p;
    p.kpitch = round_up(a.features, 16);
    p.few = a.tokens <= 64;
    if (a.x_dtype != AZ_DT_I8) {
        p.q = p.take(a.tokens * p.kpitch);
        p.scale = p.take(a.tokens * 4);
    }
    if (p.few) return p;
    auto crooked = [&](const void* q, int64_t pitch) { return (((uintptr_t)q | (uintptr_t)pitch) & 15) != 0 || (a.features & 15) != 0 || pitch > MM_MAX_PITCH; };
    p.align_w = crooked(a.weight, a.weight_pitch);
    p.align_x = a.x_dtype == AZ_DT_I8 && crooked(a.x, a.x_pitch);
    if (p.align_w) p.w = p.take(a.channels * p.kpitch);
    if (p.align_x) p.x = p.take(a.tokens * p.kpitch);
    auto tiles = [&](int64_t e) { return ((a.channels + e - 1) / e) * ((a.tokens + e - 1) / e); };
    p.edge = tiles(256) >= 192 ? 256 : tiles(128) >= 192 ? 128 : 64;
    const int steps = (int)((p.kpitch + 127) / 128);
    p.per = steps;
    if (p.edge == 64) {      // split k until there are two workgroups per compute unit, with at least 4 steps each
        int64_t s = 512 / tiles(64);
        if (s > steps / 4) s = steps / 4;
        if (s > 1) {
            p.per = (int)((steps + s - 1) / s);
            p.splits = (steps + p.per - 1) / p.per;
            if (p.splits > 1) p.part = p.take((int64_t)p.splits * tiles(64) * 64 * 64 * 4);
        }
    }
    return p;
}

int check_args(const az_int8_args* a) {
    if (!a) return fail(AZ_ERR_ARG, "null argument");
    if (a->x_dtype != AZ_DT_F32 && a->x_dtype != AZ_DT_BF16 && a->x_dtype != AZ_DT_F16 && a->x_dtype != AZ_DT_I8)
        return fail(AZ_ERR_ARG, "x is float32, bfloat16, float16 or int8");
    for (const int32_t d : {a->y_dtype, a->bias ? a->bias_dtype : (int32_t)AZ_DT_F32})
        if (d != AZ_DT_F32 && d != AZ_DT_BF16 && d != AZ_DT_F16) return fail(AZ_ERR_ARG, "the output and the bias are float32, bfloat16 or float16");
    if (a->tokens < 1 || a->features < 1 || a->channels < 1) return fail(AZ_ERR_ARG, "tokens, features and channels are at least 1");
    if (a->tokens > (1 << 30) || a->channels > (1 << 30)) return fail(AZ_ERR_ARG, "tokens and channels are at most 2^30");
    if (a->features > 131071) return fail(AZ_ERR_ARG, "features are at most 131071: 2^31 / 128^2 products fill a 32-bit sum");
    if (!a->x || !a->weight || !a->weight_scale || !a->y || (a->x_dtype == AZ_DT_I8 && !a->x_scale)) return fail(AZ_ERR_ARG, "null argument");
    if (a->x_pitch < a->features || a->weight_pitch < a->features) return fail(AZ_ERR_ARG, "a row stride is smaller than the row");
    if ((uintptr_t)a->y & 15) return fail(AZ_ERR_ARG, "the output starts at a multiple of 16 bytes");
    return AZ_OK;
}

int launched(const char* what) {
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? AZ_OK : fail(AZ_ERR_HIP, std::string(what) + ": " + hipGetErrorString(e));
}

void quantize(int dtype, const QuantArgs& q, hipStream_t st) {
    const dim3 grid((unsigned)q.rows), block(256);
    if (dtype == AZ_DT_F32) hipLaunchKernelGGL((k_quantize<DT_F32>), grid, block, 0, st, q);
    else if (dtype == AZ_DT_BF16) hipLaunchKernelGGL((k_quantize<DT_BF16>), grid, block, 0, st, q);
    else hipLaunchKernelGGL((k_quantize<DT_F16>), grid, block, 0, st, q);
}

template <class T, int DT>
void run_tiles(const TileArgs& t, hipStream_t st) {
    const unsigned tiles = (unsigned)(t.tiles_p * t.tiles_q);
    hipLaunchKernelGGL((k_int8_tile<T, DT>), dim3(tiles * t.splits), dim3(T::THREADS), 0, st, t);
    if (t.splits > 1) hipLaunchKernelGGL((k_int8_join<T, DT>), dim3(tiles * T::FP * T::FQ), dim3(T::THREADS), 0, st, t);
}

template <int DT>
int product(const az_int8_args& a, const Plan& p, const int8_t* x, int64_t x_pitch, const Scales& s, char* ws, hipStream_t st) {
    if (p.few) {
        // waves of a workgroup share its 16 channels' k: as many as it takes to have 8 per compute unit, 16 at most
        const int64_t groups = (a.channels + 15) / 16;
        int waves = 4;
        while (waves < 16 && groups * waves < 2048 && waves * 64 < a.features) waves *= 2;
        const FewArgs f{(const int8_t*)a.weight, x, a.weight_pitch, x_pitch, (int)a.features, s};
        const dim3 grid((unsigned)groups), block(waves * 64);
        if (a.tokens <= 16) hipLaunchKernelGGL((k_int8_few<DT, 1>), grid, block, 0, st, f);
        else if (a.tokens <= 32) hipLaunchKernelGGL((k_int8_few<DT, 2>), grid, block, 0, st, f);
        else hipLaunchKernelGGL((k_int8_few<DT, 4>), grid, block, 0, st, f);
        return launched("k_int8_few");
    }
    const int8_t* w = (const int8_t*)a.weight;
    int64_t w_pitch = a.weight_pitch;
    auto align = [&](const int8_t* src, int64_t pitch, int64_t rows, int64_t at) {
        hipLaunchKernelGGL(k_align, dim3((unsigned)((rows * (p.kpitch >> 4) + 255) / 256)), dim3(256), 0, st, src, pitch, rows, (int)a.features, (int8_t*)(ws + at), p.kpitch);
    };
    if (p.align_w) {
        align(w, w_pitch, a.channels, p.w);
        w = (const int8_t*)(ws + p.w);
        w_pitch = p.kpitch;
    }
    if (p.align_x) {
        align(x, x_pitch, a.tokens, p.x);
        x = (const int8_t*)(ws + p.x);
        x_pitch = p.kpitch;
    }
    TileArgs t{};
    t.w = MmOperand{(const char*)w, w_pitch, 0, (int)a.channels};
    t.x = MmOperand{(const char*)x, x_pitch, 0, (int)a.tokens};
    t.s = s;
    t.kbytes = (int)p.kpitch;
    t.tiles_p = (int)((a.channels + p.edge - 1) / p.edge);
    t.tiles_q = (int)((a.tokens + p.edge - 1) / p.edge);
    t.splits = p.splits;
    t.per = p.per;
    t.part = p.part >= 0 ? (i32x4*)(ws + p.part) : nullptr;
    if (p.edge == 256) run_tiles<Big, DT>(t, st);
    else if (p.edge == 128) run_tiles<Mid, DT>(t, st);
    else run_tiles<Small, DT>(t, st);
    return launched("k_int8_tile");
}

}  // namespace
}  // namespace az

using namespace az;

extern "C" int az_quantize_rows(const void* x, int32_t dtype, int64_t rows, int64_t cols, int64_t pitch, int8_t* q, int64_t q_pitch, float* scale,
                                void* stream) {
    if (dtype != AZ_DT_F32 && dtype != AZ_DT_BF16 && dtype != AZ_DT_F16) return fail(AZ_ERR_ARG, "dtype is float32, bfloat16 or float16");
    if (rows < 0 || cols < 1 || rows > (1 << 30) || cols > (1 << 30)) return fail(AZ_ERR_ARG, "rows are 0..2^30, cols 1..2^30");
    if (pitch < cols || q_pitch < cols) return fail(AZ_ERR_ARG, "a row stride is smaller than the row");
    if (rows == 0) return AZ_OK;
    if (!x || !q || !scale) return fail(AZ_ERR_ARG, "null argument");
    quantize(dtype, QuantArgs{x, pitch, (int)cols, rows, q, q_pitch, scale}, (hipStream_t)stream);
    return launched("k_quantize");
}

extern "C" int64_t az_int8_workspace(const az_int8_args* args) {
    if (const int rc = check_args(args)) return rc;
    return plan_of(*args).bytes;
}

extern "C" int az_int8_linear(const az_int8_args* args, void* workspace, int64_t workspace_bytes, void* stream) {
    if (const int rc = check_args(args)) return rc;
    const az_int8_args& a = *args;
    const Plan p = plan_of(a);
    if (p.bytes && (!workspace || workspace_bytes < p.bytes || ((uintptr_t)workspace & 255)))
        return fail(AZ_ERR_ARG, "workspace too small or not at a multiple of 256");
    hipStream_t st = (hipStream_t)stream;
    char* ws = (char*)workspace;
    Scales s{a.x_scale, a.weight_scale, a.bias, a.bias_dtype, a.y, (int)a.tokens, (int)a.channels};
    const int8_t* x = (const int8_t*)a.x;
    int64_t x_pitch = a.x_pitch;
    if (a.x_dtype != AZ_DT_I8) {
        quantize(a.x_dtype, QuantArgs{a.x, a.x_pitch, (int)a.features, a.tokens, (int8_t*)(ws + p.q), p.kpitch, (float*)(ws + p.scale)}, st);
        if (const int rc = launched("k_quantize")) return rc;
        x = (const int8_t*)(ws + p.q);
        x_pitch = p.kpitch;
        s.x = (const float*)(ws + p.scale);
    }
    if (a.y_dtype == AZ_DT_F32) return product<DT_F32>(a, p, x, x_pitch, s, ws, st);
    if (a.y_dtype == AZ_DT_BF16) return product<DT_BF16>(a, p, x, x_pitch, s, ws, st);
    return product<DT_F16>(a, p, x, x_pitch, s, ws, st);
}
