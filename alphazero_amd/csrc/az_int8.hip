// Matrix product in 8-bit integers with a scale for each token and each output channel (az_quantize_rows, az_int8_linear).
//
//   q_mk = rint(127 x_mk / max_k |x_mk|) (ties to even), s_m = max_k |x_mk| / 127
//   y_mn = s_m w_n sum_k q_mk Q_nk + b_n        (the sum in 32-bit integers: exact, whatever its order)
//
// Many tokens: the tile loop of az_gemm.cuh, bound by the matrix instructions and LDS (8192^3 in 430 to 520 us by card, 2.1 to 2.5 POP/s,
// quantising 42 to 50 us). Few tokens (up to 48): bound by the bytes of Q, which stream from memory to registers once.
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
    int64_t q_pitch;    // bytes
    int64_t pad;        // columns to write, those behind the last one as zeros
    float* scale;
};

// A lane's share of a row at a time: 16 bytes of the input. It may start anywhere; columns behind the last one are zero.
template <int DT> struct Chunk {
    static constexpr int N = DT == DT_F32 ? 4 : 8;
};
template <int DT>
__device__ __forceinline__ void load_chunk(const void* x, int64_t base, int64_t c, int cols, float (&v)[Chunk<DT>::N]) {
    constexpr int NV = Chunk<DT>::N;
    if (c + NV <= cols) {
        if constexpr (DT == DT_F32) {
            __builtin_memcpy(v, (const float*)x + base + c, 16);
        } else {
            uint32_t u[4];
            __builtin_memcpy(u, (const uint16_t*)x + base + c, 16);
#pragma unroll
            for (int k = 0; k < 4; ++k) v[2 * k] = from_bits<DT>((uint16_t)u[k]), v[2 * k + 1] = from_bits<DT>((uint16_t)(u[k] >> 16));
        }
    } else {
#pragma unroll
        for (int e = 0; e < NV; ++e) v[e] = c + e < cols ? load_scalar<DT>(x, base + c + e) : 0.0f;
    }
}
// The largest magnitude, as bits: unsigned order puts infinities and NaN above every number.
__device__ __forceinline__ uint32_t larger(uint32_t top, float v) {
    const uint32_t u = __builtin_bit_cast(uint32_t, v) & 0x7fffffffu;
    return u > top ? u : top;
}
__device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) { return a > b ? a : b; }
struct Range {
    float top, inv;      // largest magnitude; 127 / top, or 0 where that has no use (zero, not finite, next to the smallest numbers)
    __device__ __forceinline__ explicit Range(uint32_t bits) : top(__builtin_bit_cast(float, bits)), inv(top >= 1e-30f && top < INFINITY ? 127.0f / top : 0.0f) {}
    __device__ __forceinline__ float scale() const { return top < INFINITY ? top / 127.0f : NAN; }     // NaN for NaN too
};

// The nearest whole numbers of the real quotients 127 v / top, ties to even, four to a word. Adding 1.5 * 2^23 in the multiply-add leaves
// the whole number in the low bits. The product is off by less than 127 * 2^-23 (the reciprocal's rounding), so only where the
// remainder comes within 2e-5 of a half does a division in 64 bits (127 v is exact there) decide.
template <int NV>
__device__ __forceinline__ void quantize_chunk(const float (&v)[NV], const Range& g, uint32_t (&u)[NV / 4]) {
    constexpr float MAGIC = 12582912.0f;
    uint32_t b[NV];
    float far = 0.0f;
#pragma unroll
    for (int e = 0; e < NV; ++e) {
        const float t = __builtin_fmaf(v[e], g.inv, MAGIC);
        far = fmaxf(far, fabsf(__builtin_fmaf(v[e], g.inv, MAGIC - t)));
        b[e] = __builtin_bit_cast(uint32_t, t);
    }
    if (far >= 0.49998f || g.inv == 0.0f) {
#pragma unroll
        for (int e = 0; e < NV; ++e) b[e] = g.top < INFINITY && g.top > 0.0f ? (uint32_t)(int)rint(127.0 * (double)v[e] / (double)g.top) : 0u;
    }
#pragma unroll
    for (int w = 0; w < NV / 4; ++w)
        u[w] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(b[4 * w + 3], b[4 * w + 2], 0x0c0c0400u), __builtin_amdgcn_perm(b[4 * w + 1], b[4 * w], 0x0c0c0400u), 0x05040100u);
}

// LANES threads per row (up to 64, or a workgroup), HELD chunks per thread stay in registers between the maximum and the quotients; a longer row is read again (from
// L2). Up to 64 lanes the maximum needs no barrier. Bound by memory: 8192 x 8192 bfloat16 in 42 us (4.8 TB/s).
template <int DT, int LANES, int HELD>
__global__ __launch_bounds__(LANES < 256 ? 256 : LANES) void k_quantize(QuantArgs a) {
    static_assert(LANES <= 64 || LANES >= 256, "the waves of a row are a workgroup");
    constexpr int NV = Chunk<DT>::N, THREADS = LANES < 256 ? 256 : LANES, ROWS = THREADS / LANES;
    const int lane = threadIdx.x % LANES;
    const int64_t row = (int64_t)blockIdx.x * ROWS + threadIdx.x / LANES, base = row * a.pitch;
    if (ROWS > 1 && row >= a.rows) return;
    uint32_t top = 0;
    float v[HELD][NV];
#pragma unroll
    for (int h = 0; h < HELD; ++h) load_chunk<DT>(a.x, base, (h * LANES + lane) * NV, a.cols, v[h]);
#pragma unroll
    for (int h = 0; h < HELD; ++h)
#pragma unroll
        for (int e = 0; e < NV; ++e) top = larger(top, v[h][e]);
    for (int64_t c = (int64_t)(HELD * LANES + lane) * NV; c < a.cols; c += LANES * NV) {
        float u[NV];
        load_chunk<DT>(a.x, base, c, a.cols, u);
#pragma unroll
        for (int e = 0; e < NV; ++e) top = larger(top, u[e]);
    }
#pragma unroll
    for (int o = 1; o < (LANES < 64 ? LANES : 64); o *= 2) top = larger(top, (uint32_t)__shfl_xor((int)top, o));
    if constexpr (LANES > 64) {
        __shared__ uint32_t tops[LANES / 64];
        if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = top;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < LANES / 64; ++w) top = larger(top, tops[w]);
    }
    const Range range(top);
    if (lane == 0) a.scale[row] = range.scale();
    auto store = [&](int64_t c, const float (&f)[NV]) {
        uint32_t u[NV / 4];
        quantize_chunk(f, range, u);
        int8_t* o = a.q + row * a.q_pitch + c;
        if (c + NV <= a.pad) {
            __builtin_memcpy(o, u, NV);      // may start anywhere
        } else {
            for (int e = 0; e < NV; ++e)
                if (c + e < a.pad) o[e] = (int8_t)(u[e >> 2] >> (8 * (e & 3)));
        }
    };
#pragma unroll
    for (int h = 0; h < HELD; ++h) {
        const int64_t c = (h * LANES + lane) * NV;
        if (c < a.pad) store(c, v[h]);
    }
    for (int64_t c = (int64_t)(HELD * LANES + lane) * NV; c < a.pad; c += LANES * NV) {
        float u[NV];
        load_chunk<DT>(a.x, base, c, a.cols, u);
        store(c, u);
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
    int piece = 0, tp, tq;
    if (a.splits == 1) {
        mm_place(blockIdx.x, a.tiles_p, a.tiles_q, tp, tq);
    } else {
        mm_place_piece(blockIdx.x, a.splits, a.tiles_p, a.tiles_q, piece, tp, tq);
    }
    const int64_t p0 = (int64_t)tp * T::BP, q0 = (int64_t)tq * T::BQ;
    typename T::acc_t acc[T::FP][T::FQ];
    const int steps = (a.kbytes + 127) >> 7, first = piece * a.per, last = first + a.per < steps ? first + a.per : steps;
    mm_tile<T>(a.w, a.x, p0, q0, a.kbytes, first, last, 1, lds, acc);
    const int lane = mm_lane_after(), wave = threadIdx.x >> 6, wp = wave / T::WQ, wq = wave % T::WQ;
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
#ifdef __HIP_DEVICE_COMPILE__
    const int ml = wp * T::TP + (lane >> 4) * 4;
    const int64_t here = a.s.channels - p0;
    float b[T::FP][4];
    auto load = [&](auto type) {
        constexpr int BT = decltype(type)::value;
        const AxisView bias((const char*)a.s.bias + p0 * (BT == DT_F32 ? 4 : 2), here * (BT == DT_F32 ? 4 : 2));
#pragma unroll
        for (int i = 0; i < T::FP; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) b[i][r] = bias.one<BT>(ml + i * 16 + r);
    };
    if (!a.s.bias) {
#pragma unroll
        for (int i = 0; i < T::FP; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) b[i][r] = 0.0f;
    } else if (a.s.bias_dtype == DT_F32) load(std::integral_constant<int, DT_F32>{});
    else if (a.s.bias_dtype == DT_BF16) load(std::integral_constant<int, DT_BF16>{});
    else load(std::integral_constant<int, DT_F16>{});
    const AxisView ws(a.s.w + p0, here);
#pragma unroll
    for (int i = 0; i < T::FP; ++i) {
        const f32x4 w = ws.four(ml + i * 16);
#pragma unroll
        for (int j = 0; j < T::FQ; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) v[i][j][r] = (float)acc[i][j][r] * sx[j] * w[r] + b[i][r];
    }
#endif
    if constexpr (DT == DT_F32) {       // 16 bytes per lane already
#pragma unroll
        for (int j = 0; j < T::FQ; ++j) {
            const int64_t n = q0 + wq * T::TQ + j * 16 + (lane & 15);
            if (n >= a.s.tokens) continue;
#pragma unroll
            for (int i = 0; i < T::FP; ++i) {
                const int64_t m = p0 + wp * T::TP + i * 16 + (lane >> 4) * 4;
                float* o = (float*)a.s.y + n * a.s.channels + m;
                if (m + 4 <= a.s.channels) {
                    __builtin_memcpy(o, &v[i][j], 16);
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
        mm_unstage<T, T::BQ, T::BP>(lds, (char*)a.s.y + (q0 * a.s.channels + p0) * 2, (int64_t)a.s.channels * 2, a.s.tokens - q0, (a.s.channels - p0) * 2);
    }
}

// Joins the pieces of k: thread t of block (tile, fragment) adds what thread t of each piece's workgroup left.
template <class T, int DT>
__global__ __launch_bounds__(T::THREADS) void k_int8_join(TileArgs a) {
    const int tiles = a.tiles_p * a.tiles_q, tile = blockIdx.x / (T::FP * T::FQ), f = blockIdx.x % (T::FP * T::FQ);
    const int tp = tile / a.tiles_q, tq = tile % a.tiles_q, i = f / T::FQ, j = f % T::FQ;
    i32x4 sum = {};
#pragma unroll 8
    for (int p = 0; p < a.splits; ++p) sum += a.part[(((int64_t)p * tiles + tile) * (T::FP * T::FQ) + f) * T::THREADS + threadIdx.x];
    const int lane = mm_lane_after(), wave = threadIdx.x >> 6, wp = wave / T::WQ, wq = wave % T::WQ;
    finish4<DT>(a.s, (int64_t)tq * T::BQ + wq * T::TQ + j * 16 + (lane & 15), (int64_t)tp * T::BP + wp * T::TP + i * 16 + (lane >> 4) * 4, sum);
}

struct FewArgs {
    const int8_t* w;
    const void* x;          // int8 rows, or the floating ones (DX)
    int64_t w_pitch, x_pitch;   // elements
    int32_t cols, share;
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

// Up to 16 * MT tokens, for which the weights' bytes are what counts. A workgroup is 16 waves; `share` of them take the same 16 channels
// and go through k in turns of 64 bytes, straight from memory to the matrix instruction's registers (lane: channel or token lane & 15,
// 16 bytes of k), U turns' loads before the first product. Rows may start anywhere. Channels and tokens behind the last one repeat it
// and are not written.
// Floating tokens (DX, one to FUSED_TOKENS of them) are quantised by every workgroup for itself, into LDS, while its first weights
// are on the way: one launch, with the values and the sums of two. One token, 4096 -> 16384: 14.3 us against 17.5 us.
constexpr int FEW_TOKENS = 48, FUSED_TOKENS = 2, FUSED_BYTES = 32768, DT_I8 = AZ_DT_I8;
// Channels of a wave in fragments of 16: two for each token fragment read from memory, as long as the sums fit.
constexpr int few_fragments(bool fused, int mt) { return !fused && mt <= 2 ? 2 : 1; }
template <int DT, int DX, int MT>
__global__ __launch_bounds__(1024) void k_int8_few(FewArgs a) {
    constexpr bool FUSED = DX != DT_I8;
    constexpr int CT = few_fragments(FUSED, MT), U = MT == 1 ? (CT == 1 ? 8 : 4) : 2;
    __shared__ i32x4 joint[16][CT][MT][64];
    __shared__ __align__(16) int8_t q[FUSED ? FUSED_BYTES : 16];
    __shared__ uint32_t tops[FUSED_TOKENS][16];
    __shared__ float scales[FUSED_TOKENS];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, turn = wave % a.share;
    const int64_t m0 = ((int64_t)blockIdx.x * (16 / a.share) + wave / a.share) * (16 * CT);
    const int8_t* wr[CT];
#pragma unroll
    for (int i = 0; i < CT; ++i) {
        const int64_t m = m0 + i * 16 + (lane & 15);
        wr[i] = a.w + (m < a.s.channels ? m : a.s.channels - 1) * a.w_pitch;
    }
    const int step = a.share * 64, own = (lane >> 4) * 16, pitch = (a.cols + 63) / 64 * 64;
    // 16 bytes at k of a row, in one load without a branch: where the row ends before they do its last 16, for which the weights become
    // zero; the bytes of a last piece that is not whole come by themselves after the loop
    const bool vector = a.cols >= 16;
    auto bytes = [&](const int8_t* row, int k) {
        i32x4 v;
        __builtin_memcpy(&v, row + (k + 16 <= a.cols ? k : a.cols - 16), 16);
        return v;
    };
    int k0 = turn * 64;
    i32x4 w[U][CT];
    auto weights = [&] {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int k = k0 + u * step + own;
#pragma unroll
            for (int i = 0; i < CT; ++i) {
                w[u][i] = bytes(wr[i], k);
                if (k + 16 > a.cols) w[u][i] = i32x4{0, 0, 0, 0};
            }
        }
    };
    if (vector && k0 < a.cols) weights();
    if constexpr (FUSED) {
        constexpr int NV = Chunk<DX>::N;
        for (int n = 0; n < a.s.tokens; ++n) {
            uint32_t top = 0;
            for (int c = threadIdx.x * NV; c < a.cols; c += 1024 * NV) {
                float v[NV];
                load_chunk<DX>(a.x, n * a.x_pitch, c, a.cols, v);
#pragma unroll
                for (int e = 0; e < NV; ++e) top = larger(top, v[e]);
            }
#pragma unroll
            for (int o = 1; o < 64; o *= 2) top = larger(top, (uint32_t)__shfl_xor((int)top, o));
            if (lane == 0) tops[n][wave] = top;
        }
        __syncthreads();
        for (int n = 0; n < a.s.tokens; ++n) {
            uint32_t top = 0;
#pragma unroll
            for (int v = 0; v < 16; ++v) top = larger(top, tops[n][v]);
            const Range range(top);
            if (threadIdx.x == 0) scales[n] = range.scale();
            for (int c = threadIdx.x * NV; c < pitch; c += 1024 * NV) {
                float v[NV];
                uint32_t u[NV / 4];
                load_chunk<DX>(a.x, n * a.x_pitch, c, a.cols, v);
                quantize_chunk(v, range, u);
                __builtin_memcpy(__builtin_assume_aligned(q + n * pitch + c, NV), u, NV);
            }
        }
        __syncthreads();
    }
    const int8_t* xr[MT];
    i32x4 acc[CT][MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        const int n = t * 16 + (lane & 15), in = n < a.s.tokens ? n : a.s.tokens - 1;
        xr[t] = FUSED ? q + in * pitch : (const int8_t*)a.x + in * a.x_pitch;
#pragma unroll
        for (int i = 0; i < CT; ++i) acc[i][t] = i32x4{};
    }
    for (; vector && k0 < a.cols; k0 += U * step) {
        i32x4 x[U][MT];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                const int k = k0 + u * step + own;
                if constexpr (FUSED) x[u][t] = *(const i32x4*)(xr[t] + (k < pitch ? k : 0));
                else x[u][t] = bytes(xr[t], k);
            }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < CT; ++i)
#pragma unroll
                for (int t = 0; t < MT; ++t) acc[i][t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[u][i], x[u][t], acc[i][t], 0, 0, 0);
        if (k0 + U * step < a.cols) {
            k0 += U * step;
            weights();
            k0 -= U * step;
        }
    }
    const int rest = a.cols / 64 * 64 + own;         // where a piece that is not whole could be
    if ((a.cols & 15) && turn == a.cols / 64 % a.share) {
        i32x4 x[MT];
#pragma unroll
        for (int t = 0; t < MT; ++t) x[t] = FUSED ? *(const i32x4*)(xr[t] + (rest < pitch ? rest : 0)) : bytes16(xr[t], rest, a.cols);
#pragma unroll
        for (int i = 0; i < CT; ++i) {
            const i32x4 v = rest + 16 > a.cols ? bytes16(wr[i], rest, a.cols) : i32x4{0, 0, 0, 0};
#pragma unroll
            for (int t = 0; t < MT; ++t) acc[i][t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(v, x[t], acc[i][t], 0, 0, 0);
        }
    }
#pragma unroll
    for (int i = 0; i < CT; ++i)
#pragma unroll
        for (int t = 0; t < MT; ++t) joint[wave][i][t][lane] = acc[i][t];
    __syncthreads();
    Scales s = a.s;
    if (FUSED) s.x = scales;
    for (int f = turn; f < CT * MT; f += a.share) {
        const int i = f / MT, t = f % MT;
        i32x4 sum = {};
        for (int v = 0; v < a.share; ++v) sum += joint[wave - turn + v][i][t][lane];
        finish4<DT>(s, t * 16 + (lane & 15), m0 + i * 16 + (lane >> 4) * 4, sum);
    }
}

// ------------------------------------------------------------------------------------------------ host side
typedef MmTile<256, 256, 2, 4, 2, MM_I8> Big;
typedef MmTile<128, 128, 2, 2, 2, MM_I8> Mid;
typedef MmTile<64, 64, 2, 2, 4, MM_I8> Small;
constexpr int MOST_THREADS = Big::THREADS;
static_assert(Mid::THREADS <= MOST_THREADS && Small::THREADS <= MOST_THREADS, "");

struct Plan {
    bool few, fused, align_w, align_x;
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
    auto crooked = [&](const void* q, int64_t pitch) { return (((uintptr_t)q | (uintptr_t)pitch) & 15) != 0 || pitch > MM_MAX_PITCH; };
    const bool copy = crooked(a.weight, a.weight_pitch);
    // Where the kernel for few tokens takes the place of the tiles. From 16384 channels on the tiles fill the chip in one walk (one int8 token,
    // 1024 -> 32000: 8.3 us against 13.6; 4096 -> 32000: 23.6 against 27). Below, they join pieces of k in a second launch (16 x 4096 ->
    // 4096: 11.4 against 9.2, 16 x 4096 -> 8000 13.1 against 9.6, 48 x 1024 -> 4096 8.7 against 7.5), which pays with more tokens and with
    // longer walks (32 x 4096 -> 1024 8.7 against 10.7, 16 x 8192 -> 1024 10 against 14, 64 x 4096 -> 32000 24.8 against 76). A weight that the
    // tiles have to copy: 4 x 4095 -> 4096 22 against 24, 32 x 4095 -> 4096 23 against 36. A weight that they read in place, its rows ending
    // inside 16 bytes, meets this kernel's byte-by-byte end of a row: tiles (floating tokens, few against tiles: 3 x 162 -> 82 7.5 and 6.2, 16 x
    // 722 -> 362 14.3 and 8.1, 48 x 2047 -> 4096 14.9 and 13.0), but for up to 4 int8 tokens, which the tiles would have to copy (4 x 162 -> 82
    // 4.6 and 5.8, 4 x 4095 -> 4096 12.4 and 12.5, though 4 x 722 -> 362 9.2 and 7.0).
    // One or two floating tokens are quantised in the same launch wherever they fit its LDS, against quantising and tiles (us, weights that lie
    // in the last-level cache): 1 x 4096 -> 4096 8.4 and 12.7, 1 x 1024 -> 16000 8.5 and 8.1, 1 x 4096 -> 16384 14.5 and 16.6, 2 x 4096 ->
    // 24576 22.6 and 23.2, 1 x 1024 -> 131072 27.4 and 30.7, 1 x 8192 -> 65536 122 and 135, 1 x 14336 -> 4096 16 and 20.5; of 32 shapes up to
    // 128 times as wide as long the tiles won at three by more than 5 % (1 x 722 -> 362 10.8 and 9.8, 2 x 1024 -> 16384 9.4 and 8.4, 2 x
    // 3584 -> 18944 21 and 19.1). Four tokens 14336 -> 4096: 29 against 25.
    const bool small = a.channels < 16384;
    const bool ragged = (a.features & 15) != 0;
    const int most = copy || (ragged && a.x_dtype == AZ_DT_I8) ? 4 : ragged ? 0 : a.features <= 2048 ? FEW_TOKENS : 16;
    p.few = small && a.features <= 4096 && a.tokens <= most;
    p.fused = a.x_dtype != AZ_DT_I8 && a.tokens <= FUSED_TOKENS && a.tokens * round_up(a.features, 64) <= FUSED_BYTES;
    if (p.fused) return p;
    if (a.x_dtype != AZ_DT_I8) {
        p.q = p.take(a.tokens * p.kpitch);
        p.scale = p.take(a.tokens * 4);
    }
    if (p.few) return p;
    p.align_w = copy;
    // A weight's row may end inside its last 16 bytes: what lies behind it meets the zeros behind a token's last feature, which quantising or
    // copying the token puts there. So one of the two is copied where features are not a multiple of 16, and that is the tokens.
    p.align_x = a.x_dtype == AZ_DT_I8 && (crooked(a.x, a.x_pitch) || ragged);
    if (p.align_w) p.w = p.take(a.channels * p.kpitch);
    if (p.align_x) p.x = p.take(a.tokens * p.kpitch);
    auto tiles = [&](int64_t e) { return ((a.channels + e - 1) / e) * ((a.tokens + e - 1) / e); };
    const int steps = (int)((p.kpitch + 127) / 128);
    p.edge = mm_tile_edge(a.channels, a.tokens, steps);
    p.per = steps;
    if (p.edge == 64) {      // split k until there is a workgroup per compute unit with at least 4 steps, or two with 24 (128 x 14336 -> 4096: 22 us, one: 25)
        int64_t s = 512 / tiles(64);
        if (s * 24 > steps) s = 256 / tiles(64);
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
    if (a->tokens > (1 << 30) || a->channels > (1 << 27)) return fail(AZ_ERR_ARG, "tokens are at most 2^30, channels 2^27");
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

// Two to four chunks per lane: more hold fewer rows in flight. From 2048 rows on a short row gets no more lanes than hold it (262144 x 64
// bfloat16: 17 us, with 256 lanes 270; 32768 x 2048: 40 against 54); with fewer rows more lanes are the shorter wait (256 x 2048: 3.6 us, with
// 64 lanes 5.4). Long rows: 1024 x 23104 bfloat16 21 us with 1024 lanes of three chunks, 33 with eight; 1024 x 14336 float32 14 with four,
// 21 with eight. What does not fit is read twice (1024 x 23104 float32: 22 us with four of six chunks held, 26 with all).
template <int DT>
void launch_quantize(const QuantArgs& q, hipStream_t st) {
    const int64_t bytes = (int64_t)q.cols * (DT == DT_F32 ? 4 : 2);
    auto run = [&](auto lanes, auto held) {
        constexpr int LANES = decltype(lanes)::value, HELD = decltype(held)::value, THREADS = LANES < 256 ? 256 : LANES, ROWS = THREADS / LANES;
        hipLaunchKernelGGL((k_quantize<DT, LANES, HELD>), dim3((unsigned)((q.rows + ROWS - 1) / ROWS)), dim3(THREADS), 0, st, q);
    };
    const std::integral_constant<int, 2> two;
    const std::integral_constant<int, 4> four;
    const std::integral_constant<int, 64> wave;
    const std::integral_constant<int, 256> group;
    const std::integral_constant<int, 1024> all;
    const bool many = q.rows >= 2048;
    if (many && bytes <= 256) run(std::integral_constant<int, 8>{}, two);
    else if (many && bytes <= 512) run(std::integral_constant<int, 16>{}, two);
    else if (many && bytes <= 1024) run(std::integral_constant<int, 32>{}, two);
    else if (many && bytes <= 2048) run(wave, two);
    else if (many && bytes <= 4096) run(wave, four);
    else if (bytes <= 8192) run(group, two);
    else if (bytes <= 16384) run(group, four);
    else if (bytes <= 32768) run(std::integral_constant<int, 512>{}, four);
    else if (bytes <= 49152) run(all, std::integral_constant<int, 3>{});
    else run(all, four);
}
template <int DT>
void quantize_as(const QuantArgs& q, hipStream_t st) {
    constexpr int64_t MOST = int64_t(1) << 21;      // rows of a launch, which holds fewer than 2^32 threads
    for (int64_t r = 0; r < q.rows; r += MOST) {
        QuantArgs part = q;
        part.x = (const char*)q.x + r * q.pitch * (DT == DT_F32 ? 4 : 2);
        part.q += r * q.q_pitch;
        part.scale += r;
        part.rows = q.rows - r < MOST ? q.rows - r : MOST;
        launch_quantize<DT>(part, st);
    }
}
void quantize(int dtype, const QuantArgs& q, hipStream_t st) {
    if (dtype == AZ_DT_F32) quantize_as<DT_F32>(q, st);
    else if (dtype == AZ_DT_BF16) quantize_as<DT_BF16>(q, st);
    else quantize_as<DT_F16>(q, st);
}

template <class T, int DT>
void run_tiles(const TileArgs& t, hipStream_t st) {
    hipLaunchKernelGGL((k_int8_tile<T, DT>), dim3((unsigned)(t.tiles_p * t.tiles_q * t.splits)), dim3(T::THREADS), 0, st, t);
}

// Up to FEW_TOKENS tokens. The waves of a workgroup that share 16 channels are as many as leave one round of workgroups: with up to 16 tokens
// a compute unit holds one (80 registers in 16 waves), and a second round for the last few doubles the time (1 x 4096 -> 6000 bfloat16: 8.3
// us, with 375 workgroups of more sharing 14.3; 16 x 2048 -> 16000 int8 8.5 and 14.4). With more tokens it holds two, and one round of 256 is
// as fast as one of 512 (48 x 2048 -> 8192 10.4 and 10.2, 48 x 512 -> 16000 7.4 and 10.4).
template <int DT, int DX>
int few(const az_int8_args& a, const void* x, int64_t x_pitch, const Scales& s, hipStream_t st) {
    auto run = [&](auto tokens) {
        constexpr int MT = decltype(tokens)::value, WIDE = 16 * few_fragments(DX != DT_I8, MT);
        const int64_t groups = (a.channels + WIDE - 1) / WIDE;
        int share = 16;
        while (share > 1 && groups * share > 256 * 16) share /= 2;
        const FewArgs f{(const int8_t*)a.weight, x, a.weight_pitch, x_pitch, (int)a.features, share, s};
        hipLaunchKernelGGL((k_int8_few<DT, DX, MT>), dim3((unsigned)((groups * share + 15) / 16)), dim3(1024), 0, st, f);
    };
    if (DX != DT_I8 || a.tokens <= 16) run(std::integral_constant<int, 1>{});
    else if constexpr (DX == DT_I8) {
        if (a.tokens <= 32) run(std::integral_constant<int, 2>{});
        else run(std::integral_constant<int, 3>{});
    }
    return launched("k_int8_few");
}

template <int DT>
int fused(const az_int8_args& a, const Scales& s, hipStream_t st) {
    if (a.x_dtype == AZ_DT_F32) return few<DT, DT_F32>(a, a.x, a.x_pitch, s, st);
    if (a.x_dtype == AZ_DT_BF16) return few<DT, DT_BF16>(a, a.x, a.x_pitch, s, st);
    return few<DT, DT_F16>(a, a.x, a.x_pitch, s, st);
}

template <int DT>
int product(const az_int8_args& a, const Plan& p, const int8_t* x, int64_t x_pitch, const Scales& s, char* ws, hipStream_t st) {
    if (p.few) return few<DT, DT_I8>(a, x, x_pitch, s, st);
    const int8_t* w = (const int8_t*)a.weight;
    int64_t w_pitch = a.weight_pitch;
    auto align = [&](const int8_t* src, int64_t pitch, int64_t rows, int64_t at) {
        const int64_t most = (int64_t(1) << 31) / (p.kpitch >> 4);      // rows of a launch, which holds fewer than 2^32 threads
        for (int64_t r = 0; r < rows; r += most) {
            const int64_t n = rows - r < most ? rows - r : most;
            hipLaunchKernelGGL(k_align, dim3((unsigned)((n * (p.kpitch >> 4) + 255) / 256)), dim3(256), 0, st, src + r * pitch, pitch, n, (int)a.features,
                               (int8_t*)(ws + at) + r * p.kpitch, p.kpitch);
        }
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
    // the last row is read up to the 4 bytes that hold its last feature
    t.w = MmOperand{(const char*)w, w_pitch, 0, (int)a.channels, p.align_w ? 0 : (int)(p.kpitch - a.features) & ~3};
    t.s = s;
    t.kbytes = (int)p.kpitch;
    t.tiles_p = (int)((a.channels + p.edge - 1) / p.edge);
    t.splits = p.splits;
    t.per = p.per;
    t.part = p.part >= 0 ? (i32x4*)(ws + p.part) : nullptr;
    const int64_t most = ((int64_t(1) << 31) / MOST_THREADS / t.tiles_p) * p.edge;      // tokens of a launch, which holds fewer than 2^32 threads
    for (int64_t r = 0; r < a.tokens; r += most) {
        const int64_t n = a.tokens - r < most ? a.tokens - r : most;
        t.x = MmOperand{(const char*)x + r * x_pitch, x_pitch, 0, (int)n};
        t.s.x = s.x + r;
        t.s.y = (char*)s.y + r * a.channels * (DT == DT_F32 ? 4 : 2);
        t.s.tokens = (int)n;
        t.tiles_q = (int)((n + p.edge - 1) / p.edge);
        if (p.edge == 256) run_tiles<Big, DT>(t, st);
        else if (p.edge == 128) run_tiles<Mid, DT>(t, st);
        else run_tiles<Small, DT>(t, st);
    }
    if (t.splits > 1)      // few tiles, one launch
        hipLaunchKernelGGL((k_int8_join<Small, DT>), dim3((unsigned)(t.tiles_p * t.tiles_q * Small::FP * Small::FQ)), dim3(Small::THREADS), 0, st, t);
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
    quantize(dtype, QuantArgs{x, pitch, (int)cols, rows, q, q_pitch, cols, scale}, (hipStream_t)stream);
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
    if (p.fused) {
        if (a.y_dtype == AZ_DT_F32) return fused<DT_F32>(a, s, st);
        if (a.y_dtype == AZ_DT_BF16) return fused<DT_BF16>(a, s, st);
        return fused<DT_F16>(a, s, st);
    }
    const int8_t* x = (const int8_t*)a.x;
    int64_t x_pitch = a.x_pitch;
    if (a.x_dtype != AZ_DT_I8) {
        quantize(a.x_dtype, QuantArgs{a.x, a.x_pitch, (int)a.features, a.tokens, (int8_t*)(ws + p.q), p.kpitch, p.kpitch, (float*)(ws + p.scale)}, st);
        if (const int rc = launched("k_quantize")) return rc;
        x = (const int8_t*)(ws + p.q);
        x_pitch = p.kpitch;
        s.x = (const float*)(ws + p.scale);
    }
    if (a.y_dtype == AZ_DT_F32) return product<DT_F32>(a, p, x, x_pitch, s, ws, st);
    if (a.y_dtype == AZ_DT_BF16) return product<DT_BF16>(a, p, x, x_pitch, s, ws, st);
    return product<DT_F16>(a, p, x, x_pitch, s, ws, st);
}
