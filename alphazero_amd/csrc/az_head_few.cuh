// The loss of a linear layer for few rows (up to 16, float32 forward up to 32; few_forward and few_backward say where): what counts is how
// often the weight goes through memory.
//
// Forward: the weight streams once, from memory to the matrix instructions' registers, with no copy and no LDS in between; rows may
// start anywhere. float32 uses the float32 matrix instruction (0.16 PFLOP/s, which is more than the memory feeds with 16 rows).
// 1 x 4096 -> 131072 bfloat16: 187 us (5.7 TB/s); 5 x 3765 -> 52111 float32: 219 to 233 us by card (3.4 to 3.6 TB/s).
// Backward: the logits are made again the same way and become G [classes][16] in float32; then one pass reads the weight, adds G W
// to dx in registers and writes dW = G^T x. That is three reads of the weight in all and one write of its gradient.
// Included by az_head.cuh.
#pragma once

namespace az {
namespace {

constexpr int FEW_GRAD_ROWS = 16, FEW_CLASSES = 32;   // classes of a wave: two 16-class fragments for each one of x

struct FewArgs {
    const void *w, *x, *bias;
    int64_t w_pitch, x_pitch;     // elements
    int32_t cols, share;          // `share` waves of a workgroup's 16 split the features of the same classes
    Rows t;
    f32x4* part;                  // [rows][workgroups]
    float *tpart, *zt;
    float *un_w, *un_x;           // float32, [workgroups]: unscale_of the largest values, which a backward pass with tiles divides transposed copies by
    const float *ref, *inv, *mean, *tsum, *grad, *scalars;   // gradient
    int32_t each, mean_of;
    float* g;                     // [classes][16 * MT]
};

// 16 bytes of a row from element k on.
template <int DT> struct FewType {
    static constexpr int SIZE = DT == DT_F32 ? 4 : 2, PIECE = 16 / SIZE, TURN = 4 * PIECE;
};
template <int DT>
__device__ __forceinline__ i32x4 few_rest(const char* row, int k, int cols) {     // the elements that are left
    constexpr int SIZE = FewType<DT>::SIZE;
    uint32_t u[4] = {0, 0, 0, 0};
#pragma unroll
    for (int e = 0; e < FewType<DT>::PIECE; ++e)
        if (k + e < cols) {
            if constexpr (SIZE == 4) u[e] = ((const uint32_t*)row)[k + e];
            else u[e >> 1] |= (uint32_t)((const uint16_t*)row)[k + e] << (16 * (e & 1));
        }
    return i32x4{(int)u[0], (int)u[1], (int)u[2], (int)u[3]};
}
template <int DT>
__device__ __forceinline__ f32x4 few_mfma(i32x4 w, i32x4 x, f32x4 c) {
    if constexpr (DT == DT_F32) {
        // element e of every lane in turn: any order of the features will do, as long as both operands have the same
        const f32x4 fw = __builtin_bit_cast(f32x4, w), fx = __builtin_bit_cast(f32x4, x);
#pragma unroll
        for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(fw[e], fx[e], c, 0, 0, 0);
        return c;
    } else {
        return mm_mfma<DT == DT_F16 ? MM_F16 : MM_BF16>(w, x, c);
    }
}

// o joined with v, whichever reference is larger.
__device__ __forceinline__ void few_join(Part& o, const Part& v) {
    Part s = {reference_size(v.ref) > reference_size(o.ref) ? v.ref : o.ref, 0.0f, 0.0f, 0.0f, 0.0f};
    join_part(s, o);
    join_part(s, v);
    o = s;
}

// A workgroup goes through groups of 16 / share * 32 classes with a stride of the grid. GRAD: writes G, else sums parts.
template <int DT, int MT, bool GRAD>
__global__ __launch_bounds__(1024) void k_ce_few(FewArgs a) {
    constexpr int CT = FEW_CLASSES / 16, U = MT == 1 ? 4 : 2, PIECE = FewType<DT>::PIECE, TURN = FewType<DT>::TURN, SIZE = FewType<DT>::SIZE;
    __shared__ f32x4 joint[16][CT][MT][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, turn = wave % a.share, own = (lane >> 4) * PIECE, step = a.share * TURN;
    const int64_t per = 16 / a.share * FEW_CLASSES;
    const bool vector = a.cols >= PIECE, dense = a.t.dense != nullptr, entropy = a.t.entropy != 0.0f || !GRAD;
    const char* xr[MT];
    i32x4 on[MT];         // all bits for a row that counts
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        const int n = t * 16 + (lane & 15), row = n < a.t.rows ? n : a.t.rows - 1;
        xr[t] = (const char*)a.x + row * a.x_pitch * SIZE;
        const int m = dense || a.t.index[row] != a.t.ignore ? -1 : 0;
        on[t] = i32x4{m, m, m, m};
    }
    auto bytes = [&](const char* row, int k) {
        i32x4 v;
        __builtin_memcpy(&v, row + (int64_t)(k + PIECE <= a.cols ? k : a.cols - PIECE) * SIZE, 16);
        return v;
    };
    uint32_t most_w = 0, most_x = 0;
    auto see = [](uint32_t& most, i32x4 v) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const uint32_t u = (uint32_t)v[e] & 0x7fffffffu;
            most = u > most ? u : most;
        }
    };
    Part st[MT];
    float abs_sum[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        st[t] = Part{-INFINITY, 0.0f, 0.0f, 0.0f, 0.0f};
        abs_sum[t] = 0.0f;
    }
    for (int64_t group = blockIdx.x; group * per < a.t.classes; group += gridDim.x) {
        const int64_t c0 = group * per + wave / a.share * FEW_CLASSES;
        const char* wr[CT];
        f32x4 acc[CT][MT];
#pragma unroll
        for (int i = 0; i < CT; ++i) {
            const int64_t c = c0 + i * 16 + (lane & 15);
            wr[i] = (const char*)a.w + (c < a.t.classes ? c : a.t.classes - 1) * a.w_pitch * SIZE;
#pragma unroll
            for (int t = 0; t < MT; ++t) acc[i][t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        }
        for (int k0 = turn * TURN; vector && k0 < a.cols; k0 += U * step) {
            i32x4 w[U][CT], x[U][MT];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int k = k0 + u * step + own;
#pragma unroll
                for (int i = 0; i < CT; ++i) w[u][i] = bytes(wr[i], k);
#pragma unroll
                for (int t = 0; t < MT; ++t) x[u][t] = bytes(xr[t], k);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                // behind the row's end both are its last ones again: made zero, both, by a mask (a choice would put the loads into branches)
                const int m = k0 + u * step + own + PIECE <= a.cols ? -1 : 0;
                const i32x4 mask = {m, m, m, m};
                if constexpr (DT == DT_F32 && !GRAD) {
#pragma unroll
                    for (int i = 0; i < CT; ++i) see(most_w, w[u][i]);
#pragma unroll
                    for (int t = 0; t < MT; ++t) see(most_x, x[u][t] & on[t]);
                }
#pragma unroll
                for (int i = 0; i < CT; ++i)
#pragma unroll
                    for (int t = 0; t < MT; ++t) acc[i][t] = few_mfma<DT>(w[u][i] & mask, x[u][t] & mask, acc[i][t]);
            }
        }
        if (a.cols % PIECE && turn == a.cols / TURN % a.share) {
            const int k = a.cols / TURN * TURN + own;
            const bool in = k < a.cols && k + PIECE > a.cols;
#pragma unroll
            for (int i = 0; i < CT; ++i) {
                const i32x4 w = in ? few_rest<DT>(wr[i], k, a.cols) : i32x4{0, 0, 0, 0};
                if constexpr (DT == DT_F32 && !GRAD) see(most_w, w);
#pragma unroll
                for (int t = 0; t < MT; ++t) {
                    const i32x4 x = in ? few_rest<DT>(xr[t], k, a.cols) : i32x4{0, 0, 0, 0};
                    if constexpr (DT == DT_F32 && !GRAD) see(most_x, x & on[t]);
                    acc[i][t] = few_mfma<DT>(w, x, acc[i][t]);
                }
            }
        }
        __syncthreads();      // the group before has been read
#pragma unroll
        for (int i = 0; i < CT; ++i)
#pragma unroll
            for (int t = 0; t < MT; ++t) joint[wave][i][t][lane] = acc[i][t];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < CT; ++i)
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                if ((i * MT + t) % a.share != turn) continue;
                f32x4 z = {0.0f, 0.0f, 0.0f, 0.0f};
                for (int v = 0; v < a.share; ++v) z += joint[wave - turn + v][i][t][lane];
                const int64_t m = c0 + i * 16 + (lane >> 4) * 4;
                const int n = t * 16 + (lane & 15);
                const bool row = n < a.t.rows;
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (m + r >= a.t.classes) z[r] = -INFINITY;
                    else if (a.bias) z[r] += load_scalar<DT>(a.bias, m + r);
                const int64_t target = row && !dense ? a.t.index[n] : -1;
                float pi[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                if (dense && row)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (m + r < a.t.classes) pi[r] = a.t.dense[n * a.t.dense_pitch + m + r];
                if constexpr (!GRAD) {
                    const float top = fmaxf(fmaxf(z[0], z[1]), fmaxf(z[2], z[3]));
                    Part v = {reference_of(top), 0.0f, 0.0f, 0.0f, 0.0f};
                    const Reference at(top == -INFINITY ? 0.0f : v.ref);
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const float q = at.t(z[r]), e = __builtin_amdgcn_exp2f(q);
                        v.l += e;
                        v.s += e == 0.0f ? 0.0f : e * q;
                        v.pi += pi[r];
                        abs_sum[t] += fabsf(pi[r]);
                        v.dot += pi[r] == 0.0f ? 0.0f : pi[r] * q;
                        if (target == m + r && target < a.t.classes) a.zt[n] = z[r];
                    }
                    few_join(st[t], v);
                } else {
                    const bool counts = row && (dense || target != a.t.ignore);
                    float f = 0.0f, total = 1.0f;
                    if (counts) {
                        f = a.each ? a.grad[n] : a.grad[0];
                        if (a.mean_of) f /= a.scalars[0];
                        if (dense) total = a.tsum[n];
                        else if (target < 0 || target >= a.t.classes) f = NAN;
                    }
                    const Reference at(row ? a.ref[n] : 0.0f);
                    const float inv = row ? a.inv[n] : 0.0f, mean = row ? a.mean[n] : 0.0f, most = most_of(inv);
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const float q = fminf(at.t(z[r]), most), e = __builtin_amdgcn_exp2f(q);
                        float g = e * (inv * total) - pi[r];
                        if (target == m + r) g -= 1.0f;
                        if (entropy && e != 0.0f) g += a.t.entropy * LN2 * inv * e * (q - mean);
                        if (m + r < a.t.classes) a.g[(m + r) * (16 * MT) + n] = counts ? g * f : 0.0f;
                    }
                }
            }
    }
    if constexpr (!GRAD) {
        // lanes 16 apart hold the same row; then the waves, through LDS
        __syncthreads();
        if constexpr (DT == DT_F32) {
            __shared__ uint32_t most[2][16];
#pragma unroll
            for (int o = 1; o < 64; o *= 2) {
                const uint32_t u = (uint32_t)__shfl_xor((int)most_w, o), v = (uint32_t)__shfl_xor((int)most_x, o);
                most_w = u > most_w ? u : most_w;
                most_x = v > most_x ? v : most_x;
            }
            if (lane == 0) most[0][wave] = most_w, most[1][wave] = most_x;
            __syncthreads();
            if (threadIdx.x == 0) {
                for (int v = 1; v < 16; ++v) {
                    most_w = most[0][v] > most_w ? most[0][v] : most_w;
                    most_x = most[1][v] > most_x ? most[1][v] : most_x;
                }
                a.un_w[blockIdx.x] = unscale_of(__builtin_bit_cast(float, most_w));
                a.un_x[blockIdx.x] = unscale_of(__builtin_bit_cast(float, most_x));
            }
        }
        float* const rows = (float*)joint;      // [16 waves][16 MT][6]
#pragma unroll
        for (int t = 0; t < MT; ++t) {
#pragma unroll
            for (int o = 16; o < 64; o *= 2) {
                const Part v = {__shfl_xor(st[t].ref, o), __shfl_xor(st[t].l, o), __shfl_xor(st[t].s, o), __shfl_xor(st[t].dot, o), __shfl_xor(st[t].pi, o)};
                few_join(st[t], v);
                abs_sum[t] += __shfl_xor(abs_sum[t], o);
            }
            if (lane < 16) {
                float* o = rows + (wave * 16 * MT + t * 16 + lane) * 6;
                o[0] = st[t].ref, o[1] = st[t].l, o[2] = st[t].s, o[3] = st[t].dot, o[4] = st[t].pi, o[5] = abs_sum[t];
            }
        }
        __syncthreads();
        const int n = threadIdx.x;
        if (n >= 16 * MT || n >= a.t.rows) return;
        Part s = {-INFINITY, 0.0f, 0.0f, 0.0f, 0.0f};
        float sum = 0.0f;
        for (int v = 0; v < 16; ++v) {
            const float* o = rows + (v * 16 * MT + n) * 6;
            few_join(s, Part{o[0], o[1], o[2], o[3], o[4]});
            sum += o[5];
        }
        const int64_t at = (int64_t)n * gridDim.x + blockIdx.x;
        a.part[at] = f32x4{s.ref, s.l, s.s, s.dot};
        if (dense) {
            a.tpart[2 * at] = s.pi;
            a.tpart[2 * at + 1] = sum;
        }
    }
}

struct FewOutArgs {
    const void *w, *x;
    int64_t w_pitch, x_pitch;
    int32_t cols, chunk;          // classes of a workgroup
    Rows t;
    const float* __restrict__ g;  // [classes][16]
    float* part;                  // [chunks][rows][cols], or null
    void *gw, *gb;
};

// Four neighbours of a row from element c on (they may start anywhere), as they are; zero behind the last column.
template <int DT> struct Four {
    uint32_t u[DT == DT_F32 ? 4 : 2];
    __device__ __forceinline__ void load(const void* p, int64_t row, int c, int cols) {
        if (c + 4 <= cols) {
            __builtin_memcpy(u, (const char*)p + (row + c) * FewType<DT>::SIZE, sizeof(u));
        } else {
            float v[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = c + e < cols ? load_scalar<DT>(p, row + c + e) : 0.0f;
            put(v);
        }
    }
    __device__ __forceinline__ void put(const float (&v)[4]) {
        if constexpr (DT == DT_F32) {
#pragma unroll
            for (int e = 0; e < 4; ++e) u[e] = __builtin_bit_cast(uint32_t, v[e]);
        } else {
            const uint2 h = pack4<DT>(v[0], v[1], v[2], v[3]);
            u[0] = h.x, u[1] = h.y;
        }
    }
    __device__ __forceinline__ float get(int e) const {
        if constexpr (DT == DT_F32) return __builtin_bit_cast(float, u[e]);
        else return from_bits<DT>((uint16_t)(u[e >> 1] >> (16 * (e & 1))));
    }
    __device__ __forceinline__ void store(void* p, int64_t row, int c, int cols) const {
        if (c + 4 <= cols) {
            __builtin_memcpy((char*)p + (row + c) * FewType<DT>::SIZE, u, sizeof(u));
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (c + e < cols) {
                    if constexpr (DT == DT_F32) ((uint32_t*)p)[row + c + e] = u[e];
                    else ((uint16_t*)p)[row + c + e] = (uint16_t)(u[e >> 1] >> (16 * (e & 1)));
                }
        }
    }
};

// dx and dW of up to NB rows: a thread owns four features, holds x and dx of them in registers and goes through its classes, the next
// eight weights on their way while eight are used; G comes from LDS. 2 NB multiply-adds for each weight read and gradient written: with
// 16 rows about what the memory allows.
template <int DT, int NB>
__global__ __launch_bounds__(256) void k_ce_few_out(FewOutArgs a) {
    constexpr int U = 8, BLOCK = 64;
    __shared__ __align__(16) float g[BLOCK][16];
    const int d = (blockIdx.x * 256 + threadIdx.x) * 4;
    const int64_t c0 = (int64_t)blockIdx.y * a.chunk, c1 = c0 + a.chunk < a.t.classes ? c0 + a.chunk : a.t.classes;
    Four<DT> x[NB];
    float acc[NB][4];
#pragma unroll
    for (int n = 0; n < NB; ++n) {
        const bool in = n < a.t.rows && !(a.t.index && a.t.index[n < a.t.rows ? n : 0] == a.t.ignore);
        if (in) x[n].load(a.x, n * a.x_pitch, d, a.cols);
        else x[n].put({0.0f, 0.0f, 0.0f, 0.0f});
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[n][e] = 0.0f;
    }
    Four<DT> w[U], next[U];
    auto weights = [&](Four<DT>(&v)[U], int64_t c) {      // classes behind the last one repeat it and are not used
#pragma unroll
        for (int u = 0; u < U; ++u) v[u].load(a.w, (c + u < c1 ? c + u : c1 - 1) * a.w_pitch, d, a.cols);
    };
    weights(w, c0);
    for (int64_t b0 = c0; b0 < c1; b0 += BLOCK) {
        __syncthreads();
        {
            const int64_t c = b0 + (threadIdx.x >> 2);
            if (c < c1) *(f32x4*)&g[threadIdx.x >> 2][(threadIdx.x & 3) * 4] = *(const f32x4*)(a.g + c * 16 + (threadIdx.x & 3) * 4);
        }
        __syncthreads();
        for (int64_t c = b0; c < b0 + BLOCK && c < c1; c += U) {
            weights(next, c + U);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (c + u >= c1) break;
                const float* gu = g[c - b0 + u];
                float o[4] = {0.0f, 0.0f, 0.0f, 0.0f}, sum = 0.0f;
#pragma unroll
                for (int n = 0; n < NB; ++n) {
                    const float gn = gu[n];
                    sum += gn;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        acc[n][e] = __builtin_fmaf(gn, w[u].get(e), acc[n][e]);
                        o[e] = __builtin_fmaf(gn, x[n].get(e), o[e]);
                    }
                }
                if (a.gw) {
                    Four<DT> v;
                    v.put(o);
                    v.store(a.gw, (c + u) * a.cols, d, a.cols);
                }
                if (a.gb && d == 0) store_scalar<DT>(a.gb, c + u, sum);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) w[u] = next[u];
        }
    }
    if (a.part)
#pragma unroll
        for (int n = 0; n < NB; ++n)
            if (n < a.t.rows)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (d + e < a.cols) a.part[((int64_t)blockIdx.y * a.t.rows + n) * a.cols + d + e] = acc[n][e];
}

// dx: the sums of the classes' chunks, in their order.
template <int DT>
__global__ __launch_bounds__(256) void k_ce_few_join(const float* part, int chunks, int64_t size, void* gx) {
    const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (at >= size) return;
    float s = 0.0f;
#pragma unroll 8
    for (int i = 0; i < chunks; ++i) s += part[i * size + at];
    store_scalar<DT>(gx, at, s);
}

}  // namespace
}  // namespace az
