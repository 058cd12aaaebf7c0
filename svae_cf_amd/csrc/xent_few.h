// Softmax cross entropy for few rows: bound by reading W and writing its gradient, so that W is taken as it lies, once for the
// loss and once for the gradients, without copies.  Part of xent.hip, whose formulas stand there.
//
//   loss       a wave holds z^T of 64 vocabulary entries and all rows; W goes from memory straight into the matrix units' registers.
//              For a gradient z is kept (fp32, 4 R bytes a vocabulary entry; W has 2 D or 4 D).
//   gradients  a workgroup makes G of 32 or 64 entries after the other from z, in LDS; its waves have 64 columns each, read W once
//              for dH, whose sums stay in registers, and write dW.  Workgroups share the vocabulary and leave slabs of dH that are
//              added in order.
//
// fp32 products are fp32 (v_mfma_f32_16x16x4); for one tile of 16 rows G and the gradients' products are fp32 for all types.  More
// rows of 16 bits: 16-bit products, G rounded as by the kernels for many rows.
// At NT tiles of 16 rows fp32 products take 28 NT us for the loss and 55 NT us for the gradients where W has 131072 x 1024 numbers;
// reading W once takes 53 us (16 bits) or 106 us (fp32), writing its gradient as long.
//
// Measured there, loss | loss and gradients (us), against the kernels for many rows:
//   fp32   1 row 133 | 365    (566 | 1285)     32 rows 143 | 408    (555 | 1320)     64 rows 249 | 762    (554 | 1333)
//   bf16   1 row  59 | 217    ( 53 |  400)     32 rows  58 | 207    ( 52 |  397)     64 rows  61 | 240    ( 53 |  401)
// (inputs in rotation, so that W comes from memory; the same ones again and again: bf16 1 row 48 | 203.)
// xent.hip has the limits.  The loss of 64 rows of 16 bits is the one that loses (a million x 256: 138 | 490 against 113 | 1065): loss
// and gradients have to take the same kernels, as z has to have the same bits in both, or errors of z and of lse do not cancel in
// the gradient of a confident row.
#pragma once

struct FewArgs {
    const void *w, *h;        // W as it is; H as it is or its copy (few_logit_kernel)
    const void* hidden;       // H as it is, with ldh
    const void* bias;         // or NULL
    int* tgt;                 // [Rp], -1: left out
    const void* tok;          // the caller's targets, with tok64
    const float *lse, *row_weight;        // gradient: the caller's, [R]
    float2* part;             // loss: [vocabulary tiles][Rp], or NULL (z only)
    float *zt, *z;            // z: [V][R4] or NULL
    float* slab;              // [chunks * waves along V][R][Dp], or NULL: no dH
    void *dw, *db;            // or NULL
    long long ldw, ld_dw, ldh;      // elements
    int tok64, V, D, Dp, R, R4, Rp, ndt, chunks;
};

template <typename T, int N>
using Some = typename SvVec<T, N>::type;                               // from any address a number may have

// the loss's copy of H and the rows' targets
struct FewPrepArgs {
    const void *h, *tok;
    void* hc;
    int* tgt;
    long long ldh;
    int tok64, R, Rp, V, D, Dp;
};
__device__ __forceinline__ int target_at(const void* tok, int tok64, long long r, int V) {
    const long long t = tok64 ? reinterpret_cast<const long long*>(tok)[r] : (long long)reinterpret_cast<const int*>(tok)[r];
    return t >= 0 && t < V ? (int)t : -1;
}

template <typename T>
__global__ __launch_bounds__(256) void few_prep_kernel(FewPrepArgs a) {
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x, r = i / a.Dp;
    const int c = (int)(i - r * a.Dp);
    if (r >= a.Rp) return;
    const int tg = r < a.R ? target_at(a.tok, a.tok64, r, a.V) : -1;
    if (c == 0) a.tgt[r] = tg;
    // in the order in which the matrix units take it, zeros for a left out row: 1 KiB for 16 rows and four times 16 bytes of them (rows
    // a power of two apart fall on few channels of the cache: 64 rows of 256 fp32 took 457 us instead of 381 against a million)
    constexpr int N = 16 / (int)sizeof(T);
    const long long at = ((((long long)(c / (4 * N) / 2) * (a.Rp / 16) + r / 16) * 2 + c / (4 * N) % 2) * 64 + c / N % 4 * 16 + r % 16) * N + c % N;
    reinterpret_cast<T*>(a.hc)[at] = tg >= 0 && c < a.D ? reinterpret_cast<const T*>(a.h)[r * a.ldh + c] : (T)0.f;
}

// weight (0: no part in the gradient), lse and target of the rows, in LDS; ends behind a barrier
template <int ROWS>
__device__ __forceinline__ void few_rows(const FewArgs& a, float* wrow, float* lse, int* tgt) {
    if ((int)threadIdx.x < ROWS) {
        const int r = threadIdx.x;
        const int t = r < a.R ? target_at(a.tok, a.tok64, r, a.V) : -1;
        wrow[r] = t >= 0 ? a.row_weight[r] : 0.f;
        lse[r] = t >= 0 ? a.lse[r] : 0.f;
        tgt[r] = t;
    }
    __syncthreads();
}
// H for dW: zeros behind a row's end and for rows without a part
template <typename T>
__device__ __forceinline__ T few_hidden(const FewArgs& a, const float* wrow, int r, int d) {
    return d < a.D && wrow[r] != 0.f ? reinterpret_cast<const T*>(a.hidden)[r * a.ldh + d] : (T)0.f;
}

__device__ __forceinline__ f32x4 mfma_f32(float a, float b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }

// OWN: H and the targets as the caller has them, without a launch for copies (a left out row, whatever it holds, is a column of
// its own in every product, and its statistics are not taken)
template <typename T, int NT, bool OWN>
__global__ __launch_bounds__(256, NT == 1 ? 4 : 2) void few_logit_kernel(FewArgs a) {
    constexpr int N = 16 / (int)sizeof(T), STEP = 8 * N, MT = 4;       // 128 bytes of a row at a time, in two loads
    typedef Some<T, N> Chunk;
    __shared__ float2 red[4][16 * NT];
    const int lane = threadIdx.x & 63, i16 = lane & 15, q = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const long long v0 = (long long)blockIdx.x * 256 + wave * 64;
    const T* w[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        const long long v = v0 + 16 * t + i16;                         // (entries behind V: another's row, put out below)
        w[t] = reinterpret_cast<const T*>(a.w) + (v < a.V ? v : a.V - 1) * a.ldw + q * N;
    }
    int target[NT];
    const T* h[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        const int r = 16 * n + i16;
        target[n] = !OWN ? a.tgt[r] : r < a.R ? target_at(a.tok, a.tok64, r, a.V) : -1;
        h[n] = reinterpret_cast<const T*>(a.h) + (OWN ? (r < a.R ? r : 0) * a.ldh + q * N : (long long)(n * 2 * 64 + lane) * N);
        if (OWN && blockIdx.x == 0 && threadIdx.x < 16) a.tgt[r] = target[n];
    }
    f32x4 acc[MT][NT];
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int n = 0; n < NT; ++n) acc[t][n] = (f32x4){0.f, 0.f, 0.f, 0.f};
    Chunk x[MT][2], y[NT][2];
    auto part = [&](const T* row, int k) {                             // a lane's 16 bytes from k on, zeros behind the row's end
        const int left = a.D - k - q * N;
        Chunk x;
        if (left >= N) x = *reinterpret_cast<const Chunk*>(row + k);
        else {
#pragma unroll
            for (int e = 0; e < N; ++e) x[e] = e < left ? row[k + e] : (T)0.f;
        }
        return x;
    };
    auto load_h = [&](int k, Chunk (&to)[NT][2]) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                if (!OWN) to[n][c] = *reinterpret_cast<const Chunk*>(h[n] + (k / STEP * NT * 2 + c) * (64 * N));
                else if (k + STEP <= a.D) to[n][c] = *reinterpret_cast<const Chunk*>(h[n] + k + c * 4 * N);
                else to[n][c] = part(h[n], k + c * 4 * N);
            }
    };
    auto load_w = [&](int k, Chunk (&to)[MT][2]) {
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int c = 0; c < 2; ++c) to[t][c] = *reinterpret_cast<const Chunk*>(w[t] + k + c * 4 * N);
    };
    auto multiply = [&]() {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            if constexpr (N == 8) {
#pragma unroll
                for (int t = 0; t < MT; ++t)
#pragma unroll
                    for (int n = 0; n < NT; ++n) acc[t][n] = mfma<T>(__builtin_bit_cast(s16x8, x[t][c]), __builtin_bit_cast(s16x8, y[n][c]), acc[t][n]);
            } else {
#pragma unroll
                for (int e = 0; e < N; ++e)                            // (products of one sum do not follow on each other)
#pragma unroll
                    for (int t = 0; t < MT; ++t)
#pragma unroll
                        for (int n = 0; n < NT; ++n) acc[t][n] = mfma_f32(x[t][c][e], y[n][c][e], acc[t][n]);
            }
        }
    };
    const int full = a.D / STEP;
    if (full > 0) {
        load_w(0, x);
        load_h(0, y);
    }
    for (int s = 1; s < full; ++s) {                                   // the next step's loads are under way during the products
        Chunk x2[MT][2], y2[NT][2];
        load_w(s * STEP, x2);
        load_h(s * STEP, y2);
        __builtin_amdgcn_sched_barrier(0);                             // (the compiler would put them behind)
        multiply();
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
#pragma unroll
            for (int t = 0; t < MT; ++t) x[t][c] = x2[t][c];
#pragma unroll
            for (int n = 0; n < NT; ++n) y[n][c] = y2[n][c];
        }
    }
    if (full > 0) multiply();
    if (full * STEP < a.D) {                                           // the rest of a row; copies of H have zeros there, up to Dp
        load_h(full * STEP, y);
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int c = 0; c < 2; ++c) x[t][c] = part(w[t], full * STEP + c * 4 * N);
        multiply();
    }

    // C: lane has row i16 of tile n, entries 4 q + i of tile t
    const int rest = (int)(a.V - v0 < 64 ? a.V - v0 : 64);
    if (a.bias != nullptr) {
        const T* bias = reinterpret_cast<const T*>(a.bias) + v0;
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int e = 16 * t + 4 * q + i;
                const float b = rest == 64 || e < rest ? (float)bias[e] : 0.f;
#pragma unroll
                for (int n = 0; n < NT; ++n) acc[t][n][i] += b;
            }
    }
    if (rest < 64) {
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int n = 0; n < NT; ++n) acc[t][n][i] = 16 * t + 4 * q + i < rest ? acc[t][n][i] : -INFINITY;
    }
    if (a.z != nullptr) {
        float* z = a.z + (v0 + 4 * q) * a.R4 + i16;
#pragma unroll
        for (int n = 0; n < NT; ++n)
            if (16 * n + i16 < a.R4) {
#pragma unroll
                for (int t = 0; t < MT; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (16 * t + 4 * q + i < rest) z[(16 * t + i) * a.R4 + 16 * n] = acc[t][n][i];
            }
    }
    if (a.part == nullptr) return;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        const int rel = target[n] - ((int)v0 + 4 * q);       // (v0 is below 2^28)
        if (__any(rel >= 0 && rel < 64)) {
#pragma unroll
            for (int t = 0; t < MT; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (rel == 16 * t + i) a.zt[16 * n + i16] = acc[t][n][i];
        }
        float m = -INFINITY, s = 0.f;
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) m = fmaxf(m, acc[t][n][i]);
        // fmaxf leaves NaN out; the sum brings it back (exp(NaN - top)).  The difference first: exact where logits are far from 0
        const float base = m == -INFINITY ? 0.f : m;
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) s += __builtin_amdgcn_exp2f((acc[t][n][i] - base) * LOG2E);
#pragma unroll
        for (int o = 16; o < 64; o <<= 1) {
            const float m2 = __shfl_xor(m, o, 64), s2 = __shfl_xor(s, o, 64);
            join_sums(m, s, m2, s2);
        }
        if (q == 0) red[wave][16 * n + i16] = make_float2(m, s);
    }
    __syncthreads();
    if ((int)threadIdx.x < 16 * NT) {
        float m = red[0][threadIdx.x].x, s = red[0][threadIdx.x].y;
#pragma unroll
        for (int k = 1; k < 4; ++k) join_sums(m, s, red[k][threadIdx.x].x, red[k][threadIdx.x].y);
        a.part[(long long)blockIdx.x * a.Rp + threadIdx.x] = make_float2(m, s);
    }
}

// WD waves along the columns of W, 64 each; the others share the entries of a step
constexpr int few_step(int wd) { return wd == 4 ? 32 : 64; }
constexpr int few_step16(int wd) { return 128 / wd; }

template <typename T, int NT, int WD>
__global__ __launch_bounds__(256, 2) void few_grad_kernel(FewArgs a) {
    constexpr int WV = 4 / WD, STEP = few_step(WD), MINE = STEP / WV, ROWS = 16 * NT, PITCH = ROWS + 1;
    constexpr int QUADS = (STEP * ROWS / 4 + 255) / 256;               // of G, that a thread makes in a step, at most
    typedef Some<T, 4> Quad;
    __shared__ float gs[2][STEP][PITCH];
    __shared__ float wrow[ROWS], lse[ROWS];
    __shared__ int tgt[ROWS];
    const int lane = threadIdx.x & 63, i16 = lane & 15, q = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int dt = blockIdx.x % a.ndt, chunk = blockIdx.x / a.ndt;
    const int d0 = (dt * WD + wave % WD) * 64, first = wave / WD * MINE;        // the wave's columns; its first entry in a step
    const int steps = (a.V + STEP - 1) / STEP;
    const int s0 = (int)((long long)steps * chunk / a.chunks), s1 = (int)((long long)steps * (chunk + 1) / a.chunks);
    for (int i = threadIdx.x; i < 2 * STEP * PITCH; i += 256) (&gs[0][0][0])[i] = 0.f;
    few_rows<ROWS>(a, wrow, lse, tgt);

    const bool on = d0 < a.D;                                          // (else the wave only makes G)
    // column of dW's tile j: a lane's entries 4 q ... 4 q + 3 of two tiles are eight columns in a row
    auto column = [&](int j, int m) { return d0 + 32 * (j >> 1) + 8 * (m >> 2) + 4 * (j & 1) + (m & 3); };
    float ah[4 * NT][4];                                               // H for dW: rows 4 k + q, column i16 of tile j
#pragma unroll
    for (int k = 0; k < 4 * NT; ++k)
#pragma unroll
        for (int j = 0; j < 4; ++j) ah[k][j] = (float)few_hidden<T>(a, wrow, 4 * k + q, column(j, i16));
    f32x4 sum[4][NT];                                                  // dH: columns 4 (4 q + i) + j, row i16 of tile n
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int n = 0; n < NT; ++n) sum[j][n] = (f32x4){0.f, 0.f, 0.f, 0.f};

    const int per = a.R4 / 4, left = on ? a.D - d0 - 4 * i16 : 0;      // quads of an entry; columns of W that the lane has
    f32x4 z[QUADS];
    Quad x[MINE / 4], x2[MINE / 4];
    auto load_z = [&](int s) {
#pragma unroll
        for (int k = 0; k < QUADS; ++k) {
            const int i = threadIdx.x + 256 * k;
            const long long at = (long long)s * STEP * per + i;
            z[k] = (f32x4){0.f, 0.f, 0.f, 0.f};
            if (i < STEP * per && at < (long long)a.V * per) z[k] = reinterpret_cast<const f32x4*>(a.z)[at];
        }
    };
    auto make_g = [&](int s, float (*to)[PITCH]) {
#pragma unroll
        for (int k = 0; k < QUADS; ++k) {
            const int i = threadIdx.x + 256 * k;
            if (i >= STEP * per) break;
            const int e = i / per, r = (i - e * per) * 4;
            const long long v = (long long)s * STEP + e;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float wr = wrow[r + j];
                const float p = __builtin_amdgcn_exp2f((z[k][j] - lse[r + j]) * LOG2E) - (tgt[r + j] == v ? 1.f : 0.f);
                to[e][r + j] = wr == 0.f || v >= a.V ? 0.f : p * wr;   // (a row without a part comes to nothing, whatever its z is)
            }
        }
    };
    auto load_w = [&](int s, Quad (&to)[MINE / 4]) {
#pragma unroll
        for (int g = 0; g < MINE / 4; ++g) {
            const long long v = (long long)s * STEP + first + 4 * g + q;        // (entries behind V: another's row times zero)
            const T* p = reinterpret_cast<const T*>(a.w) + (v < a.V ? v : a.V - 1) * a.ldw + d0 + 4 * i16;
#pragma unroll
            for (int e = 0; e < 4; ++e) to[g][e] = (T)0.f;
            if (left >= 4) to[g] = *reinterpret_cast<const Quad*>(p);
            else if (left > 0) {
#pragma unroll
                for (int e = 0; e < 3; ++e)
                    if (e < left) to[g][e] = p[e];
            }
        }
    };
    if (s0 < s1) {
        load_z(s0);
        if (a.slab != nullptr) load_w(s0, x);
        make_g(s0, gs[s0 & 1]);
    }
    __syncthreads();
    for (int s = s0; s < s1; ++s) {
        const float (*g)[PITCH] = gs[s & 1];
        const bool more = s + 1 < s1;
        if (more) {
            load_z(s + 1);
            if (a.slab != nullptr) load_w(s + 1, x2);
            __builtin_amdgcn_sched_barrier(0);
        }
        if (a.slab != nullptr && on) {
#pragma unroll
            for (int k = 0; k < MINE / 4; ++k) {
                float b[NT];
#pragma unroll
                for (int n = 0; n < NT; ++n) b[n] = g[first + 4 * k + q][16 * n + i16];
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int n = 0; n < NT; ++n) sum[j][n] = mfma_f32((float)x[k][j], b[n], sum[j][n]);
            }
        }
        if (a.dw != nullptr && on) {
#pragma unroll
            for (int t = 0; t < MINE / 16; ++t) {
                f32x4 c[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) c[j] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int k = 0; k < 4 * NT; ++k) {
                    const float b = g[first + 16 * t + i16][4 * k + q];
#pragma unroll
                    for (int j = 0; j < 4; ++j) c[j] = mfma_f32(ah[k][j], b, c[j]);
                }
                const long long v = (long long)s * STEP + first + 16 * t + i16;
                if (v < a.V) {
#pragma unroll
                    for (int j = 0; j < 4; j += 2) {
                        const int d = column(j, 4 * q);
                        T* o = reinterpret_cast<T*>(a.dw) + v * a.ld_dw + d;
                        Some<T, 8> out;
#pragma unroll
                        for (int e = 0; e < 8; ++e) out[e] = (T)c[j + e / 4][e % 4];
                        if (d + 7 < a.D) *reinterpret_cast<Some<T, 8>*>(o) = out;
                        else {
#pragma unroll
                            for (int e = 0; e < 7; ++e)
                                if (d + e < a.D) o[e] = out[e];
                        }
                    }
                }
            }
        }
        if (a.db != nullptr && dt == 0 && (int)threadIdx.x < STEP) {
            const long long v = (long long)s * STEP + threadIdx.x;
            float b = 0.f;
            for (int r = 0; r < a.R; ++r) b += g[threadIdx.x][r];
            if (v < a.V) reinterpret_cast<T*>(a.db)[v] = (T)b;
        }
        if (more) {
            make_g(s + 1, gs[(s + 1) & 1]);                            // (read by every wave before the last barrier)
#pragma unroll
            for (int k = 0; k < MINE / 4; ++k) x[k] = x2[k];
        }
        __syncthreads();
    }
    if (a.slab == nullptr || !on) return;
    float* slab = a.slab + (long long)(chunk * WV + wave / WD) * a.R * a.Dp;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (16 * n + i16 < a.R)
                *reinterpret_cast<f32x4*>(slab + (long long)(16 * n + i16) * a.Dp + d0 + 16 * q + 4 * i) =
                    (f32x4){sum[0][n][i], sum[1][n][i], sum[2][n][i], sum[3][n][i]};
}

// The same for 16-bit types and more than one tile of rows: G in the inputs' type like the kernels for many rows, whose scale it
// has, so that products are v_mfma_f32_16x16x32.  A contraction may take its terms in any order that both operands have:
//   dH  over entries: a lane has four columns of the entries q + 4 g from memory (as they lie); eight of them, g = 0 .. 7, are
//       its part of A, and G lies in that order in LDS (to_h).
//   dW  over rows: eight rows 8 q ... of G lie side by side in LDS (to_w), those of H stay in registers.
template <typename T, int NT, int WD>
__global__ __launch_bounds__(256, 2) void few_grad16_kernel(FewArgs a, float top) {
    constexpr int WV = 4 / WD, MINE = 32, STEP = MINE * WV, ROWS = 16 * NT, PITCH = ROWS + 8;
    constexpr int QUADS = STEP * ROWS / 4 / 256;
    typedef Some<T, 4> Quad;
    __shared__ __attribute__((aligned(16))) T to_h[2][WV][ROWS][MINE], to_w[2][STEP][PITCH];
    __shared__ float wrow[ROWS], lse[ROWS];
    __shared__ int tgt[ROWS];
    const int lane = threadIdx.x & 63, i16 = lane & 15, q = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int dt = blockIdx.x % a.ndt, chunk = blockIdx.x / a.ndt;
    const int d0 = (dt * WD + wave % WD) * 64, part = wave / WD;       // the wave's columns; its entries in a step
    const int steps = (a.V + STEP - 1) / STEP;
    const int s0 = (int)((long long)steps * chunk / a.chunks), s1 = (int)((long long)steps * (chunk + 1) / a.chunks);
    for (int i = threadIdx.x; i < 2 * STEP * ROWS; i += 256) (&to_h[0][0][0][0])[i] = (T)0.f;
    for (int i = threadIdx.x; i < 2 * STEP * PITCH; i += 256) (&to_w[0][0][0])[i] = (T)0.f;
    few_rows<ROWS>(a, wrow, lse, tgt);
    float most = sv_wave_max(fmaxf(lane < ROWS ? fabsf(wrow[lane]) : 0.f, 0.f));        // (ROWS is at most 64; fmaxf leaves NaN out)
    most = most < INFINITY ? fmaxf(most, 0x1p-100f) : top;
    const float up = top / most, down = most / top;

    const bool on = d0 < a.D;                                          // (else the wave only makes G)
    auto column = [&](int j, int m) { return d0 + 32 * (j >> 1) + 8 * (m >> 2) + 4 * (j & 1) + (m & 3); };
    Some<T, 8> ah[NT / 2][4];                                          // H for dW: rows 32 k + 8 q ..., column i16 of tile j
#pragma unroll
    for (int k = 0; k < NT / 2; ++k)
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int e = 0; e < 8; ++e) ah[k][j][e] = few_hidden<T>(a, wrow, 32 * k + 8 * q + e, column(j, i16));
    f32x4 sum[4][NT];                                                  // dH: columns 4 (4 q + i) + j, row i16 of tile n
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int n = 0; n < NT; ++n) sum[j][n] = (f32x4){0.f, 0.f, 0.f, 0.f};

    const int per = a.R4 / 4, left = on ? a.D - d0 - 4 * i16 : 0;      // quads of an entry; columns of W that the lane has
    f32x4 z[QUADS];
    Quad x[8], x2[8];
    auto load_z = [&](int s) {
#pragma unroll
        for (int k = 0; k < QUADS; ++k) {
            const int i = threadIdx.x + 256 * k;
            const long long at = (long long)s * STEP * per + i;
            z[k] = (f32x4){0.f, 0.f, 0.f, 0.f};
            if (i < STEP * per && at < (long long)a.V * per) z[k] = reinterpret_cast<const f32x4*>(a.z)[at];
        }
    };
    auto make_g = [&](int s) {
#pragma unroll
        for (int k = 0; k < QUADS; ++k) {
            const int i = threadIdx.x + 256 * k;
            if (i < STEP * per) {
                const int e = i / per, r = (i - e * per) * 4;
                const long long v = (long long)s * STEP + e;
                Some<T, 4> g;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float wr = wrow[r + j];
                    const float p = __builtin_amdgcn_exp2f((z[k][j] - lse[r + j]) * LOG2E) - (tgt[r + j] == v ? 1.f : 0.f);
                    g[j] = (T)(wr == 0.f || v >= a.V ? 0.f : p * (wr * up));     // (a row without a part comes to nothing, whatever its z is)
                    to_h[s & 1][e / MINE][r + j][(e & 3) * 8 + (e % MINE >> 2)] = g[j];
                }
                *reinterpret_cast<Some<T, 4>*>(&to_w[s & 1][e][r]) = g;
            }
        }
    };
    auto load_w = [&](int s, Quad (&to)[8]) {
#pragma unroll
        for (int g = 0; g < 8; ++g) {
            const long long v = (long long)s * STEP + part * MINE + 4 * g + q;  // (entries behind V: another's row times zero)
            const T* p = reinterpret_cast<const T*>(a.w) + (v < a.V ? v : a.V - 1) * a.ldw + d0 + 4 * i16;
#pragma unroll
            for (int e = 0; e < 4; ++e) to[g][e] = (T)0.f;
            if (left >= 4) to[g] = *reinterpret_cast<const Quad*>(p);
            else if (left > 0) {
#pragma unroll
                for (int e = 0; e < 3; ++e)
                    if (e < left) to[g][e] = p[e];
            }
        }
    };
    if (s0 < s1) {
        load_z(s0);
        if (a.slab != nullptr) load_w(s0, x);
        make_g(s0);
    }
    __syncthreads();
    for (int s = s0; s < s1; ++s) {
        const int b = s & 1;
        const bool more = s + 1 < s1;
        if (more) {
            load_z(s + 1);
            if (a.slab != nullptr) load_w(s + 1, x2);
            __builtin_amdgcn_sched_barrier(0);
        }
        if (a.slab != nullptr && on) {
            s16x8 g[NT];
#pragma unroll
            for (int n = 0; n < NT; ++n) g[n] = *reinterpret_cast<const s16x8*>(&to_h[b][part][16 * n + i16][8 * q]);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                Some<T, 8> w;
#pragma unroll
                for (int e = 0; e < 8; ++e) w[e] = x[e][j];
#pragma unroll
                for (int n = 0; n < NT; ++n) sum[j][n] = mfma<T>(__builtin_bit_cast(s16x8, w), g[n], sum[j][n]);
            }
        }
        if (a.dw != nullptr && on) {
#pragma unroll
            for (int t = 0; t < MINE / 16; ++t) {
                f32x4 c[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) c[j] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int k = 0; k < NT / 2; ++k) {
                    const s16x8 g = *reinterpret_cast<const s16x8*>(&to_w[b][part * MINE + 16 * t + i16][32 * k + 8 * q]);
#pragma unroll
                    for (int j = 0; j < 4; ++j) c[j] = mfma<T>(__builtin_bit_cast(s16x8, ah[k][j]), g, c[j]);
                }
                const long long v = (long long)s * STEP + part * MINE + 16 * t + i16;
                if (v < a.V) {
#pragma unroll
                    for (int j = 0; j < 4; j += 2) {
                        const int d = column(j, 4 * q);
                        T* o = reinterpret_cast<T*>(a.dw) + v * a.ld_dw + d;
                        Some<T, 8> out;
#pragma unroll
                        for (int e = 0; e < 8; ++e) out[e] = (T)(c[j + e / 4][e % 4] * down);
                        if (d + 7 < a.D) *reinterpret_cast<Some<T, 8>*>(o) = out;
                        else {
#pragma unroll
                            for (int e = 0; e < 7; ++e)
                                if (d + e < a.D) o[e] = out[e];
                        }
                    }
                }
            }
        }
        if (a.db != nullptr && dt == 0 && (int)threadIdx.x < STEP) {
            const long long v = (long long)s * STEP + threadIdx.x;
            float sum_g = 0.f;
            for (int r = 0; r < a.R; ++r) sum_g += (float)to_w[b][threadIdx.x][r];
            if (v < a.V) reinterpret_cast<T*>(a.db)[v] = (T)(sum_g * down);
        }
        if (more) {
            make_g(s + 1);                                             // (read by every wave before the last barrier)
#pragma unroll
            for (int k = 0; k < 8; ++k) x[k] = x2[k];
        }
        __syncthreads();
    }
    if (a.slab == nullptr || !on) return;
    float* slab = a.slab + (long long)(chunk * WV + part) * a.R * a.Dp;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (16 * n + i16 < a.R)
                *reinterpret_cast<f32x4*>(slab + (long long)(16 * n + i16) * a.Dp + d0 + 16 * q + 4 * i) =
                    (f32x4){sum[0][n][i], sum[1][n][i], sum[2][n][i], sum[3][n][i]} * down;
}

// dH: sum of the slabs in a fixed order; a workgroup has 8 quads of columns, 32 threads share the slabs of each
template <typename T>
__global__ __launch_bounds__(256) void few_sum_kernel(const float* __restrict__ slab, int slabs, int R, int D, int Dp, T* __restrict__ out, long long ld) {
    __shared__ f32x4 red[32][8];
    const int i = threadIdx.x & 7, s = threadIdx.x >> 3;
    const long long at = (long long)blockIdx.x * 8 + i, all = (long long)R * (Dp / 4);        // (Dp / 4 is a multiple of 16)
    f32x4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int k = s; k < slabs; k += 32) x += *reinterpret_cast<const f32x4*>(slab + ((long long)k * all + at) * 4);
    red[s][i] = x;
    __syncthreads();
    if (s != 0) return;
    for (int k = 1; k < 32; ++k) x += red[k][i];
    const long long r = at / (Dp / 4);
    const int d = (int)(at - r * (Dp / 4)) * 4;
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (d + j < D) out[r * ld + d + j] = (T)x[j];
}
