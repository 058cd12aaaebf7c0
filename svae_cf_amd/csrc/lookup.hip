// Embedding lookup with scaling for tables of any width and type, and its gradient by sorted tokens.
//
//   y[r][:]  = scale * table[t_r][:]                      (t_r outside [0, V): a padded place, zero row)
//   dT[v][:] = scale * sum over { r : t_r = v } of dy[r][:], added in the order of r
//
// Both are bound by HBM: the lookup reads a table row and writes an output row per token, the gradient reads every dy row
// once and writes every table row once (rows without a token as zeros).  The gradient uses no atomics on sums: a stable radix
// sort brings the rows of one token together in their order, so results are the same in every run.
#include "elem.h"

namespace {

__device__ __forceinline__ long long token_at(const void* tok, int tok64, long long i) {
    return tok64 ? reinterpret_cast<const long long*>(tok)[i] : (long long)reinterpret_cast<const int*>(tok)[i];
}

// 1 << lg lanes share a row (the power of two that covers its vectors, at most the workgroup), so narrow rows do not leave
// lanes idle and no index needs a division.
template <int VEC, typename T, typename O>
__global__ __launch_bounds__(256) void lookup_fwd_kernel(const T* __restrict__ table, long long ldt, const void* __restrict__ tok,
                                                         int tok64, O* __restrict__ out, long long ldo, int R, int V, int D,
                                                         int lg, float scale) {
    const long long row = (long long)blockIdx.x * (256 >> lg) + (threadIdx.x >> lg);
    if (row >= R) return;
    const int lane = threadIdx.x & ((1 << lg) - 1);
    const long long t = token_at(tok, tok64, row);
    const bool here = t >= 0 && t < V;
    const T* src = table + (here ? t : 0) * ldt;
    O* dst = out + row * ldo;
    for (int c = lane * VEC; c < D; c += VEC << lg) {
        float v[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[i] = 0.f;
        if (here) {
            sv_load<VEC>(src + c, v);
#pragma unroll
            for (int i = 0; i < VEC; ++i) v[i] *= scale;
        }
        sv_store<VEC>(dst + c, v);
    }
}

// ------------------------------------------------------------------------------------------------
// Stable radix sort of (token, place) by token.  Least significant digit first, the fewest passes of at most 11 bits, equal
// digits; two launches a pass: digit counts per workgroup, then every workgroup adds up the counts in front of it (there are
// at most 256 workgroups, so that is a few microseconds from the L2 and saves a launch for the scan) and places its keys.
// Places outside [0, V) and the padding token get the key V and end up behind all others.
// ------------------------------------------------------------------------------------------------
constexpr int SORT_MAX_BITS = 11, SORT_MAX_WG = 256, SORT_MIN_TILE = 4096;

struct SortShape {
    int passes, bits, nwg, tile;          // digits, bits of a digit, workgroups, keys of a workgroup (a multiple of 1024)
};
inline SortShape sort_shape(int R, int V) {
    SortShape s;
    int bits = 1;
    while (((long long)V >> bits) != 0) ++bits;              // keys 0 .. V
    s.passes = (bits + SORT_MAX_BITS - 1) / SORT_MAX_BITS;
    s.bits = (bits + s.passes - 1) / s.passes;
    long long tile = ((long long)R + SORT_MAX_WG - 1) / SORT_MAX_WG;
    tile = (tile + 1023) / 1024 * 1024;
    s.tile = (int)(tile < SORT_MIN_TILE ? SORT_MIN_TILE : tile);
    s.nwg = (int)(((long long)R + s.tile - 1) / s.tile);
    return s;
}

struct SortArgs {
    const void* tok;                      // first pass: the tokens; later passes: kin / pin
    const int *kin, *pin;
    int *kout, *pout;
    unsigned* cnt;                        // [nwg][1 << bits]
    int tok64, R, V, pad, shift, bits, tile;
};

__device__ __forceinline__ unsigned sort_key(const SortArgs& a, long long i) {
    if (a.kin != nullptr) return (unsigned)a.kin[i];
    const long long t = token_at(a.tok, a.tok64, i);
    return t < 0 || t >= a.V || t == a.pad ? (unsigned)a.V : (unsigned)t;
}

__global__ __launch_bounds__(1024) void sort_count_kernel(SortArgs a) {
    __shared__ unsigned hist[1 << SORT_MAX_BITS];
    const int nb = 1 << a.bits;
    for (int d = threadIdx.x; d < nb; d += 1024) hist[d] = 0;
    __syncthreads();
    const long long base = (long long)blockIdx.x * a.tile;
    for (int j = threadIdx.x; j < a.tile; j += 1024)
        if (base + j < a.R) atomicAdd(&hist[(sort_key(a, base + j) >> a.shift) & (nb - 1)], 1u);     // counts: any order gives the same
    __syncthreads();
    for (int d = threadIdx.x; d < nb; d += 1024) a.cnt[(size_t)blockIdx.x * nb + d] = hist[d];
}

__global__ __launch_bounds__(1024) void sort_place_kernel(SortArgs a) {
    extern __shared__ unsigned lds[];                        // [16 waves][1 << bits], then 16 wave totals
    const int nb = 1 << a.bits, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    unsigned* mine = lds + wave * nb;
    unsigned* wtot = lds + 16 * nb;
    for (int d = tid; d < 16 * nb; d += 1024) lds[d] = 0;
    __syncthreads();
    // each wave owns a run of consecutive keys, so that waves in order and rounds in order are the keys' order
    const int run = a.tile / 16;
    const long long base = (long long)blockIdx.x * a.tile + (long long)wave * run;
    for (int j = lane; j < run; j += 64)
        if (base + j < a.R) atomicAdd(&mine[(sort_key(a, base + j) >> a.shift) & (nb - 1)], 1u);
    // digits 2 tid and 2 tid + 1: keys of this digit in the workgroups in front, and in all
    unsigned before[2] = {0, 0}, total[2] = {0, 0};
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        const int d = 2 * tid + q;
        if (d < nb) {
#pragma unroll 8
            for (int b = 0; b < (int)gridDim.x; ++b) {
                const unsigned n = a.cnt[(size_t)b * nb + d];
                total[q] += n;
                before[q] += b < (int)blockIdx.x ? n : 0u;
            }
        }
    }
    unsigned scan = total[0] + total[1];                     // inclusive scan over the workgroup's threads
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const unsigned up = __shfl_up(scan, o, 64);
        if (lane >= o) scan += up;
    }
    if (lane == 63) wtot[wave] = scan;
    __syncthreads();
    unsigned first = scan - total[0] - total[1];
    for (int w = 0; w < wave; ++w) first += wtot[w];
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        const int d = 2 * tid + q;
        if (d < nb) {
            unsigned at = first + (q ? total[0] : 0u) + before[q];
            for (int w = 0; w < 16; ++w) {
                const unsigned n = lds[w * nb + d];
                lds[w * nb + d] = at;
                at += n;
            }
        }
    }
    __syncthreads();
    volatile unsigned* next = mine;                          // read and written by this wave alone from here on
    for (int j = 0; j < run; j += 64) {
        const long long i = base + j + lane;
        const bool live = i < a.R;
        const unsigned key = live ? sort_key(a, i) : 0u;
        const unsigned digit = (key >> a.shift) & (nb - 1);
        unsigned long long same = __ballot(live);            // the lanes of this round with the same digit
        for (int b = 0; b < a.bits; ++b) {
            const unsigned long long one = __ballot((digit >> b) & 1u);
            same &= (digit >> b) & 1u ? one : ~one;
        }
        const unsigned rank = __popcll(same & ((1ull << lane) - 1ull));
        if (live) {
            const unsigned at = next[digit];
            __builtin_amdgcn_wave_barrier();
            if (rank == 0) next[digit] = at + (unsigned)__popcll(same);
            a.kout[at + rank] = (int)key;
            a.pout[at + rank] = a.pin != nullptr ? a.pin[i] : (int)i;
        }
        __builtin_amdgcn_wave_barrier();
    }
}

// ------------------------------------------------------------------------------------------------
// The gradient over sorted tokens.  A wave owns GROUP table rows and finds their segments of the sorted list by bisection;
// a segment of up to LONG rows is added by that wave, an empty one is written as zeros.  Popular tokens have longer segments:
// those are added in pieces of CHUNK sorted places by workgroups of their own into fp32 partial sums (first workgroups of the
// same launch), which a second launch adds up in order.  A chunk meets at most two long segments, the one at its first place
// (slot 0) and the one at its last (slot 1): anything between is shorter than the chunk.
// ------------------------------------------------------------------------------------------------
constexpr int CHUNK = 64, LONG = 64, GROUP = 4;
static_assert(LONG >= CHUNK, "a chunk could meet a third long segment");

// first place whose key is not below k
__device__ __forceinline__ int lower_bound(const int* __restrict__ keys, int R, long long k) {
    int lo = 0, hi = R;
    while (lo < hi) {
        const int mid = lo + ((hi - lo) >> 1);
        if (keys[mid] < k) lo = mid + 1;
        else hi = mid;
    }
    return lo;
}

// acc += sum of dy[perm[i]][c .. c + VEC) over i = b, b + step, .. < e, eight rows in flight
template <int VEC, typename T>
__device__ __forceinline__ void sum_rows(const T* __restrict__ dy, long long ldd, const int* __restrict__ perm, int b, int e,
                                         int step, int c, float* acc) {
    for (int i = b; i < e; i += 8 * step) {
        float v[8][VEC];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const bool in = i + j * step < e;
            if (in) sv_load<VEC>(dy + (long long)perm[i + j * step] * ldd + c, v[j]);
            else {
#pragma unroll
                for (int q = 0; q < VEC; ++q) v[j][q] = 0.f;
            }
        }
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
            for (int q = 0; q < VEC; ++q) acc[q] += v[j][q];
    }
}

template <int VEC, typename G>
__device__ __forceinline__ void put_row(G* __restrict__ dst, float* acc, float scale, int accumulate) {
#pragma unroll
    for (int q = 0; q < VEC; ++q) acc[q] *= scale;
    if (accumulate) {
        float old[VEC];
        sv_load<VEC>(dst, old);
#pragma unroll
        for (int q = 0; q < VEC; ++q) acc[q] += old[q];
    }
    sv_store<VEC>(dst, acc);
}

template <int VEC, typename T, typename G>
__global__ __launch_bounds__(256) void lookup_bwd_kernel(const T* __restrict__ dy, long long ldd, const int* __restrict__ keys,
                                                         const int* __restrict__ perm, int R, int V, int D, float scale,
                                                         G* __restrict__ grad, long long ldg, int accumulate, int nchunk,
                                                         float* __restrict__ part) {
    __shared__ float red[4][64 * VEC];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if ((int)blockIdx.x < nchunk) {
        const long long p0 = (long long)blockIdx.x * CHUNK;
        const int p1 = (int)(p0 + CHUNK < R ? p0 + CHUNK : R);
        const int kf = keys[p0], kl = keys[p1 - 1];
#pragma unroll 1
        for (int slot = 0; slot < (kf == kl ? 1 : 2); ++slot) {
            const int k = slot == 0 ? kf : kl;
            if (k >= V) continue;
            const int s = lower_bound(keys, R, k), e = lower_bound(keys, R, (long long)k + 1);
            if (e - s <= LONG) continue;
            const int b = s > (int)p0 ? s : (int)p0, z = e < p1 ? e : p1;
            for (int c0 = 0; c0 < D; c0 += 64 * VEC) {
                const int c = c0 + lane * VEC;
                float acc[VEC];
#pragma unroll
                for (int q = 0; q < VEC; ++q) acc[q] = 0.f;
                if (c < D) sum_rows<VEC>(dy, ldd, perm, b + wave, z, 4, c, acc);
#pragma unroll
                for (int q = 0; q < VEC; ++q) red[wave][q * 64 + lane] = acc[q];
                __syncthreads();
                if (wave == 0 && c < D) {
#pragma unroll
                    for (int q = 0; q < VEC; ++q)
                        part[((size_t)blockIdx.x * 2 + slot) * D + c + q] =
                            (red[0][q * 64 + lane] + red[1][q * 64 + lane]) + (red[2][q * 64 + lane] + red[3][q * 64 + lane]);
                }
                __syncthreads();
            }
        }
        return;
    }
    const long long v0 = ((long long)((int)blockIdx.x - nchunk) * 4 + wave) * GROUP;
    if (v0 >= V) return;
    const int mine = lower_bound(keys, R, v0 + (lane < GROUP ? lane : GROUP));
#pragma unroll 1
    for (int g = 0; g < GROUP; ++g) {
        if (v0 + g >= V) return;
        const int s = __builtin_amdgcn_readlane(mine, g), e = __builtin_amdgcn_readlane(mine, g + 1);
        if (e - s > LONG || (accumulate && e == s)) continue;
        G* dst = grad + (v0 + g) * ldg;
        for (int c = lane * VEC; c < D; c += 64 * VEC) {
            float acc[VEC];
#pragma unroll
            for (int q = 0; q < VEC; ++q) acc[q] = 0.f;
            sum_rows<VEC>(dy, ldd, perm, s, e, 1, c, acc);
            put_row<VEC>(dst + c, acc, scale, accumulate);
        }
    }
}

// workgroup p adds up the long segment that starts in chunk p, if one does (it is then the one at the chunk's last place)
template <int VEC, typename G>
__global__ __launch_bounds__(256) void lookup_bwd_long_kernel(const int* __restrict__ keys, int R, int V, int D, float scale,
                                                              G* __restrict__ grad, long long ldg, int accumulate,
                                                              const float* __restrict__ part) {
    __shared__ float red[4][64 * VEC];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const long long p0 = (long long)blockIdx.x * CHUNK;
    const int p1 = (int)(p0 + CHUNK < R ? p0 + CHUNK : R);
    const int k = keys[p1 - 1];
    if (k >= V) return;
    const int s = lower_bound(keys, R, k);
    if (s < (int)p0) return;
    const int e = lower_bound(keys, R, (long long)k + 1);
    if (e - s <= LONG) return;
    const int last = (e - 1) / CHUNK;
    const int slot0 = s == (int)p0 ? 0 : 1;                  // in chunk p; the following ones have it at their first place
    for (int c0 = 0; c0 < D; c0 += 64 * VEC) {
        const int c = c0 + lane * VEC;
        float acc[VEC];
#pragma unroll
        for (int q = 0; q < VEC; ++q) acc[q] = 0.f;
        if (c < D) {
#pragma unroll 4
            for (int j = (int)blockIdx.x + wave; j <= last; j += 4) {
                const int slot = j == (int)blockIdx.x ? slot0 : 0;
#pragma unroll
                for (int q = 0; q < VEC; ++q) acc[q] += part[((size_t)j * 2 + slot) * D + c + q];
            }
        }
#pragma unroll
        for (int q = 0; q < VEC; ++q) red[wave][q * 64 + lane] = acc[q];
        __syncthreads();
        if (wave == 0 && c < D) {
#pragma unroll
            for (int q = 0; q < VEC; ++q)
                acc[q] = (red[0][q * 64 + lane] + red[1][q * 64 + lane]) + (red[2][q * 64 + lane] + red[3][q * 64 + lane]);
            put_row<VEC>(grad + (long long)k * ldg + c, acc, scale, accumulate);
        }
        __syncthreads();
    }
}

inline long long align256(long long n) { return (n + 255) / 256 * 256; }
inline long long chunks_of(int R) { return ((long long)R + CHUNK - 1) / CHUNK; }

}  // namespace

extern "C" int svae_lookup_fwd(const void* table, int table_type, long long ld_table, const void* tokens, int tok64, void* out,
                               int out_type, long long ld_out, int R, int V, int D, float scale, void* stream) {
    SV_CHECK_ARG(R >= 0 && V > 0 && D > 0 && ld_table >= D && ld_out >= D, "svae_lookup_fwd: sizes R %d, V %d, D %d, ld %lld, %lld", R, V, D, ld_table, ld_out);
    SV_CHECK_ARG(table_type >= 0 && table_type <= 2 && out_type >= 0 && out_type <= 2, "svae_lookup_fwd: types %d, %d", table_type, out_type);
    if (R == 0) return 0;
    SV_CHECK_ARG(table && tokens && out, "svae_lookup_fwd: null pointer");
    const int vec = sv_vec_for(8, D, table, ld_table, sv_elem_size(table_type), out, ld_out, sv_elem_size(out_type));
    int lg = 0;
    while (lg < 8 && (vec << lg) < D) ++lg;
    const unsigned nwg = (unsigned)(((long long)R + (256 >> lg) - 1) / (256 >> lg));
    sv_by_type(table_type, [&](auto t) {
        sv_by_type(out_type, [&](auto o) {
            typedef decltype(t) T;
            typedef decltype(o) O;
            auto go = [&](auto kernel) {
                hipLaunchKernelGGL(kernel, dim3(nwg), dim3(256), 0, (hipStream_t)stream, (const T*)table, ld_table, tokens, tok64,
                                   (O*)out, ld_out, R, V, D, lg, scale);
            };
            if (vec == 8) go(lookup_fwd_kernel<8, T, O>);
            else if (vec == 4) go(lookup_fwd_kernel<4, T, O>);
            else if (vec == 2) go(lookup_fwd_kernel<2, T, O>);
            else go(lookup_fwd_kernel<1, T, O>);
        });
    });
    SV_LAUNCH_CHECK();
    return 0;
}

extern "C" int svae_token_sort_bytes(int R, int V, long long* bytes) {
    SV_CHECK_ARG(bytes && R >= 0 && V > 0 && V < 0x7fffffff, "svae_token_sort_bytes: bad arguments");
    const SortShape s = sort_shape(R, V);
    *bytes = align256(4ll * s.nwg << s.bits) + (s.passes > 1 ? 2 * align256(4ll * R) : 0);
    return 0;
}

extern "C" int svae_token_sort(const void* tokens, int tok64, int R, int V, int pad, int* keys, int* perm, void* work,
                               long long work_bytes, void* stream) {
    SV_CHECK_ARG(R >= 0 && R <= 1 << 30 && V > 0 && V < 0x7fffffff, "svae_token_sort: sizes R %d, V %d", R, V);
    if (R == 0) return 0;
    long long need = 0;
    svae_token_sort_bytes(R, V, &need);
    SV_CHECK_ARG(tokens && keys && perm && work, "svae_token_sort: null pointer");
    SV_CHECK_ARG(work_bytes >= need, "svae_token_sort: workspace of %lld bytes, %lld needed", work_bytes, need);
    const SortShape s = sort_shape(R, V);
    char* w = (char*)work;
    SortArgs a;
    a.tok = tokens; a.tok64 = tok64; a.R = R; a.V = V; a.pad = pad; a.bits = s.bits; a.tile = s.tile;
    a.cnt = (unsigned*)w;
    w += align256(4ll * s.nwg << s.bits);
    int* k2 = (int*)w;
    int* p2 = (int*)(w + align256(4ll * R));
    const size_t lds = ((size_t)16 << s.bits) * 4 + 64;
    const hipError_t attr = hipFuncSetAttribute(reinterpret_cast<const void*>(sort_place_kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    if (attr != hipSuccess) return svae_fail((int)attr, "svae_token_sort: %s", hipGetErrorString(attr));
    for (int p = 0; p < s.passes; ++p) {
        const bool to_out = ((s.passes - 1 - p) & 1) == 0;
        a.kin = p == 0 ? nullptr : to_out ? k2 : keys;
        a.pin = p == 0 ? nullptr : to_out ? p2 : perm;
        a.kout = to_out ? keys : k2;
        a.pout = to_out ? perm : p2;
        a.shift = p * s.bits;
        hipLaunchKernelGGL(sort_count_kernel, dim3(s.nwg), dim3(1024), 0, (hipStream_t)stream, a);
        SV_LAUNCH_CHECK();
        hipLaunchKernelGGL(sort_place_kernel, dim3(s.nwg), dim3(1024), lds, (hipStream_t)stream, a);
        SV_LAUNCH_CHECK();
    }
    return 0;
}

extern "C" int svae_lookup_bwd_bytes(int R, int D, long long* bytes) {
    SV_CHECK_ARG(bytes && R >= 0 && D > 0, "svae_lookup_bwd_bytes: bad arguments");
    *bytes = align256(chunks_of(R) * 2 * D * 4);
    return 0;
}

extern "C" int svae_lookup_bwd(const void* dy, int dy_type, long long ld_dy, const int* keys, const int* perm, int R, int V, int D,
                               float scale, void* grad, int grad_type, long long ld_grad, int accumulate, void* work,
                               long long work_bytes, void* stream) {
    SV_CHECK_ARG(R >= 0 && R <= 1 << 30 && V > 0 && D > 0 && ld_dy >= D && ld_grad >= D, "svae_lookup_bwd: sizes R %d, V %d, D %d, ld %lld, %lld", R, V, D, ld_dy, ld_grad);
    SV_CHECK_ARG(dy_type >= 0 && dy_type <= 2 && grad_type >= 0 && grad_type <= 2, "svae_lookup_bwd: types %d, %d", dy_type, grad_type);
    SV_CHECK_ARG(grad && (R == 0 || (dy && keys && perm && work)), "svae_lookup_bwd: null pointer");
    long long need = 0;
    svae_lookup_bwd_bytes(R, D, &need);
    SV_CHECK_ARG(work_bytes >= need, "svae_lookup_bwd: workspace of %lld bytes, %lld needed", work_bytes, need);
    if (R == 0 && accumulate) return 0;
    const int nchunk = (int)chunks_of(R);
    const long long nrow = ((long long)V + 4 * GROUP - 1) / (4 * GROUP);
    SV_CHECK_ARG(nchunk + nrow < 0x7fffffffll, "svae_lookup_bwd: R %d and V %d need too many workgroups", R, V);
    int vec = sv_vec_for(8, D, R ? dy : grad, R ? ld_dy : ld_grad, sv_elem_size(dy_type), grad, ld_grad, sv_elem_size(grad_type));
    while (vec > 2 && 32 * vec >= D) vec >>= 1;              // rather all 64 lanes with shorter vectors
    sv_by_type(dy_type, [&](auto t) {
        sv_by_type(grad_type, [&](auto o) {
            typedef decltype(t) T;
            typedef decltype(o) G;
            auto go = [&](auto kernel, auto join) {
                hipLaunchKernelGGL(kernel, dim3((unsigned)(nchunk + nrow)), dim3(256), 0, (hipStream_t)stream, (const T*)dy, ld_dy, keys,
                                   perm, R, V, D, scale, (G*)grad, ld_grad, accumulate, nchunk, (float*)work);
                if (R > LONG)
                    hipLaunchKernelGGL(join, dim3((unsigned)nchunk), dim3(256), 0, (hipStream_t)stream, keys, R, V, D, scale, (G*)grad,
                                       ld_grad, accumulate, (const float*)work);
            };
            if (vec == 8) go(lookup_bwd_kernel<8, T, G>, lookup_bwd_long_kernel<8, G>);
            else if (vec == 4) go(lookup_bwd_kernel<4, T, G>, lookup_bwd_long_kernel<4, G>);
            else if (vec == 2) go(lookup_bwd_kernel<2, T, G>, lookup_bwd_long_kernel<2, G>);
            else go(lookup_bwd_kernel<1, T, G>, lookup_bwd_long_kernel<1, G>);
        });
    });
    SV_LAUNCH_CHECK();
    return 0;
}
