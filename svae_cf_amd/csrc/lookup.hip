// Embedding lookup with scaling for tables of any width and type, and its gradient by sorted tokens.
//
//   y[r][:]  = scale * table[t_r][:]                      (t_r outside [0, V): a padded place, zero row)
//   dT[v][:] = scale * sum over { r : t_r = v } of dy[r][:], added in an order that is the same in every run (that of r up to 64 rows;
//              of more, sums of chunks and of every fourth row in them)
//
// Both are bound by HBM: the lookup reads a table row and writes an output row per token, the gradient reads every dy row
// once and writes every table row once (rows without a token as zeros).  The gradient uses no atomics on sums: a stable radix
// sort brings the rows of one token together in their order, so results are the same in every run.
//
// Measured: lookup of 131072 x 1024 bf16 92 us (268 MB written, as much read, popular rows from the caches); its gradient 131 us
// (4.1 TB/s of rows in random order and gradient), with 11603 tokens against 1000000 x 256 fp32 186 us (1.02 GB, nearly all
// zeros, 5.5 TB/s); the sort 20 us for 21800 tokens (latency of four launches), 33 us for 131072.
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
    for (int c0 = lane * VEC; c0 < D; c0 += VEC << lg) {
        const int c = c0 < D - VEC ? c0 : D - VEC;               // (the last vector of an odd width: some columns twice)
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
// Stable radix sort of (token, place) by token, least significant digit first.  Places outside [0, V) and the padding token get
// the key V and end up behind all others.
//   up to SMALL places: one workgroup, digits of 8 bits, keys and places in LDS (vocabulary of 20 000: 256 places 6 us, 4096
//   15.5 us; the four launches that 4097 take 16.5 us);
//   more: the fewest passes of at most 11 bits, equal digits; two launches a pass: digit counts per workgroup, then every
//   workgroup adds up the counts in front of it (there are at most 256 workgroups, so that is a few microseconds from the L2 and
//   saves a launch for the scan) and places its keys.  21 800 places: 1024 a workgroup, 22 workgroups; bound by latency.
// ------------------------------------------------------------------------------------------------
constexpr int SORT_MAX_BITS = 11, SORT_MAX_WG = 256, SORT_MIN_TILE = 1024, SMALL = 4096, SMALL_BITS = 8;

struct SortShape {
    int passes, bits, nwg, tile;          // digits, bits of a digit, workgroups, keys of a workgroup (a multiple of 1024)
};
inline SortShape sort_shape(int R, int V) {
    SortShape s;
    int bits = 1;
    while (((long long)V >> bits) != 0) ++bits;              // keys 0 .. V
    const int most = R <= SMALL ? SMALL_BITS : SORT_MAX_BITS;
    s.passes = (bits + most - 1) / most;
    s.bits = R <= SMALL ? SMALL_BITS : (bits + s.passes - 1) / s.passes;
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
// lanes of the wave that are `live` and have this lane's digit
__device__ __forceinline__ unsigned long long same_digit(bool live, unsigned digit, int bits) {
    unsigned long long same = __ballot(live);
    for (int b = 0; b < bits; ++b) {
        const unsigned long long one = __ballot((digit >> b) & 1u);
        same &= (digit >> b) & 1u ? one : ~one;
    }
    return same;
}
// exclusive sum over the 1024 threads of a workgroup; wtot: 16 words of LDS; ends behind a barrier
__device__ __forceinline__ unsigned scan1024(unsigned v, unsigned* wtot) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    unsigned scan = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const unsigned up = __shfl_up(scan, o, 64);
        if (lane >= o) scan += up;
    }
    if (lane == 63) wtot[wave] = scan;
    __syncthreads();
    unsigned first = scan - v;
    for (int w = 0; w < wave; ++w) first += wtot[w];
    return first;
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
    extern __shared__ unsigned lds[];                        // [16 waves][1 << bits] counts, [1 << bits] x 2 sums, 16 wave totals
    const int nb = 1 << a.bits, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    unsigned* mine = lds + wave * nb;
    unsigned *before = lds + 16 * nb, *total = before + nb, *wtot = total + nb;
    for (int d = tid; d < 18 * nb; d += 1024) lds[d] = 0;
    // each wave owns a run of consecutive keys, so that waves in order and rounds in order are the keys' order
    const int run = a.tile / 16;
    const long long base = (long long)blockIdx.x * a.tile + (long long)wave * run;
    const unsigned key0 = base + lane < a.R ? sort_key(a, base + lane) : 0u;
    __syncthreads();
    for (int j = 0; j < run; j += 64) {
        const long long i = base + j + lane;
        if (i < a.R) atomicAdd(&mine[((j == 0 ? key0 : sort_key(a, i)) >> a.shift) & (nb - 1)], 1u);
    }
    // keys of each digit in the workgroups in front, and in all: the rows of counts are dealt to the threads of a digit
    const int per = nb < 1024 ? 1024 >> a.bits : 1;
    for (int d = tid & (nb - 1), row = tid >> a.bits; d < nb; d += 1024) {
        unsigned b = 0, t = 0;
#pragma unroll 8
        for (int w = nb < 1024 ? row : 0; w < (int)gridDim.x; w += per) {
            const unsigned n = a.cnt[(size_t)w * nb + d];
            t += n;
            b += w < (int)blockIdx.x ? n : 0u;
        }
        if (b) atomicAdd(&before[d], b);
        if (t) atomicAdd(&total[d], t);
    }
    __syncthreads();
    unsigned mine2[2] = {0, 0};                              // digits 2 tid and 2 tid + 1
#pragma unroll
    for (int q = 0; q < 2; ++q)
        if (2 * tid + q < nb) mine2[q] = total[2 * tid + q];
    const unsigned first = scan1024(mine2[0] + mine2[1], wtot);
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        const int d = 2 * tid + q;
        if (d < nb) {
            unsigned at = first + (q ? mine2[0] : 0u) + before[d];
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
        const unsigned key = j == 0 ? key0 : live ? sort_key(a, i) : 0u;
        const unsigned digit = (key >> a.shift) & (nb - 1);
        const unsigned long long same = same_digit(live, digit, a.bits);
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

__global__ __launch_bounds__(1024) void sort_small_kernel(SortArgs a, int passes) {
    constexpr int NB = 1 << SMALL_BITS;
    __shared__ unsigned key[2][SMALL];
    __shared__ unsigned short place[2][SMALL];
    __shared__ unsigned hist[16][NB];
    __shared__ unsigned wtot[16];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int run = (a.R + 1023) / 1024 * 64;                // keys of a wave
    for (int i = tid; i < a.R; i += 1024) {
        key[0][i] = sort_key(a, i);
        place[0][i] = (unsigned short)i;
    }
    for (int p = 0; p < passes; ++p) {
        const int from = p & 1, shift = p * SMALL_BITS;
        for (int d = lane; d < NB; d += 64) hist[wave][d] = 0;
        __syncthreads();
        volatile unsigned* next = hist[wave];
        for (int i = wave * run + lane; i < (wave + 1) * run; i += 64) {
            const bool live = i < a.R;
            const unsigned digit = live ? (key[from][i] >> shift) & (NB - 1) : 0u;
            const unsigned long long same = same_digit(live, digit, SMALL_BITS);
            if (live && (same & ((1ull << lane) - 1ull)) == 0) next[digit] += (unsigned)__popcll(same);
            __builtin_amdgcn_wave_barrier();
        }
        __syncthreads();
        unsigned n = 0;
        if (tid < NB)
            for (int w = 0; w < 16; ++w) n += hist[w][tid];
        unsigned at = scan1024(n, wtot);
        if (tid < NB)
            for (int w = 0; w < 16; ++w) {
                const unsigned c = hist[w][tid];
                hist[w][tid] = at;
                at += c;
            }
        __syncthreads();
        for (int i = wave * run + lane; i < (wave + 1) * run; i += 64) {
            const bool live = i < a.R;
            const unsigned k = live ? key[from][i] : 0u, digit = (k >> shift) & (NB - 1);
            const unsigned long long same = same_digit(live, digit, SMALL_BITS);
            const unsigned rank = __popcll(same & ((1ull << lane) - 1ull));
            if (live) {
                const unsigned to = next[digit];
                __builtin_amdgcn_wave_barrier();
                if (rank == 0) next[digit] = to + (unsigned)__popcll(same);
                key[from ^ 1][to + rank] = k;
                place[from ^ 1][to + rank] = place[from][i];
            }
            __builtin_amdgcn_wave_barrier();
        }
        __syncthreads();
    }
    for (int i = tid; i < a.R; i += 1024) {
        a.kout[i] = (int)key[passes & 1][i];
        a.pout[i] = place[passes & 1][i];
    }
}

// ------------------------------------------------------------------------------------------------
// The gradient over sorted tokens.  A wave owns `group` table rows and finds their segments of the sorted list; a segment of up
// to LONG rows is added by that wave, an empty one is written as zeros.  Popular tokens have longer segments: those are added in
// pieces of CHUNK sorted places by workgroups of their own into fp32 partial sums (first workgroups of the same launch), which a
// second launch adds up in order.  A chunk meets at most two long segments, the one at its first place (slot 0) and the one at
// its last (slot 1): anything between is shorter than the chunk.
// ------------------------------------------------------------------------------------------------
constexpr int CHUNK = 64, LONG = 64, MOST_GROUP = 16;
static_assert(CHUNK == 64 && LONG == CHUNK, "a lane has one place of a chunk, and a chunk meets no third long segment");

// first place in [lo, R) whose key is not below k: 64 ways at a time, so a few loads in a row instead of log2 R
__device__ __forceinline__ int lower_bound(const int* __restrict__ keys, int lo, int R, long long k, int lane) {
    int hi = R;
    while (hi - lo > 64) {
        const long long n = hi - lo;
        const bool below = keys[lo + (int)(n * lane >> 6)] < k;                        // places spread over [lo, hi)
        const int c = __popcll(__ballot(below));                                       // lanes 0 .. c - 1 are below
        hi = c == 64 ? hi : lo + (int)(n * c >> 6) + (c == 0 ? 0 : 1);
        lo = c == 0 ? lo : lo + (int)(n * (c - 1) >> 6) + 1;
        if (c == 0) return lo;
    }
    const bool below = lo + lane < hi && keys[lo + lane < hi ? lo + lane : lo] < k;
    return lo + __popcll(__ballot(below));
}
// the end of the segment of key k that has place i
__device__ __forceinline__ int segment_end(const int* __restrict__ keys, int i, int R, int k, int lane) {
    return lower_bound(keys, i, R, (long long)k + 1, lane);
}

// acc += sum of dy[place(i)][c .. c + VEC) over i = b, b + step, .. < e, sixteen rows in flight (as they lie, 4 registers each)
template <int U, int VEC, typename T, typename P>
__device__ __forceinline__ void add_rows(const T* __restrict__ dy, long long ldd, P place, int b, int e, int step, int c, float* acc) {
    typename SvVec<T, VEC>::type v[U];
#pragma unroll
    for (int j = 0; j < U; ++j)
        if (b + j * step < e) v[j] = *reinterpret_cast<const typename SvVec<T, VEC>::type*>(dy + (long long)place(b + j * step) * ldd + c);
#pragma unroll
    for (int j = 0; j < U; ++j)
        if (b + j * step < e) {
#pragma unroll
            for (int q = 0; q < VEC; ++q) acc[q] += (float)v[j][q];
        }
}
template <int VEC, typename T, typename P>
__device__ __forceinline__ void sum_rows(const T* __restrict__ dy, long long ldd, P place, int b, int e, int step, int c, float* acc) {
    if (e - b <= 4 * step) {                                 // most rows of a table have few
        add_rows<4, VEC>(dy, ldd, place, b, e, step, c, acc);
        return;
    }
    for (int i = b; i < e; i += 16 * step) add_rows<16, VEC>(dy, ldd, place, i, e, step, c, acc);
}

// skip: columns at the front of a vector that reaches back, which another lane has too (written twice, but not added twice)
template <int VEC, typename G>
__device__ __forceinline__ void put_row(G* __restrict__ dst, float* acc, float scale, int accumulate, int skip) {
#pragma unroll
    for (int q = 0; q < VEC; ++q) acc[q] *= scale;
    if (accumulate && skip > 0) {
#pragma unroll
        for (int q = 0; q < VEC; ++q)
            if (q >= skip) dst[q] = (G)(acc[q] + (float)dst[q]);
        return;
    }
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
                                                         G* __restrict__ grad, long long ldg, int accumulate, int nchunk, int group,
                                                         float* __restrict__ part) {
    __shared__ float red[4][64 * VEC];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // the launch's second dimension goes over slices of the columns; the last vector of an odd width takes some columns twice
    const int c0 = ((int)blockIdx.y * 64 + lane) * VEC, c = c0 < D && c0 > D - VEC ? D - VEC : c0;
    const int block = (int)(blockIdx.z * gridDim.x + blockIdx.x);
    if (block < nchunk) {
        const int p0 = block * CHUNK, p1 = R - p0 < CHUNK ? R : p0 + CHUNK;
        // the chunk's keys and those of 64 places on either side: enough to tell which runs are long
        const int kin = p0 + lane < p1 ? keys[p0 + lane] : -1;
        const int kf = __builtin_amdgcn_readfirstlane(kin), kl = __builtin_amdgcn_readlane(kin, p1 - p0 - 1);
        const int kb = p0 > lane ? keys[p0 - 1 - lane] : -1, ka = p1 + lane < R ? keys[p1 + lane] : -1;
        const unsigned long long all = ~0ull;
        auto run = [&](unsigned long long m) { return m == all ? 64 : __builtin_ctzll(~m); };      // lanes from 0 on
        const unsigned long long mf = __ballot(kin == kf), ml = __ballot(kin == kl);
#pragma unroll 1
        for (int slot = 0; slot < (kf == kl ? 1 : 2); ++slot) {
            if ((slot == 0 ? kf : kl) >= V) continue;
            const int b = slot == 0 ? p0 : p0 + __builtin_ctzll(ml), z = slot == 0 ? p0 + __popcll(mf) : p1;
            const int length = z - b + (slot == 0 ? run(__ballot(kb == kf)) : 0) + (z == p1 ? run(__ballot(ka == kl)) : 0);
            if (length <= LONG) continue;
            float acc[VEC];
#pragma unroll
            for (int q = 0; q < VEC; ++q) acc[q] = 0.f;
            if (c < D) sum_rows<VEC>(dy, ldd, [&](int i) { return perm[i]; }, b + wave, z, 4, c, acc);
#pragma unroll
            for (int q = 0; q < VEC; ++q) red[wave][q * 64 + lane] = acc[q];
            __syncthreads();
            if (wave == 0 && c < D) {
#pragma unroll
                for (int q = 0; q < VEC; ++q)
                    acc[q] = (red[0][q * 64 + lane] + red[1][q * 64 + lane]) + (red[2][q * 64 + lane] + red[3][q * 64 + lane]);
                sv_store<VEC>(part + ((size_t)block * 2 + slot) * D + c, acc);
            }
            __syncthreads();
        }
        return;
    }
    const long long v0 = ((long long)(block - nchunk) * 4 + wave) * group;
    if (v0 >= V) return;
    const int s0 = lower_bound(keys, 0, R, v0, lane);
    // the keys from there on tell the other bounds, unless there are more than 64 of them
    const int near = s0 + lane < R ? keys[s0 + lane] : 0x7fffffff;
    const int place = s0 + lane < R ? perm[s0 + lane] : 0;
    int s = s0;
#pragma unroll 1
    for (int g = 0; g < group && v0 + g < V; ++g) {
        int e = s0 + __popcll(__ballot((long long)near <= v0 + g));
        const bool far = e == s0 + 64;
        if (far) e = segment_end(keys, s > e ? s : e, R, (int)(v0 + g), lane);
        G* dst = grad + (v0 + g) * ldg;
        if (e - s <= LONG && !(accumulate && e == s)) {
            if (c < D) {
                float acc[VEC];
#pragma unroll
                for (int q = 0; q < VEC; ++q) acc[q] = 0.f;
                if (far) sum_rows<VEC>(dy, ldd, [&](int i) { return perm[i]; }, s, e, 1, c, acc);
                else if (e > s) sum_rows<VEC>(dy, ldd, [&](int i) { return __builtin_amdgcn_readlane(place, i - s0); }, s, e, 1, c, acc);
                put_row<VEC>(dst + c, acc, scale, accumulate, c0 - c);
            }
        }
        s = e;
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
    const int block = (int)(blockIdx.z * gridDim.x + blockIdx.x);
    const int p0 = block * CHUNK;
    if (R - p0 <= CHUNK) return;                             // no segment of more than LONG starts in the last places
    const int kin = keys[p0 + lane];
    const int k = __builtin_amdgcn_readlane(kin, 63);
    const int ahead = p0 + CHUNK + lane < R ? keys[p0 + CHUNK + lane] : -1;
    const int back = p0 > 0 ? keys[p0 - 1] : -1;
    const unsigned long long here = __ballot(kin == k);
    const int s = p0 + __builtin_ctzll(here);
    const unsigned long long on = __ballot(ahead == k);
    if (k >= V || (s == p0 && back == k) || __popcll(here) + __popcll(on) <= LONG) return;
    const int e = segment_end(keys, p0 + CHUNK, R, k, lane);
    const int last = (e - 1) / CHUNK;
    const int slot0 = s == p0 ? 0 : 1;                       // in chunk p; the following ones have it at their first place
    const int c0 = ((int)blockIdx.y * 64 + lane) * VEC, c = c0 < D && c0 > D - VEC ? D - VEC : c0;
    float acc[VEC];
#pragma unroll
    for (int q = 0; q < VEC; ++q) acc[q] = 0.f;
    if (c < D) {
        // partial sums are rows of D floats, two for a chunk; only the first chunk's may be in the second one
        auto at = [&](int j) { return 2 * j + (j == block ? slot0 : 0); };
        sum_rows<VEC>(part, D, at, block + wave, last + 1, 4, c, acc);
    }
#pragma unroll
    for (int q = 0; q < VEC; ++q) red[wave][q * 64 + lane] = acc[q];
    __syncthreads();
    if (wave == 0 && c < D) {
#pragma unroll
        for (int q = 0; q < VEC; ++q)
            acc[q] = (red[0][q * 64 + lane] + red[1][q * 64 + lane]) + (red[2][q * 64 + lane] + red[3][q * 64 + lane]);
        put_row<VEC>(grad + (long long)k * ldg + c, acc, scale, accumulate, c0 - c);
    }
}

inline long long align256(long long n) { return (n + 255) / 256 * 256; }
inline long long chunks_of(int R) { return ((long long)R + CHUNK - 1) / CHUNK; }

}  // namespace

extern "C" int svae_lookup_fwd(const void* table, int table_type, long long ld_table, const void* tokens, int tok64, void* out,
                               int out_type, long long ld_out, int R, int V, int D, float scale, void* stream) {
    // (the kernel counts columns in 32 bits, one step past the last)
    SV_CHECK_ARG(R >= 0 && V > 0 && D > 0 && D <= 1 << 30 && ld_table >= D && ld_out >= D, "svae_lookup_fwd: sizes R %d, V %d, D %d, ld %lld, %lld", R, V, D, ld_table, ld_out);
    SV_CHECK_ARG(table_type >= 0 && table_type <= 2 && out_type >= 0 && out_type <= 2, "svae_lookup_fwd: types %d, %d", table_type, out_type);
    if (R == 0) return 0;
    SV_CHECK_ARG(table && tokens && out, "svae_lookup_fwd: null pointer");
    const int vec = sv_vec_for(8, D, false);
    int lg = 0;
    while (lg < 8 && (vec << lg) < D) ++lg;
    const long long most = 1ll << (31 - lg);                        // rows of a launch: its threads are counted in 32 bits
    for (long long r0 = 0; r0 < R; r0 += most) sv_by_type(table_type, [&](auto t) {
        sv_by_type(out_type, [&](auto o) {
            typedef decltype(t) T;
            typedef decltype(o) O;
            const int rows = R - r0 < most ? (int)(R - r0) : most;
            const unsigned nwg = (unsigned)(((long long)rows + (256 >> lg) - 1) / (256 >> lg));
            auto go = [&](auto kernel) {
                hipLaunchKernelGGL(kernel, dim3(nwg), dim3(256), 0, (hipStream_t)stream, (const T*)table, ld_table,
                                   (const char*)tokens + r0 * (tok64 ? 8 : 4), tok64, (O*)out + r0 * ld_out, ld_out, rows, V, D, lg, scale);
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
    if (R <= SMALL) {
        *bytes = 0;
        return 0;
    }
    *bytes = align256(4ll * s.nwg << s.bits) + (s.passes > 1 ? 2 * align256(4ll * R) : 0);
    return 0;
}

extern "C" int svae_token_sort(const void* tokens, int tok64, int R, int V, int pad, int* keys, int* perm, void* work,
                               long long work_bytes, void* stream) {
    SV_CHECK_ARG(R >= 0 && R <= 1 << 30 && V > 0 && V < 0x7fffffff, "svae_token_sort: sizes R %d, V %d", R, V);
    if (R == 0) return 0;
    long long need = 0;
    svae_token_sort_bytes(R, V, &need);
    SV_CHECK_ARG(tokens && keys && perm && (work || need == 0), "svae_token_sort: null pointer");
    SV_CHECK_ARG(work_bytes >= need, "svae_token_sort: workspace of %lld bytes, %lld needed", work_bytes, need);
    const SortShape s = sort_shape(R, V);
    char* w = (char*)work;
    SortArgs a;
    a.tok = tokens; a.tok64 = tok64; a.R = R; a.V = V; a.pad = pad; a.bits = s.bits; a.tile = s.tile;
    a.cnt = (unsigned*)w;
    a.kin = a.pin = nullptr; a.kout = keys; a.pout = perm; a.shift = 0;
    if (R <= SMALL) {
        hipLaunchKernelGGL(sort_small_kernel, dim3(1), dim3(1024), 0, (hipStream_t)stream, a, s.passes);
        SV_LAUNCH_CHECK();
        return 0;
    }
    w += align256(4ll * s.nwg << s.bits);
    int* k2 = (int*)w;
    int* p2 = (int*)(w + align256(4ll * R));
    const size_t lds = ((size_t)18 << s.bits) * 4 + 64;
    // (always the most that a call may need, so that calls from several threads do not take it from each other)
    const hipError_t attr = hipFuncSetAttribute(reinterpret_cast<const void*>(sort_place_kernel), hipFuncAttributeMaxDynamicSharedMemorySize,
                                                (18 << SORT_MAX_BITS) * 4 + 64);
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
    // rows of a wave: as many as leave 8192 waves (131072 rows of 1024, as many tokens: 16 rows 170 us, 4 rows 179 us; 20000
    // rows of 256, 21800 tokens: 16 rows 16.6 us, 4 rows 12.7 us)
    const int group = V >= 8192 * MOST_GROUP ? MOST_GROUP : V >= 8192 * 8 ? 8 : 4;
    const long long nrow = ((long long)V + 4 * group - 1) / (4 * group);
    int vec = sv_vec_for(8, D, false);
    while (vec > 2 && 32 * vec >= D) vec >>= 1;              // rather all 64 lanes with shorter vectors
    const long long slices = ((long long)D + 64 * vec - 1) / (64 * vec);
    SV_CHECK_ARG(slices <= 65535, "svae_lookup_bwd: D %d is wider than %d", D, 65535 * 64 * 8);
    // (threads of a dimension are counted in 32 bits: more workgroups than 2^23 go on in the third one)
    auto grid = [&](long long blocks) {
        const long long most = 1ll << 23;
        return dim3((unsigned)(blocks < most ? blocks : most), (unsigned)slices, (unsigned)((blocks + most - 1) / most));
    };
    sv_by_type(dy_type, [&](auto t) {
        sv_by_type(grad_type, [&](auto o) {
            typedef decltype(t) T;
            typedef decltype(o) G;
            auto go = [&](auto kernel, auto join) {
                hipLaunchKernelGGL(kernel, grid(nchunk + nrow), dim3(256), 0, (hipStream_t)stream, (const T*)dy, ld_dy, keys,
                                   perm, R, V, D, scale, (G*)grad, ld_grad, accumulate, nchunk, group, (float*)work);
                if (R > LONG)
                    hipLaunchKernelGGL(join, grid(nchunk), dim3(256), 0, (hipStream_t)stream, keys, R, V, D, scale, (G*)grad,
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
