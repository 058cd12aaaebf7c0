// Dropout from a counter-based generator: the mask is a function of (seed, step, row key, column) and is made again wherever it
// is needed, never stored.
//
//   y[r][c] = keep(r, c) ? x[r][c] / (1 - q) : 0        q = k / 65536, k = round(65536 p)
//   keep(r, c): the 16-bit half (c & 1) of word (c % 8) / 2 of Philox4x32-10(key = seed, counter = (row key low, row key high,
//               c / 8 + 2^31, step)) is at least k
//
// 16 bits an element: one generator call (20 products of 32 x 32 bits) serves 8 elements.  With 32 bits an element the
// generator, not HBM, would bound the bf16 form.  The 2^31 keeps the counters apart from those of the reparameterisation noise
// (svae_philox_normal: column group below 16), so the same seed and step can serve both.  The gradient of dropout is the same
// map of dy.  65536 x 2048 bf16: 89 us, 6.1 TB/s; 21800 x 150: 5.3 us; 256 x 256: 2.6 us, less than its launch.
#include "elem.h"
#include "philox.h"

namespace {

// a thread makes one group of 8 columns, the last one of an odd width in vectors of TAIL (which divides the width); division by the
// groups of a row through a precomputed reciprocal
template <int TAIL, typename T>
__global__ __launch_bounds__(256) void dropout_kernel(const T* x, long long ldx, T* y, long long ldy, long long row0,
                                                      unsigned n, int C, unsigned ng, unsigned long long magic, unsigned below,
                                                      float up, unsigned long long seed, unsigned step,
                                                      const long long* __restrict__ step_dev, const long long* __restrict__ row_key) {
    const unsigned i = blockIdx.x * 256u + threadIdx.x;
    if (i >= n) return;
    const unsigned r = ng == 1 ? i : (unsigned)__umul64hi(magic, (unsigned long long)i);
    const unsigned g = i - r * ng;
    const long long row = row0 + r;
    const unsigned long long key = row_key != nullptr ? (unsigned long long)row_key[row] : (unsigned long long)row;
    if (step_dev != nullptr) step = (unsigned)*step_dev;
    uint32_t c[4] = {(uint32_t)key, (uint32_t)(key >> 32), g | 0x80000000u, step};
    const T* src = x + row * ldx + (long long)g * 8;
    T* dst = y + row * ldy + (long long)g * 8;
    const int left = C - (int)g * 8;
    float v[8] = {};
    if (TAIL == 8 || left >= 8) sv_load<8>(src, v);
    else {
#pragma unroll
        for (int j = 0; j < 8; j += TAIL)
            if (j < left) sv_load<TAIL>(src + j, v + j);
    }
    philox4x32_10(c, (uint32_t)seed, (uint32_t)(seed >> 32));
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const unsigned u = (j & 1) ? c[j >> 1] >> 16 : c[j >> 1] & 0xFFFFu;
        v[j] = u >= below ? v[j] * up : 0.f;
    }
    if (TAIL == 8 || left >= 8) sv_store<8>(dst, v);
    else {
#pragma unroll
        for (int j = 0; j < 8; j += TAIL)
            if (j < left) sv_store<TAIL>(dst + j, v + j);
    }
}

}  // namespace

extern "C" int svae_dropout(const void* x, long long ldx, void* y, long long ldy, int type, int R, int C, double p,
                            unsigned long long seed, unsigned step, const long long* step_dev, const long long* row_key,
                            void* stream) {
    SV_CHECK_ARG(R >= 0 && C > 0 && C <= 1 << 30 && ldx >= C && ldy >= C, "svae_dropout: sizes R %d, C %d, ld %lld, %lld", R, C, ldx, ldy);
    SV_CHECK_ARG(type >= 0 && type <= 2, "svae_dropout: type %d", type);
    SV_CHECK_ARG(p >= 0.0 && p <= 1.0, "svae_dropout: p = %g is no probability", p);
    const unsigned below = (unsigned)(p * 65536.0 + 0.5);
    SV_CHECK_ARG((below == 0) == (p == 0.0) && (below == 65536u) == (p == 1.0), "svae_dropout: p = %g is nearer to 0 or 1 than 2^-17", p);
    if (R == 0) return 0;
    SV_CHECK_ARG(x && y, "svae_dropout: null pointer");
    const float up = below == 65536u ? 0.f : (float)(65536.0 / (65536.0 - below));
    const int tail = sv_vec_for(8, C, true);
    const unsigned ng = (unsigned)((C + 7) / 8);
    // i / ng = high word of i * ceil(2^64 / ng), exact for i and ng below 2^32 (ng = 1, whose reciprocal does not fit, apart)
    const unsigned long long magic = ng == 1 ? 0 : ~0ull / ng + 1;
    const int rows_at_once = (int)(0x7fffff00u / ng);        // indices of a launch stay below 2^31
    for (long long r0 = 0; r0 < R; r0 += rows_at_once) {
        const long long rows = R - r0 < rows_at_once ? R - r0 : rows_at_once;
        const unsigned n = (unsigned)(rows * ng);
        sv_by_type(type, [&](auto t) {
            typedef decltype(t) T;
            auto go = [&](auto kernel) {
                hipLaunchKernelGGL(kernel, dim3((n + 255u) / 256u), dim3(256), 0, (hipStream_t)stream, (const T*)x, ldx, (T*)y, ldy, r0, n, C,
                                   ng, magic, below, up, seed, step, step_dev, row_key);
            };
            if (tail == 8) go(dropout_kernel<8, T>);
            else if (tail == 4) go(dropout_kernel<4, T>);
            else if (tail == 2) go(dropout_kernel<2, T>);
            else go(dropout_kernel<1, T>);
        });
        SV_LAUNCH_CHECK();
    }
    return 0;
}
