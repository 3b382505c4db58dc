// Rotary positions in general: interleaved pairs or halves, part of a head, scaled
// frequencies, fp32 or bf16, any strides.
//
// y[i] = x[i] c - x[j] s, y[j] = x[i] s + x[j] c for the pair (i, j), c and s the cosine and sine of
// pos * freq times mscale.  One read and one write of the tensor is what it cannot do without;
// an angle costs a 64-bit product and reduction, then fp32 sine and cosine of at most an eighth of a
// turn.  So a thread keeps the angles of its 16 bytes of a head and walks over ROPE_HEADS heads, all of
// whose loads are made before the angles are needed.  8191 tokens x 40 heads of 128, half of each
// turning, bf16: 168 MB in 38 us, 4.4 TB/s of the 5.1 that a copy of 1 GiB reaches here.  16 tokens: 4.8 us,
// the launch.
#include "jas_common.hpp"

#include <cmath>

namespace jas {

struct RopeArgs {
    const void *x;
    void *y;
    const int32_t *pos;
    const double *freq;
    int n, nh, dh, rot;
    long x_st, x_sh, y_st, y_sh;
    float mscale;
    int units, groups;  // threads per head; head groups per token
};

constexpr int ROPE_HEADS = 4;  // heads per thread

template <typename T>
struct RopeIo;
template <>
struct RopeIo<float> {
    static constexpr int E = 4;  // elements of 16 bytes
    static __device__ float get(const float *p) { return *p; }
    static __device__ void put(float *p, float v) { *p = v; }
    static __device__ void get(const float *p, float (&v)[4])
    {
        const floatx4 t = __builtin_nontemporal_load((const floatx4 *)p);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = t[e];
    }
    static __device__ void put(float *p, const float (&v)[4]) { *(floatx4 *)p = floatx4{v[0], v[1], v[2], v[3]}; }
};
template <>
struct RopeIo<uint16_t> {
    static constexpr int E = 8;
    static __device__ float get(const uint16_t *p) { return bf16_to_f32(*p); }
    static __device__ void put(uint16_t *p, float v) { *p = __builtin_bit_cast(uint16_t, (__bf16)v); }
    static __device__ void get(const uint16_t *p, float (&v)[8])
    {
        const u32x4 t = __builtin_nontemporal_load((const u32x4 *)p);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[2 * e] = __uint_as_float(t[e] << 16), v[2 * e + 1] = __uint_as_float(t[e] & 0xffff0000u);
    }
    static __device__ void put(uint16_t *p, const float (&v)[8])
    {
        typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
        u32x4 t;
#pragma unroll
        for (int e = 0; e < 4; ++e) t[e] = __builtin_bit_cast(uint32_t, bf16x2{(__bf16)v[2 * e], (__bf16)v[2 * e + 1]});
        *(u32x4 *)p = t;
    }
};

// cos and sin of pos * freq: turns in 64 bits less their nearest quarter, so what is rounded to
// fp32 is at most an eighth of a turn
__device__ __forceinline__ void rope_angle(double pos, double freq, float mscale, float &c, float &s)
{
    const double turns = pos * freq * 0.15915494309189533577;  // 1 / (2 pi)
    const double quarter = rint(4.0 * turns);
    const float f = (float)(2.0 * (turns - 0.25 * quarter));  // half turns
    const float cf = cospif(f), sf = sinpif(f);
    const int k = (int)(quarter - 4.0 * rint(0.25 * quarter)) & 3;
    c = k & 1 ? sf : cf;
    s = k & 1 ? cf : sf;
    if (k == 1 || k == 2) c = -c;
    if (k & 2) s = -s;
    c *= mscale, s *= mscale;
}

// One thread: unit `u` of a head (W elements of turning pairs, or W elements that are copied) for
// ROPE_HEADS heads of one token.  VEC: 16-byte accesses, W = E; else single elements, W = 2 (one
// pair) or 1.
template <typename T, bool HALVES, bool VEC>
__global__ void __launch_bounds__(256) rope_kernel(const RopeArgs p)
{
    using Io = RopeIo<T>;
    constexpr int E = VEC ? Io::E : 1;
    constexpr int NP = VEC ? (HALVES ? E : E / 2) : 1;  // pairs of a unit
    const long id = (long)blockIdx.x * 256 + threadIdx.x;
    const int u = (int)(id % p.units);
    const long r = id / p.units;
    const int hg = (int)(r % p.groups);
    const long tok = r / p.groups;
    if (tok >= p.n) return;
    const int half = p.rot / 2, turning = half / NP;  // units that turn come first
    const int h0 = hg * ROPE_HEADS, h1 = min(h0 + ROPE_HEADS, p.nh);
    const T *x = (const T *)p.x + tok * p.x_st;
    T *y = (T *)p.y + tok * p.y_st;
    if (u >= turning) {
        const int at = p.rot + (u - turning) * E;
#pragma unroll
        for (int k = 0; k < ROPE_HEADS; ++k)
            if (h0 + k < h1) {
                if constexpr (VEC) *(u32x4 *)(y + (h0 + k) * p.y_sh + at) = *(const u32x4 *)(x + (h0 + k) * p.x_sh + at);
                else y[(h0 + k) * p.y_sh + at] = x[(h0 + k) * p.x_sh + at];
            }
        return;
    }
    float c[NP], s[NP];
    const double pos = p.pos[tok];
#pragma unroll
    for (int i = 0; i < NP; ++i) rope_angle(pos, p.freq[u * NP + i], p.mscale, c[i], s[i]);
    if constexpr (VEC) {  // every head's loads, then its products
        constexpr int P = HALVES ? 2 : 1;
        float v[ROPE_HEADS][P][E];
#pragma unroll
        for (int k = 0; k < ROPE_HEADS; ++k) {
            const T *xr = x + min(h0 + k, h1 - 1) * p.x_sh + u * E;
            Io::get(xr, v[k][0]);
            if constexpr (HALVES) Io::get(xr + half, v[k][1]);
        }
#pragma unroll
        for (int k = 0; k < ROPE_HEADS; ++k) {
            if (h0 + k >= h1) break;
            T *yr = y + (h0 + k) * p.y_sh + u * E;
#pragma unroll
            for (int i = 0; i < NP; ++i) {
                float &a = HALVES ? v[k][0][i] : v[k][0][2 * i], &b = HALVES ? v[k][P - 1][i] : v[k][0][2 * i + 1];
                const float t = a * c[i] - b * s[i];
                b = a * s[i] + b * c[i];
                a = t;
            }
            Io::put(yr, v[k][0]);
            if constexpr (HALVES) Io::put(yr + half, v[k][1]);
        }
    } else {
        const int i = HALVES ? u : 2 * u, j = HALVES ? u + half : 2 * u + 1;
        for (int h = h0; h < h1; ++h) {
            const float a = Io::get(x + h * p.x_sh + i), b = Io::get(x + h * p.x_sh + j);
            Io::put(y + h * p.y_sh + i, a * c[0] - b * s[0]);
            Io::put(y + h * p.y_sh + j, a * s[0] + b * c[0]);
        }
    }
}

template <typename T>
static jas_status rope_launch(RopeArgs &p, int layout, hipStream_t s)
{
    constexpr int E = RopeIo<T>::E;
    const bool halves = layout == JAS_ROPE_HALVES;
    // 16-byte accesses where every row, the turning part and its halves start on 16 bytes
    const bool vec = (((uintptr_t)p.x | (uintptr_t)p.y) & 15) == 0 &&
                     ((p.x_st | p.x_sh | p.y_st | p.y_sh | p.dh | p.rot | (halves ? p.rot / 2 : 0)) & (E - 1)) == 0;
    const int pairs = vec ? (halves ? E : E / 2) : 1;
    p.units = p.rot / 2 / pairs + (p.dh - p.rot) / (vec ? E : 1);
    p.groups = (p.nh + ROPE_HEADS - 1) / ROPE_HEADS;
    // (a launch holds less than 2^32 threads)
    JAS_CHECK((double)p.n * p.units * p.groups <= 4294967040.0, JAS_ERR_RANGE, "jas_rope: too many elements for one call");
    const dim3 grid(ceil_div((long)p.n * p.units * p.groups, 256)), block(256);
    if (halves && vec) hipLaunchKernelGGL((rope_kernel<T, true, true>), grid, block, 0, s, p);
    else if (halves) hipLaunchKernelGGL((rope_kernel<T, true, false>), grid, block, 0, s, p);
    else if (vec) hipLaunchKernelGGL((rope_kernel<T, false, true>), grid, block, 0, s, p);
    else hipLaunchKernelGGL((rope_kernel<T, false, false>), grid, block, 0, s, p);
    JAS_LAUNCH_CHECK();
    return JAS_OK;
}

} // namespace jas

using namespace jas;

extern "C" {

jas_status jas_rope(const void *x, void *y, const int32_t *pos, const double *freq, int n, int nh, int dh, int rot,
                    int64_t x_st, int64_t x_sh, int64_t y_st, int64_t y_sh, int layout, float mscale, int dtype,
                    jas_stream_t stream)
{
    JAS_CHECK(x && y && pos && (freq || rot == 0), JAS_ERR_INVALID, "jas_rope: null pointer");
    JAS_CHECK(n >= 0 && nh > 0 && dh > 0 && rot >= 0 && rot <= dh && rot % 2 == 0, JAS_ERR_INVALID,
              "jas_rope: need n >= 0, nh and dh > 0, an even rot of 0 to dh");
    JAS_CHECK(dtype == JAS_F32 || dtype == JAS_BF16, JAS_ERR_INVALID, "jas_rope: dtype is JAS_F32 or JAS_BF16");
    JAS_CHECK(layout == JAS_ROPE_PAIRS || layout == JAS_ROPE_HALVES, JAS_ERR_INVALID, "jas_rope: unknown layout");
    JAS_CHECK(x != y || (x_st == y_st && x_sh == y_sh), JAS_ERR_INVALID, "jas_rope: in place needs the same strides");
    JAS_CHECK((uintptr_t)freq % 8 == 0 && (uintptr_t)pos % 4 == 0 && ((uintptr_t)x | (uintptr_t)y) % (dtype == JAS_F32 ? 4 : 2) == 0,
              JAS_ERR_INVALID, "jas_rope: pointers aligned to their elements");
    if (!n) return JAS_OK;
    RopeArgs p{x, y, pos, freq, n, nh, dh, rot, (long)x_st, (long)x_sh, (long)y_st, (long)y_sh, mscale, 0, 0};
    return dtype == JAS_F32 ? rope_launch<float>(p, layout, stream_or_default(stream)) : rope_launch<uint16_t>(p, layout, stream_or_default(stream));
}

jas_status jas_rope_freqs(int rot, double theta, const jas_rope_scaling *sc, double *h_freq, float *h_mscale)
{
    JAS_CHECK(h_freq && rot >= 2 && rot % 2 == 0 && theta > 1.0 && std::isfinite(theta), JAS_ERR_INVALID,
              "jas_rope_freqs: need an even rot >= 2, a finite theta > 1 and an output");
    const int kind = sc ? sc->kind : JAS_ROPE_SCALE_NONE;
    JAS_CHECK(kind >= JAS_ROPE_SCALE_NONE && kind <= JAS_ROPE_SCALE_BANDS, JAS_ERR_INVALID, "jas_rope_freqs: unknown scaling");
    if (kind != JAS_ROPE_SCALE_NONE)
        JAS_CHECK(sc->factor > 0.0 && std::isfinite(sc->factor), JAS_ERR_INVALID, "jas_rope_freqs: need a finite factor > 0");
    if (kind == JAS_ROPE_SCALE_YARN || kind == JAS_ROPE_SCALE_BANDS)
        JAS_CHECK(sc->orig_ctx > 0 && sc->low > 0.0 && sc->high > sc->low && std::isfinite(sc->high), JAS_ERR_INVALID,
                  "jas_rope_freqs: need orig_ctx > 0 and 0 < low < high");
    const double two_pi = 6.283185307179586476925;
    double lo = 0.0, hi = 0.0;
    if (kind == JAS_ROPE_SCALE_YARN) {
        // the pair index (of rot, as a real number) that turns `turns` times over orig_ctx
        auto index = [&](double turns) { return rot * std::log(sc->orig_ctx / (turns * two_pi)) / (2.0 * std::log(theta)); };
        lo = std::fmax(std::floor(index(sc->high)), 0.0);
        hi = std::fmin(std::ceil(index(sc->low)), (double)(rot - 1));
    }
    for (int i = 0; i < rot / 2; ++i) {
        double f = std::pow(theta, -2.0 * i / rot);
        if (kind == JAS_ROPE_SCALE_LINEAR) f /= sc->factor;
        else if (kind == JAS_ROPE_SCALE_YARN) {
            const double t = std::fmin(std::fmax((i - lo) / std::fmax(hi - lo, 0.001), 0.0), 1.0);
            f = f / sc->factor * t + f * (1.0 - t);
        } else if (kind == JAS_ROPE_SCALE_BANDS) {
            const double t = std::fmin(std::fmax((sc->orig_ctx * f / two_pi - sc->low) / (sc->high - sc->low), 0.0), 1.0);
            f = f * t + f / sc->factor * (1.0 - t);
        }
        h_freq[i] = f;
    }
    if (h_mscale) *h_mscale = kind == JAS_ROPE_SCALE_YARN && sc->factor > 1.0 ? (float)(0.1 * std::log(sc->factor) + 1.0) : 1.0f;
    return JAS_OK;
}

} // extern "C"
