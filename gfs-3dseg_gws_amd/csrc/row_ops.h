// K8, K9: the row-wise operators beside the attention of serialised points.  Part of attention.hip.
//
// K8 rotary positions: section a of a head (2 P channels) turns by the angle positions[.., a] * freqs[p]:
//     (x, y) -> magnitude (x cos - y sin, y cos + x sin),   pairs (p, p + P) of the section ("half") or (2 p, 2 p + 1) ("interleaved")
// The angle is formed and reduced to an eighth of a turn in fp64 (a position of 10^6 in fp32 is off by 0.06 rad), its sine and cosine are
// Taylor sums in fp32 there (next term below 2e-9); both are computed once per (token, pair) into LDS and serve all heads of q and k,
// which the same launch rotates.  The backward is the same kernel with the sine's sign turned.  HBM-bound: each value is read and
// written once, in 16-byte accesses (2 x 65536 tokens x 16 heads x 64 bf16: 107 us, 5.0 TB/s; 32 x 2048 x 8 x 64 fp32: 63 us, 4.3).
//
// K9 root-mean-square norm with the residual's addition:  s = round(x + r),  y = s (mean s^2 + eps)^-1/2 w
// A group of 8 .. 256 lanes holds a row in registers (8 consecutive channels per lane and step), so that it is read once; the sum
// of squares, the maximum of |y| for the 8-bit form, and the backward's mean of dy w s are reductions over the group.  HBM-bound:
// 65536 x 256 bf16 beside an fp32 stream 38 us forward (5.3 TB/s), 46 us backward (5.8); 16384 x 4096 half to e4m3 102 - 104 us (4.6).  Rows that
// are no multiple of 8 channels, or not aligned, are read element by element: 4097 x 4095 123 and 148 us, 4096 x 4096 40 and 51.

namespace gfs3d {
namespace {

struct RoArgs {
    const void *x[2];                       // q, k (k may be NULL)
    void *y[2];
    long long sb[2], sr[2], sh[2];          // input strides (sequence, row, head) in elements
    long long ob[2], orr[2], oh[2];         // output strides
    int heads[2];
    int N, D, axes, pairs;                  // pairs: per axis
    long long tokens;
    const void *pos;
    int pos_type;                           // 0 int32, 1 int64, 2 float32
    const double *freqs;
    float magnitude, sign;
    int interleaved, tb;                    // tb: tokens of a workgroup
    int per;                                // units of a head
    unsigned m_per, m_heads;                // ceil(2^32 / per), / heads where that divides exactly (0: plain division)
};
__device__ __forceinline__ int ro_div(int u, int d, unsigned m) { return m ? (int)__umulhi((unsigned)u, m) : u / d; }
__device__ __forceinline__ float2 ro_turn(double turns)
{
    const double z = (turns - __builtin_rint(turns)) * 4.0, nq = __builtin_rint(z);
    const float x = (float)((z - nq) * 1.5707963267948966), x2 = x * x;
    const int n = (int)nq & 3;
    const float s = x * fmaf(x2, fmaf(x2, fmaf(x2, fmaf(x2, 1.f / 362880.f, -1.f / 5040.f), 1.f / 120.f), -1.f / 6.f), 1.f);
    const float c = fmaf(x2, fmaf(x2, fmaf(x2, fmaf(x2, fmaf(x2, -1.f / 3628800.f, 1.f / 40320.f), -1.f / 720.f), 1.f / 24.f), -0.5f), 1.f);
    const float cs = (n & 1) ? s : c, sn = (n & 1) ? c : s;       // quarter turns: (c, s), (-s, c), (-c, -s), (s, -c)
    return make_float2((n == 1 || n == 2) ? -cs : cs, (n & 2) ? -sn : sn);
}
// VEC: channels of one access (16 bytes), or 1
template <class T, int VEC>
__global__ void __launch_bounds__(256) rotary_kernel(const RoArgs g)
{
    extern __shared__ __attribute__((aligned(16))) float2 ro_cs[];          // [token][axis * pairs + p]
    __shared__ long long ro_at[16][4];                                      // a token's offset in q, k and their outputs
    const int t = threadIdx.x, AP = g.axes * g.pairs;
    const long long tok0 = (long long)blockIdx.x * g.tb;
    const int nt = (int)min((long long)g.tb, g.tokens - tok0);
    if (t < 4 * nt) {
        const long long b = (tok0 + t / 4) / g.N, n = (tok0 + t / 4) % g.N;
        const int w = t & 1;
        ro_at[t / 4][t & 3] = t & 2 ? b * g.ob[w] + n * g.orr[w] : b * g.sb[w] + n * g.sr[w];
    }
    for (int e = t; e < nt * AP; e += 256) {
        const long long tk = tok0 + e / AP;
        const int ap = e % AP, a = ap / g.pairs;
        const long long pi = tk * g.axes + a;
        const double pos = g.pos_type == 0 ? (double)static_cast<const int *>(g.pos)[pi]
                         : g.pos_type == 1 ? (double)static_cast<const long long *>(g.pos)[pi] : (double)static_cast<const float *>(g.pos)[pi];
        const float2 cs = ro_turn(pos * g.freqs[ap % g.pairs] * 0.15915494309189535);
        ro_cs[e] = make_float2(cs.x * g.magnitude, cs.y * g.magnitude * g.sign);
    }
    __syncthreads();
    typedef T Tv __attribute__((ext_vector_type(VEC)));
    const int P = g.pairs, heads = g.heads[0] + g.heads[1];
    if (g.interleaved) {
        constexpr int W = VEC > 1 ? VEC : 2;                                // channels of a unit: whole pairs
        const int per = g.per, units = nt * heads * per;
#pragma unroll 4
        for (int u = t; u < units; u += 256) {
            const int th = ro_div(u, per, g.m_per), c0 = (u - th * per) * W, tk = ro_div(th, heads, g.m_heads), hd = th - tk * heads;
            const int w = hd >= g.heads[0], hh = w ? hd - g.heads[0] : hd;
            const T *x = (const T *)g.x[w] + ro_at[tk][w] + hh * g.sh[w] + c0;
            T *y = (T *)g.y[w] + ro_at[tk][2 + w] + hh * g.oh[w] + c0;
            typedef T Tw __attribute__((ext_vector_type(W)));
            Tw v;
            if constexpr (VEC > 1) v = *reinterpret_cast<const Tw *>(x);
            else {
                v[0] = x[0];
                v[1] = c0 + 1 < g.D ? x[1] : (T)0.f;
            }
#pragma unroll
            for (int e = 0; e < W; e += 2) {
                const int ap = (c0 + e) >> 1;
                if (ap < AP) {
                    const float2 cs = ro_cs[tk * AP + ap];
                    const float a = (float)v[e], bb = (float)v[e + 1];
                    v[e] = (T)fmaf(a, cs.x, -(bb * cs.y));
                    v[e + 1] = (T)fmaf(bb, cs.x, a * cs.y);
                }
            }
            if constexpr (VEC > 1) *reinterpret_cast<Tw *>(y) = v;
            else {
                y[0] = v[0];
                if (c0 + 1 < g.D) y[1] = v[1];
            }
        }
        return;
    }
    // half: a unit is VEC pairs of one section, or VEC channels behind the sections
    const int pu = AP / VEC, per = g.per, units = nt * heads * per;
#pragma unroll 4
    for (int u = t; u < units; u += 256) {
        const int th = ro_div(u, per, g.m_per), k = u - th * per, tk = ro_div(th, heads, g.m_heads), hd = th - tk * heads;
        const int w = hd >= g.heads[0], hh = w ? hd - g.heads[0] : hd;
        const T *x = (const T *)g.x[w] + ro_at[tk][w] + hh * g.sh[w];
        T *y = (T *)g.y[w] + ro_at[tk][2 + w] + hh * g.oh[w];
        if (k < pu) {
            const int ap = k * VEC, ch = ap / P * 2 * P + ap % P;
            Tv a = *reinterpret_cast<const Tv *>(x + ch), c = *reinterpret_cast<const Tv *>(x + ch + P);
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float2 cs = ro_cs[tk * AP + ap + e];
                const float fa = (float)a[e], fb = (float)c[e];
                a[e] = (T)fmaf(fa, cs.x, -(fb * cs.y));
                c[e] = (T)fmaf(fb, cs.x, fa * cs.y);
            }
            *reinterpret_cast<Tv *>(y + ch) = a;
            *reinterpret_cast<Tv *>(y + ch + P) = c;
        } else {
            const int ch = 2 * AP + (k - pu) * VEC;
            *reinterpret_cast<Tv *>(y + ch) = *reinterpret_cast<const Tv *>(x + ch);
        }
    }
}

// ------------------------------------------------------------------ K9
enum { RN_NONE = 0, RN_SAME = 1, RN_F32 = 2 };         // the residual: none, x's type, fp32
struct RnArgs {
    const void *x, *r, *dy, *ds;                        // r: residual (backward: unused); ds: gradient of the stream
    const void *w;
    void *s, *y;                                        // stream (forward: written, residual's type), normed rows; backward: dx in y, dr in s
    float *scale, *rstd, *part;
    long long xs, rs, ds_s, dys;                        // row strides in elements
    long long rows;
    int C, rkind, wf32, group, vec;                     // group: 0 = row; vec: 8-channel accesses are aligned
    float eps, inv_c;
};
template <class T> __device__ __forceinline__ void rn_load8(const T *p, int n, bool vec, float (&v)[8])
{
    typedef T Tv __attribute__((ext_vector_type(16 / sizeof(T))));
    if (vec) {
        if (n >= 8) {
#pragma unroll
            for (int q = 0; q < 8; q += 16 / (int)sizeof(T)) {
                const Tv a = *reinterpret_cast<const Tv *>(p + q);
#pragma unroll
                for (int e = 0; e < 16 / (int)sizeof(T); ++e) v[q + e] = (float)a[e];
            }
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = 0.f;
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = e < n ? (float)p[e] : 0.f;
    }
}
template <class T> __device__ __forceinline__ void rn_store8(T *p, int n, bool vec, const float (&v)[8])
{
    typedef T Tv __attribute__((ext_vector_type(16 / sizeof(T))));
    if (vec) {
        if (n < 8) return;
#pragma unroll
        for (int q = 0; q < 8; q += 16 / (int)sizeof(T)) {
            Tv a;
#pragma unroll
            for (int e = 0; e < 16 / (int)sizeof(T); ++e) a[e] = (T)v[q + e];
            *reinterpret_cast<Tv *>(p + q) = a;
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (e < n) p[e] = (T)v[e];
    }
}
__device__ __forceinline__ float rn_nanmax(float a, float b) { return (b > a || b != b) ? b : a; }        // a NaN stays
// sum / maximum over the TPR lanes of a row (TPR = 256: the workgroup, through `sh`; `slot` alternates so that one barrier is enough)
template <int TPR> __device__ __forceinline__ float rn_sum(float v, float (*sh)[4], int &slot)
{
    v = group8_sum(v);
    if (TPR >= 16) v = GFS3D_DPP_ADD(v, 0x140);
    if (TPR >= 32) v += __shfl_xor(v, 16, 64);
    if (TPR >= 64) v += __shfl_xor(v, 32, 64);
    if (TPR == 256) {
        if ((threadIdx.x & 63) == 0) sh[slot][threadIdx.x >> 6] = v;
        __syncthreads();
        v = (sh[slot][0] + sh[slot][1]) + (sh[slot][2] + sh[slot][3]);
        slot = slot == 2 ? 0 : slot + 1;
    }
    return v;
}
template <int TPR> __device__ __forceinline__ float rn_max(float v, float (*sh)[4], int &slot)
{
#pragma unroll
    for (int st = 1; st < (TPR < 64 ? TPR : 64); st <<= 1) v = rn_nanmax(v, lane_xor_f(v, st));
    if (TPR == 256) {
        if ((threadIdx.x & 63) == 0) sh[slot][threadIdx.x >> 6] = v;
        __syncthreads();
        v = rn_nanmax(rn_nanmax(sh[slot][0], sh[slot][1]), rn_nanmax(sh[slot][2], sh[slot][3]));
        slot = slot == 2 ? 0 : slot + 1;
    }
    return v;
}
constexpr float RN_FP8_MAX = 448.f, RN_AMAX_FLOOR = 1e-12f;

template <class T, int TPR, int VPL, bool FP8>
__global__ void __launch_bounds__(256) rms_fwd_kernel(const RnArgs g)
{
    __shared__ float sh[3][4];
    int slot = 0;
    const int lane = threadIdx.x % TPR, sub = threadIdx.x / TPR;
    constexpr int RPB = 256 / TPR;
    const bool vec = g.vec != 0;
    float w[VPL][8];
#pragma unroll
    for (int v = 0; v < VPL; ++v) {
        const int c0 = (v * TPR + lane) * 8;
        if (g.wf32) rn_load8<float>((const float *)g.w + c0, g.C - c0, vec, w[v]);
        else rn_load8<T>((const T *)g.w + c0, g.C - c0, vec, w[v]);
    }
    // every lane of a workgroup takes the same number of turns (the row's reductions need them all)
    for (long long row0 = (long long)blockIdx.x * RPB; row0 < g.rows; row0 += (long long)gridDim.x * RPB) {
        const long long row = row0 + sub;
        const bool on = row < g.rows;
        float h[VPL][8], ss = 0.f;
#pragma unroll
        for (int v = 0; v < VPL; ++v) {
            const int c0 = (v * TPR + lane) * 8, n = on ? g.C - c0 : 0;
            rn_load8<T>((const T *)g.x + row * g.xs + c0, n, vec, h[v]);
            if (g.rkind != RN_NONE) {
                float r8[8];
                if (g.rkind == RN_F32) rn_load8<float>((const float *)g.r + row * g.rs + c0, n, vec, r8);
                else rn_load8<T>((const T *)g.r + row * g.rs + c0, n, vec, r8);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    h[v][e] += r8[e];
                    if (g.rkind == RN_SAME) h[v][e] = (float)(T)h[v][e];          // the norm is of the stream as it is stored
                }
                if (g.rkind == RN_F32) rn_store8<float>((float *)g.s + row * g.C + c0, n, vec, h[v]);
                else rn_store8<T>((T *)g.s + row * g.C + c0, n, vec, h[v]);
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) ss = fmaf(h[v][e], h[v][e], ss);
        }
        ss = rn_sum<TPR>(ss, sh, slot);
        const float rstd = 1.f / sqrtf(fmaf(ss, g.inv_c, g.eps));
        if (g.rstd && on && lane == 0) g.rstd[row] = rstd;
#pragma unroll
        for (int v = 0; v < VPL; ++v)
#pragma unroll
            for (int e = 0; e < 8; ++e) h[v][e] = h[v][e] * rstd * w[v][e];
        if constexpr (!FP8) {
#pragma unroll
            for (int v = 0; v < VPL; ++v) {
                const int c0 = (v * TPR + lane) * 8;
                rn_store8<T>((T *)g.y + row * g.C + c0, on ? g.C - c0 : 0, vec, h[v]);
            }
        } else {
            float am[VPL];
#pragma unroll
            for (int v = 0; v < VPL; ++v) {
                am[v] = 0.f;
#pragma unroll
                for (int e = 0; e < 8; ++e) am[v] = rn_nanmax(am[v], fabsf(h[v][e]));
            }
            if (g.group == 0) {
#pragma unroll
                for (int v = 1; v < VPL; ++v) am[0] = rn_nanmax(am[0], am[v]);
                am[0] = rn_max<TPR>(am[0], sh, slot);
#pragma unroll
                for (int v = 1; v < VPL; ++v) am[v] = am[0];
            } else {
                const int lanes = g.group / 8;                                       // 4, 8 or 16 consecutive lanes
#pragma unroll
                for (int v = 0; v < VPL; ++v) {
                    am[v] = rn_nanmax(am[v], lane_xor_f(am[v], 1));
                    am[v] = rn_nanmax(am[v], lane_xor_f(am[v], 2));
                    if (lanes >= 8) am[v] = rn_nanmax(am[v], lane_xor_f(am[v], 4));
                    if (lanes >= 16) am[v] = rn_nanmax(am[v], lane_xor_f(am[v], 8));
                }
            }
#pragma unroll
            for (int v = 0; v < VPL; ++v) {
                const int c0 = (v * TPR + lane) * 8, n = on ? g.C - c0 : 0;
                if (n <= 0) continue;
                const float sc = (am[v] < RN_AMAX_FLOOR ? RN_AMAX_FLOOR : am[v]) / RN_FP8_MAX, inv = 1.f / sc;
                if (g.group == 0) {
                    if (c0 == 0) g.scale[row] = sc;
                } else if (c0 % g.group == 0) g.scale[row * (g.C / g.group) + c0 / g.group] = sc;
                unsigned b[2];
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    float f[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float z = h[v][4 * q + e] * inv;
                        f[e] = z > RN_FP8_MAX ? RN_FP8_MAX : z < -RN_FP8_MAX ? -RN_FP8_MAX : z;          // (a NaN stays)
                    }
                    int p = __builtin_amdgcn_cvt_pk_fp8_f32(f[0], f[1], 0, false);
                    b[q] = (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(f[2], f[3], p, true);
                }
                uint8_t *o = (uint8_t *)g.y + row * g.C + c0;
                if (vec) *reinterpret_cast<uint2 *>(o) = make_uint2(b[0], b[1]);
                else
                    for (int e = 0; e < 8 && e < n; ++e) o[e] = (uint8_t)(b[e >> 2] >> (8 * (e & 3)));
            }
        }
    }
}

// x: the stream (or x without a residual).  dx (T) in g.y; dr, fp32 residual only, in g.s.  part: [workgroup][C] sums of dy n
template <class T, int TPR, int VPL>
__global__ void __launch_bounds__(256) rms_bwd_kernel(const RnArgs g)
{
    __shared__ float sh[3][4];
    extern __shared__ __attribute__((aligned(16))) float rn_dw[];
    int slot = 0;
    const int lane = threadIdx.x % TPR, sub = threadIdx.x / TPR;
    constexpr int RPB = 256 / TPR;
    const bool vec = g.vec != 0;
    float w[VPL][8], dw[VPL][8];
#pragma unroll
    for (int v = 0; v < VPL; ++v) {
        const int c0 = (v * TPR + lane) * 8;
        if (g.wf32) rn_load8<float>((const float *)g.w + c0, g.C - c0, vec, w[v]);
        else rn_load8<T>((const T *)g.w + c0, g.C - c0, vec, w[v]);
#pragma unroll
        for (int e = 0; e < 8; ++e) dw[v][e] = 0.f;
    }
    for (long long row0 = (long long)blockIdx.x * RPB; row0 < g.rows; row0 += (long long)gridDim.x * RPB) {
        const long long row = row0 + sub;
        const bool on = row < g.rows;
        const float rstd = on ? g.rstd[row] : 0.f;
        float h[VPL][8], dy[VPL][8], cs = 0.f;
#pragma unroll
        for (int v = 0; v < VPL; ++v) {
            const int c0 = (v * TPR + lane) * 8, n = on ? g.C - c0 : 0;
            if (g.rkind == RN_F32) rn_load8<float>((const float *)g.x + row * g.xs + c0, n, vec, h[v]);
            else rn_load8<T>((const T *)g.x + row * g.xs + c0, n, vec, h[v]);
            rn_load8<T>((const T *)g.dy + row * g.dys + c0, n, vec, dy[v]);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                h[v][e] *= rstd;
                dw[v][e] = fmaf(dy[v][e], h[v][e], dw[v][e]);
                dy[v][e] *= w[v][e];
                cs = fmaf(dy[v][e], h[v][e], cs);
            }
        }
        cs = rn_sum<TPR>(cs, sh, slot) * g.inv_c;
#pragma unroll
        for (int v = 0; v < VPL; ++v) {
            const int c0 = (v * TPR + lane) * 8, n = on ? g.C - c0 : 0;
            float o[8], d8[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) d8[e] = 0.f;
            if (g.ds) {
                if (g.rkind == RN_F32) rn_load8<float>((const float *)g.ds + row * g.ds_s + c0, n, vec, d8);
                else rn_load8<T>((const T *)g.ds + row * g.ds_s + c0, n, vec, d8);
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) o[e] = fmaf(rstd, fmaf(-h[v][e], cs, dy[v][e]), d8[e]);
            if (g.y) rn_store8<T>((T *)g.y + row * g.C + c0, n, vec, o);
            if (g.s) rn_store8<float>((float *)g.s + row * g.C + c0, n, vec, o);
        }
    }
    if (!g.part) return;
    // the row groups of the workgroup join in order
    float *o = g.part + (size_t)blockIdx.x * g.C;
    if constexpr (RPB == 1) {
#pragma unroll
        for (int v = 0; v < VPL; ++v) rn_store8<float>(o + (v * TPR + lane) * 8, g.C - (v * TPR + lane) * 8, false, dw[v]);
    } else {
        for (int s = 0; s < RPB; ++s) {
            if (sub == s) {
#pragma unroll
                for (int v = 0; v < VPL; ++v)
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const int c = (v * TPR + lane) * 8 + e;
                        rn_dw[c] = s ? rn_dw[c] + dw[v][e] : dw[v][e];
                    }
            }
            __syncthreads();
        }
        for (int c = threadIdx.x; c < g.C; c += 256) o[c] = rn_dw[c];
    }
}
// dw[c] = sum over the parts, in order within each of 32 slices, then over the slices
template <class W>
__global__ void __launch_bounds__(1024) rms_dw_kernel(const float *__restrict__ part, int nparts, int C, W *__restrict__ dw)
{
    __shared__ float sh[32][33];
    const int tc = threadIdx.x & 31, c = blockIdx.x * 32 + tc, sl = threadIdx.x >> 5;
    float s = 0.f;
    if (c < C) {
#pragma unroll 8
        for (int p = sl; p < nparts; p += 32) s += part[(size_t)p * C + c];
    }
    sh[sl][tc] = s;
    __syncthreads();
    if (sl == 0 && c < C) {
#pragma unroll
        for (int k = 1; k < 32; ++k) s += sh[k][tc];
        dw[c] = (W)s;
    }
}

template <class T> int rn_forward(const RnArgs &g, bool fp8, hipStream_t st)
{
    const int C = g.C;
#define RN_FWD(TPR, VPL)                                                                                                              \
    {                                                                                                                                 \
        const long long need = (g.rows + 256 / TPR - 1) / (256 / TPR);                                                                \
        const unsigned blocks = (unsigned)(need < 2048 ? need : 2048);                                                                \
        if (fp8) hipLaunchKernelGGL((rms_fwd_kernel<T, TPR, VPL, true>), dim3(blocks), dim3(256), 0, st, g);                          \
        else hipLaunchKernelGGL((rms_fwd_kernel<T, TPR, VPL, false>), dim3(blocks), dim3(256), 0, st, g);                             \
        GFS3D_LAUNCH_CHECK("rms_fwd_kernel");                                                                                         \
        return GFS3D_OK;                                                                                                              \
    }
    if (C <= 64) RN_FWD(8, 1)
    if (C <= 128) RN_FWD(16, 1)
    if (C <= 256) RN_FWD(32, 1)
    if (C <= 512) RN_FWD(64, 1)
    if (C <= 1024) RN_FWD(64, 2)
    if (C <= 2048) RN_FWD(256, 1)
    if (C <= 4096) RN_FWD(256, 2)
    if (C <= 8192) RN_FWD(256, 4)
    RN_FWD(256, 8)
#undef RN_FWD
}
constexpr int RN_PARTS = 512;         // workgroups of the backward: two per CU; each leaves one row of weight-gradient sums
template <class T> int rn_backward(const RnArgs &g, int &parts, hipStream_t st)
{
    const int C = g.C;
#define RN_BWD(TPR, VPL)                                                                                                              \
    {                                                                                                                                 \
        const long long need = (g.rows + 256 / TPR - 1) / (256 / TPR);                                                                \
        parts = (int)(need < RN_PARTS ? need : RN_PARTS);                                                                             \
        hipLaunchKernelGGL((rms_bwd_kernel<T, TPR, VPL>), dim3(parts), dim3(256), TPR < 256 ? TPR * VPL * 8 * sizeof(float) : 0, st, g); \
        GFS3D_LAUNCH_CHECK("rms_bwd_kernel");                                                                                         \
        return GFS3D_OK;                                                                                                              \
    }
    if (C <= 64) RN_BWD(8, 1)
    if (C <= 128) RN_BWD(16, 1)
    if (C <= 256) RN_BWD(32, 1)
    if (C <= 512) RN_BWD(64, 1)
    if (C <= 1024) RN_BWD(64, 2)
    if (C <= 2048) RN_BWD(256, 1)
    if (C <= 4096) RN_BWD(256, 2)
    if (C <= 8192) RN_BWD(256, 4)
    RN_BWD(256, 8)
#undef RN_BWD
}
constexpr int RN_MAX_C = 16384;

bool rn_aligned(const void *p, long long stride, int esize) { return ((uintptr_t)p & 15) == 0 && stride * esize % 16 == 0; }

int rn_check(const char *who, const gfs3d_rms_norm_args *a)
{
    GFS3D_REQUIRE(a, "%s: NULL args", who);
    GFS3D_REQUIRE(a->type == GFS3D_COMPUTE_F32 || a->type == GFS3D_COMPUTE_BF16 || a->type == GFS3D_COMPUTE_F16,
                  "%s: type must be one of GFS3D_COMPUTE_*", who);
    GFS3D_REQUIRE(a->rows >= 1 && a->C >= 1 && a->C <= RN_MAX_C, "%s: bad shape rows=%lld C=%d (1..%d)", who, a->rows, a->C, RN_MAX_C);
    GFS3D_REQUIRE(a->eps >= 0.f && a->eps < 3e38f, "%s: eps %g", who, (double)a->eps);
    GFS3D_REQUIRE(a->x && a->weight, "%s: NULL buffer", who);
    GFS3D_REQUIRE(a->x_stride >= 0 && a->r_stride >= 0 && a->dy_stride >= 0 && a->ds_stride >= 0, "%s: a negative stride", who);
    return GFS3D_OK;
}

}  // namespace
}  // namespace gfs3d

extern "C" int gfs3d_rotary(const gfs3d_rotary_args *a, void *stream)
{
    const char *who = "gfs3d_rotary";
    GFS3D_REQUIRE(a, "%s: NULL args", who);
    GFS3D_REQUIRE(a->type == GFS3D_COMPUTE_F32 || a->type == GFS3D_COMPUTE_BF16 || a->type == GFS3D_COMPUTE_F16,
                  "%s: type must be one of GFS3D_COMPUTE_*", who);
    GFS3D_REQUIRE(a->B >= 1 && a->N >= 1 && a->D >= 2, "%s: bad shape B=%d N=%d D=%d", who, a->B, a->N, a->D);
    GFS3D_REQUIRE(a->axes >= 1 && a->axes <= 3 && a->pairs >= 1 && (long long)2 * a->axes * a->pairs <= a->D,
                  "%s: %d axes of %d pairs do not fit a head of %d", who, a->axes, a->pairs, a->D);
    GFS3D_REQUIRE(a->axes * a->pairs <= 1024, "%s: %d pairs of a head (at most 1024)", who, a->axes * a->pairs);
    GFS3D_REQUIRE(a->q && a->q_out && a->q_heads >= 1 && (a->k ? a->k_out && a->k_heads >= 1 : a->k_heads == 0), "%s: NULL buffer", who);
    GFS3D_REQUIRE(a->positions && a->freqs && a->position_type >= 0 && a->position_type <= 2, "%s: positions", who);
    RoArgs g{};
    const int es = a->type == GFS3D_COMPUTE_F32 ? 4 : 2, vec = 16 / es;
    bool al = a->D % vec == 0 && (a->interleaved || a->pairs % vec == 0);
    const void *xi[2] = {a->q, a->k};
    void *yo[2] = {a->q_out, a->k_out};
    const long long *si[2] = {a->q_stride, a->k_stride}, *so[2] = {a->q_out_stride, a->k_out_stride};
    for (int w = 0; w < 2; ++w) {
        g.x[w] = xi[w]; g.y[w] = yo[w];
        g.sb[w] = si[w][0]; g.sr[w] = si[w][1]; g.sh[w] = si[w][2];
        g.ob[w] = so[w][0]; g.orr[w] = so[w][1]; g.oh[w] = so[w][2];
        if (!xi[w]) continue;
        al = al && ((uintptr_t)xi[w] & 15) == 0 && ((uintptr_t)yo[w] & 15) == 0;
        for (int e = 0; e < 3; ++e) {
            GFS3D_REQUIRE(si[w][e] >= 0 && so[w][e] >= 0, "%s: a negative stride", who);
            al = al && si[w][e] % vec == 0 && so[w][e] % vec == 0;
        }
    }
    g.heads[0] = a->q_heads; g.heads[1] = a->k_heads;
    g.N = a->N; g.D = a->D; g.axes = a->axes; g.pairs = a->pairs;
    g.tokens = (long long)a->B * a->N;
    g.pos = a->positions; g.pos_type = a->position_type; g.freqs = a->freqs;
    g.magnitude = a->magnitude; g.sign = a->inverse ? -1.f : 1.f;
    g.interleaved = a->interleaved;
    // 16 tokens to a workgroup (8 KB of cosines at 64 pairs) once there are enough for four workgroups on every CU
    const int AP = a->axes * a->pairs, most = 1024 / AP < 16 ? 1024 / AP : 16;
    const long long want = (g.tokens + 1023) / 1024;
    g.tb = (int)(want < 1 ? 1 : want > most ? most : want);
    const long long blocks = (g.tokens + g.tb - 1) / g.tb;
    GFS3D_REQUIRE(blocks * 256 < (1ll << 32) && (long long)g.tb * (g.heads[0] + g.heads[1]) * a->D < (1ll << 31), "%s: too many values", who);
    const int V = al ? vec : 1, W = V > 1 ? V : 2, heads = g.heads[0] + g.heads[1];
    g.per = g.interleaved ? (a->D + W - 1) / W : AP / V + (a->D - 2 * AP + V - 1) / V;
    const long long units = (long long)g.tb * heads * g.per;             // u < 2^32 / d: the product with the rounded-up reciprocal is exact
    auto magic = [&](int d) { return d > 1 && units * d < (1ll << 32) ? (unsigned)(((1ull << 32) + d - 1) / d) : 0u; };
    g.m_per = magic(g.per);
    g.m_heads = magic(heads);
    hipStream_t st = static_cast<hipStream_t>(stream);
    const size_t lds = (size_t)g.tb * AP * sizeof(float2);
#define RO_GO(T, V) hipLaunchKernelGGL((rotary_kernel<T, V>), dim3((unsigned)blocks), dim3(256), lds, st, g)
    if (a->type == GFS3D_COMPUTE_F32) { if (al) RO_GO(float, 4); else RO_GO(float, 1); }
    else if (a->type == GFS3D_COMPUTE_BF16) { if (al) RO_GO(__bf16, 8); else RO_GO(__bf16, 1); }
    else { if (al) RO_GO(_Float16, 8); else RO_GO(_Float16, 1); }
#undef RO_GO
    GFS3D_LAUNCH_CHECK("rotary_kernel");
    return GFS3D_OK;
}

extern "C" int gfs3d_rms_norm_forward(const gfs3d_rms_norm_args *a, void *stream)
{
    const char *who = "gfs3d_rms_norm_forward";
    if (int rc = rn_check(who, a)) return rc;
    GFS3D_REQUIRE(a->y && (!a->residual || a->stream_out) && (!a->fp8 || a->scale), "%s: NULL buffer", who);
    GFS3D_REQUIRE(!a->fp8 || a->group == 0 || ((a->group == 32 || a->group == 64 || a->group == 128) && a->C % a->group == 0),
                  "%s: groups of %d channels in rows of %d (32, 64 or 128, and a divisor)", who, a->group, a->C);
    RnArgs g{};
    const int es = a->type == GFS3D_COMPUTE_F32 ? 4 : 2;
    g.x = a->x; g.r = a->residual; g.w = a->weight; g.s = a->stream_out; g.y = a->y; g.scale = a->scale; g.rstd = a->rstd;
    g.xs = a->x_stride; g.rs = a->r_stride; g.rows = a->rows; g.C = a->C;
    g.rkind = !a->residual ? RN_NONE : a->residual_f32 && a->type != GFS3D_COMPUTE_F32 ? RN_F32 : RN_SAME;
    g.wf32 = a->weight_f32 || a->type == GFS3D_COMPUTE_F32;
    g.group = a->fp8 ? a->group : 0;
    const int re = g.rkind == RN_F32 ? 4 : es;
    g.vec = a->C % 8 == 0 && rn_aligned(a->x, a->x_stride, es) && rn_aligned(a->y, 0, 1) && rn_aligned(a->weight, 0, 1)
            && (!a->residual || (rn_aligned(a->residual, a->r_stride, re) && rn_aligned(a->stream_out, 0, 1)));
    g.eps = a->eps; g.inv_c = 1.f / (float)a->C;
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (a->type == GFS3D_COMPUTE_F32) return rn_forward<float>(g, a->fp8 != 0, st);
    if (a->type == GFS3D_COMPUTE_BF16) return rn_forward<__bf16>(g, a->fp8 != 0, st);
    return rn_forward<_Float16>(g, a->fp8 != 0, st);
}

extern "C" size_t gfs3d_rms_norm_workspace_bytes(long long rows, int C)
{
    return rows >= 1 && C >= 1 && C <= RN_MAX_C ? (size_t)RN_PARTS * C * sizeof(float) : 0;
}

extern "C" int gfs3d_rms_norm_backward(const gfs3d_rms_norm_args *a, void *stream)
{
    const char *who = "gfs3d_rms_norm_backward";
    if (int rc = rn_check(who, a)) return rc;
    GFS3D_REQUIRE(a->rstd && a->dy && (!a->dweight || a->workspace), "%s: NULL buffer", who);
    if (a->dweight && a->workspace_bytes < gfs3d_rms_norm_workspace_bytes(a->rows, a->C)) {
        set_error("%s: workspace too small (%zu)", who, a->workspace_bytes);
        return GFS3D_ERR_WORKSPACE;
    }
    RnArgs g{};
    const int es = a->type == GFS3D_COMPUTE_F32 ? 4 : 2;
    g.x = a->x; g.w = a->weight; g.dy = a->dy; g.ds = a->ds; g.y = a->dx; g.s = a->dresidual; g.rstd = a->rstd;
    g.part = a->dweight ? (float *)a->workspace : nullptr;
    g.xs = a->x_stride; g.dys = a->dy_stride; g.ds_s = a->ds_stride; g.rows = a->rows; g.C = a->C;
    g.rkind = a->residual_f32 && a->type != GFS3D_COMPUTE_F32 ? RN_F32 : RN_SAME;       // the type of x (the stream) and of ds here
    g.wf32 = a->weight_f32 || a->type == GFS3D_COMPUTE_F32;
    const int re = g.rkind == RN_F32 ? 4 : es;
    GFS3D_REQUIRE(!a->dresidual || g.rkind == RN_F32 || a->type == GFS3D_COMPUTE_F32, "%s: dresidual is for an fp32 residual", who);
    g.vec = a->C % 8 == 0 && rn_aligned(a->x, a->x_stride, re) && rn_aligned(a->dy, a->dy_stride, es) && rn_aligned(a->weight, 0, 1)
            && rn_aligned(a->ds, a->ds ? a->ds_stride : 0, re) && rn_aligned(a->dx, 0, 1) && rn_aligned(a->dresidual, 0, 1);
    g.inv_c = 1.f / (float)a->C;
    hipStream_t st = static_cast<hipStream_t>(stream);
    int parts = 0, rc;
    if (a->type == GFS3D_COMPUTE_F32) rc = rn_backward<float>(g, parts, st);
    else if (a->type == GFS3D_COMPUTE_BF16) rc = rn_backward<__bf16>(g, parts, st);
    else rc = rn_backward<_Float16>(g, parts, st);
    if (rc || !a->dweight) return rc;
    const dim3 grid((a->C + 31) / 32);
    if (g.wf32) hipLaunchKernelGGL((rms_dw_kernel<float>), grid, dim3(1024), 0, st, g.part, parts, a->C, (float *)a->dweight);
    else if (a->type == GFS3D_COMPUTE_BF16) hipLaunchKernelGGL((rms_dw_kernel<__bf16>), grid, dim3(1024), 0, st, g.part, parts, a->C, (__bf16 *)a->dweight);
    else hipLaunchKernelGGL((rms_dw_kernel<_Float16>), grid, dim3(1024), 0, st, g.part, parts, a->C, (_Float16 *)a->dweight);
    GFS3D_LAUNCH_CHECK("rms_dw_kernel");
    return GFS3D_OK;
}
