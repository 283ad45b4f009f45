// K7: attention with a sliding window and a few first tokens that stay visible (sinks), over serialised points
//
//     o_i = sum_j p_ij v_j,   p_i. = softmax over the visible j of  scale q_i . k_j
//     j visible to i:  i, j < length  and  j <= i + right  and  (j >= i - left  or  j < sinks)
//
// q (B, N, H, D), k / v (B, N, G, D) point-major with any strides, head h reads key head h / (H / G); fp32, bf16 or half.
// Part of attention.hip (the operand images and the transposed LDS read are those of K5 there).
//
// Forward: a wave owns one unit = 32 queries of one head (the QUERY on the lane, S^T = K Q^T, so that a query's running maximum,
// sum and accumulators are in-lane), the four or eight waves of a workgroup own consecutive units with the heads of one key head innermost:
// they share every staged key tile.  Tiles outside all of their windows are never staged, tiles outside a wave's own window cost it
// nothing but the barrier, and only tiles that a window edge, the diagonal or the length cuts pay for the element mask.
// Backward: dQ with the query on the lane (it also leaves delta_i = dout_i . o_i), dK / dV with the key on the lane, looping over the
// heads of the key head; what the sinks receive from queries beyond their window (all rows of a long sequence) is summed by
// its own kernel in row chunks, the chunks are added in order by another, and their sum joins where dK / dV of those keys are
// written.  No atomics.
// Scores, softmax statistics, accumulators and all sums over heads or chunks are fp32.  Probabilities and dS are rounded to the operand
// type of the matrix cores: bf16 / half for those tensors, exact 3-way bf16 splits (PREC_X6) for fp32; the gradients of half
// tensors take two bf16 pieces (PREC_X3), whose range is fp32's - a mean loss underflows in half.
// Measured (2 x 65536 rows, 8 heads x 64, 512 to either side + 16 sinks; medians of a warm device, three cards): bf16 forward 400 - 427 us
// (0.65 - 0.70 PFLOP/s of visible pairs), dQ 540 - 575 (0.73 - 0.77), dK / dV 730 - 776 (0.72 - 0.76), sinks 71; half 402, 1100, 1520, 136 (three
// products for one in the backward) on the fastest of them; fp32, a quarter of the rows: 395, 516, 663, 58.  In the bf16 forward the vector pipe is busy 64 % of the time, the matrix pipe 32 %, and
// 30 % of the LDS's active cycles are bank conflicts; four waves per SIMD (128 registers) did better than every form that overlaps the
// pipes within a wave at two.  Head sizes other than 32, 64 and 128 are padded to the next of them in every product, and their loads
// are masked by channel (7 x 1777 rows x 6 / 2 heads, forward: 40 channels 61.5 us, 64 channels 61; 80 and 96 channels 127, as 128).

namespace gfs3d {
namespace {

struct WaStride { long long b, r, h; };          // elements between sequences, rows, heads
struct WaArgs {
    const void *q, *k, *v, *out, *dout;
    void *low;                                    // (B, N, H, D) what rounding took from out (16-bit types): delta is formed from both
    WaStride qs, ks, vs, gs;                      // gs: dout
    const int *lengths;                           // (B) device, or NULL: all S
    float *lse, *delta;                           // (B, H, N): log2-sum-exp2 of the scaled scores; dout . out
    float *part, *part2;                          // partial sums: sinks' gradients / split keys; split rows of dK, dV
    int B, N, S, H, G, HG, D;                     // N query rows, S keys per sequence
    int left, right, sinks;
    int nblk;                                     // workgroups per (sequence, key head)
    int nst, nchunk, nsplit;                      // sinks' key tiles, row chunks of their gradient; row chunks of dK, dV
    float scale, c;                               // c = scale log2(e)
};

template <class T> struct WaT;
template <> struct WaT<float> { static constexpr int PF = PREC_X6, PB = PREC_X6; };
template <> struct WaT<__bf16> { static constexpr int PF = PREC_BF16, PB = PREC_BF16; };
template <> struct WaT<_Float16> { static constexpr int PF = PREC_F16, PB = PREC_X3; };
// keys of a staged tile in the forward (eight waves, 128 channels: 4 x 8192 rows x 16 / 4 heads half, causal over 2048: 568 us with 128 keys, 593
// with 64; 64 channels: no difference)
template <class T, int DP, int NW> constexpr int WA_KT = sizeof(T) == 4 ? 32 : NW == 8 && DP == 128 ? 128 : 64;

// eight consecutive channels as they lie in memory
template <class T> struct WaRaw { uint4 a; };
template <> struct WaRaw<float> { float4 a, b; };
template <class T> __device__ __forceinline__ WaRaw<T> wa_zero() { return WaRaw<T>{make_uint4(0u, 0u, 0u, 0u)}; }
template <> __device__ __forceinline__ WaRaw<float> wa_zero<float>() { return WaRaw<float>{make_float4(0.f, 0.f, 0.f, 0.f), make_float4(0.f, 0.f, 0.f, 0.f)}; }
template <class T> __device__ __forceinline__ WaRaw<T> wa_load8(const T *p) { return *reinterpret_cast<const WaRaw<T> *>(p); }
template <class T> __device__ __forceinline__ void wa_floats(const WaRaw<T> &r, float (&v)[8])
{
    if constexpr (sizeof(T) == 4) {
        v[0] = r.a.x; v[1] = r.a.y; v[2] = r.a.z; v[3] = r.a.w; v[4] = r.b.x; v[5] = r.b.y; v[6] = r.b.z; v[7] = r.b.w;
    } else {
        typedef T Tx8 __attribute__((ext_vector_type(8)));
        const Tx8 x = __builtin_bit_cast(Tx8, r.a);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = (float)x[e];
    }
}
template <class T, int PREC> __device__ __forceinline__ void wa_pieces(const WaRaw<T> &r, uint4 (&f)[Mx<PREC>::NP])
{
    if constexpr (sizeof(T) == 2 && Mx<PREC>::NP == 1) {
        f[0] = r.a;
    } else {
        float v[8];
        wa_floats<T>(r, v);
        mm_pieces8<PREC>(v, f);
    }
}
template <class T> __device__ __forceinline__ void wa_store4(T *p, float a, float b, float c, float d)
{
    if constexpr (sizeof(T) == 4) *reinterpret_cast<float4 *>(p) = make_float4(a, b, c, d);
    else {
        constexpr int P = WaT<T>::PF;
        *reinterpret_cast<uint2 *>(p) = make_uint2(mm_pack2<P>(a, b), mm_pack2<P>(c, d));
    }
}

// images: [plane][row][2 DP bytes | 16 pad]: the pad turns 16 consecutive rows of one 16-byte column onto 64 different banks
template <int DP> struct WaImg {
    static constexpr int ROWB = 2 * DP + 16;
    template <int R> static constexpr int plane() { return R * ROWB; }
};
template <int PREC, int DP, int R>
__device__ __forceinline__ void wa_rowfrag(const unsigned char *img, int j, int h, int kb, uint4 (&f)[Mx<PREC>::NP])
{
#pragma unroll
    for (int p = 0; p < Mx<PREC>::NP; ++p)
        f[p] = *reinterpret_cast<const uint4 *>(img + p * WaImg<DP>::template plane<R>() + j * WaImg<DP>::ROWB + 32 * kb + 16 * h);
}
// rows = channels 32 dt + (lane & 31), k-step s: positions at_drow(8 s + e, h) of the 32 rows at `img` (see at_trfrag)
template <int PREC, int DP, int R>
__device__ __forceinline__ void wa_trfrag(const unsigned char *img, int lane, int dt, int s, uint4 (&f)[Mx<PREC>::NP])
{
    constexpr int ROWB = WaImg<DP>::ROWB;
    const int h = lane >> 5, g1 = (lane >> 4) & 1, q = (lane >> 2) & 3, p4 = lane & 3;
    const unsigned char *base = img + (16 * s + 4 * h + q) * ROWB + 2 * (32 * dt + 16 * g1 + 4 * p4);
#pragma unroll
    for (int p = 0; p < Mx<PREC>::NP; ++p) {
        const unsigned char *bp = base + p * WaImg<DP>::template plane<R>();
        const at_s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((at_lds_s16x4 *)(bp));
        const at_s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((at_lds_s16x4 *)(bp + 8 * ROWB));
        const uint2 a = __builtin_bit_cast(uint2, lo), b = __builtin_bit_cast(uint2, hi);
        f[p] = make_uint4(a.x, a.y, b.x, b.y);
    }
}
// the per-wave constant operand: lane (column, half h) holds channels 16 kb + 8 h .. of its row (zeros past D or where !ok)
template <class T, int PREC, int DP>
__device__ __forceinline__ void wa_colfrags(const T *row, bool ok, int D, int h, uint4 (&f)[DP / 16][Mx<PREC>::NP])
{
#pragma unroll
    for (int kb = 0; kb < DP / 16; ++kb) {
        const int ch = 16 * kb + 8 * h;
        WaRaw<T> r = wa_zero<T>();
        if (ok && ch < D) r = wa_load8<T>(row + ch);
        wa_pieces<T, PREC>(r, f[kb]);
    }
}

// The per-wave operands are loaded before a loop whose own loads are still in flight when they are used: having them arrive here
// keeps the compiler from waiting, in every turn, for everything that is in flight
template <int A, int B> __device__ __forceinline__ void wa_settle(uint4 (&f)[A][B])
{
#pragma unroll
    for (int a = 0; a < A; ++a)
#pragma unroll
        for (int b = 0; b < B; ++b) asm volatile("" : "+v"(f[a][b].x), "+v"(f[a][b].y), "+v"(f[a][b].z), "+v"(f[a][b].w));
}

// R rows of a (rows, D) matrix staged by NT threads: thread t takes the 8-channel chunks t, t + NT, ..  A chunk's place relative to the
// tile's first row is fixed: 32-bit offsets from a base that is the same for all threads (scalar), no address arithmetic per tile
template <class T, int DP, int R, int NT> struct WaStage {
    static constexpr int CPR = DP / 8, NCH = (R * CPR + NT - 1) / NT;
    static constexpr bool RAGGED = R * CPR % NT != 0;
    WaRaw<T> r[NCH];
    unsigned off[NCH];
    __device__ __forceinline__ void init(long long stride, int t)
    {
#pragma unroll
        for (int n = 0; n < NCH; ++n) {
            const int c = t + n * NT;
            off[n] = RAGGED && c >= R * CPR ? 0u : (unsigned)(c / CPR) * (unsigned)(stride * sizeof(T)) + (unsigned)(c % CPR) * (unsigned)(8 * sizeof(T));
        }
    }
    // the R rows from `base` on; of them `left` are there, rows behind and channels >= D read as zeros
    __device__ __forceinline__ void load(const T *base, int left, int D, int t)
    {
        const char *p = reinterpret_cast<const char *>(base);
        if (left >= R && D == DP) {
#pragma unroll
            for (int n = 0; n < NCH; ++n) r[n] = *reinterpret_cast<const WaRaw<T> *>(p + off[n]);
        } else {
#pragma unroll
            for (int n = 0; n < NCH; ++n) {
                const int c = t + n * NT;
                r[n] = wa_zero<T>();
                if ((!RAGGED || c < R * CPR) && c / CPR < left && 8 * (c % CPR) < D) r[n] = *reinterpret_cast<const WaRaw<T> *>(p + off[n]);
            }
        }
    }
    template <int PREC> __device__ __forceinline__ void put(unsigned char *img, int t) const
    {
#pragma unroll
        for (int n = 0; n < NCH; ++n) {
            const int c = t + n * NT, row = c / CPR, ch = c % CPR;
            uint4 f[Mx<PREC>::NP];
            wa_pieces<T, PREC>(r[n], f);
            if (!RAGGED || c < R * CPR) {
#pragma unroll
                for (int p = 0; p < Mx<PREC>::NP; ++p)
                    *reinterpret_cast<uint4 *>(img + p * WaImg<DP>::template plane<R>() + row * WaImg<DP>::ROWB + 16 * ch) = f[p];
            }
        }
    }
};

// (x of the lower half, x of the upper half) in every lane: one register's upper half changes places with another's lower half
__device__ __forceinline__ float2 wa_halves(float x)
{
    const unsigned a = __builtin_bit_cast(unsigned, x);
    const auto r = __builtin_amdgcn_permlane32_swap(a, a, false, false);
    const unsigned lo = r[0], hi = r[1];              // (a bit cast of r[1] itself reads r[0])
    return make_float2(__builtin_bit_cast(float, lo), __builtin_bit_cast(float, hi));
}
__device__ __forceinline__ float wa_max32(float x) { const float2 r = wa_halves(x); return fmaxf(r.x, r.y); }
__device__ __forceinline__ float wa_sum32(float x) { const float2 r = wa_halves(x); return r.x + r.y; }
__device__ __forceinline__ int wa_length(const int *lengths, int b, int S) { return lengths ? min(max(lengths[b], 0), S) : S; }
// workgroups go to the 8 XCDs in turn: give each XCD (its own L2) a contiguous run, so that neighbours share their key tiles there
__device__ __forceinline__ unsigned wa_order(unsigned id, unsigned total)
{
    const unsigned per = total / 8, x = id & 7;
    return id < per * 8 ? x * per + id / 8 : id;
}
constexpr float WA_LAZY = 8.f;        // the running maximum may lag the true one by 2^8: p, its sum and its products stay in range in fp32 and half

// A wave's 32 x DP result (C/D registers: column = row of the output, registers = channels) to memory in whole 16-byte pieces of
// rows, through the wave's own part of LDS: straight from the registers a row would be written in 8-byte pieces by two lanes
template <class T, int DP> constexpr int WA_OUT = 32 * (DP * (int)sizeof(T) + 16);
template <class T, int DP>
__device__ __forceinline__ void wa_store_rows(unsigned char *lds, const f32x16 (&X)[DP / 32], float f, int lane, T *out, size_t stride, int rows, int D)
{
    constexpr int RB = DP * (int)sizeof(T) + 16, V = 16 / (int)sizeof(T), PR = DP / V, RPI = 64 / PR;
    const int j = lane & 31, h = lane >> 5;
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int r = 0; r < 16; r += 4)
            wa_store4<T>(reinterpret_cast<T *>(lds + j * RB) + 32 * d + at_drow(r, h), X[d][r] * f, X[d][r + 1] * f, X[d][r + 2] * f, X[d][r + 3] * f);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");       // LDS serves a wave in order
    __builtin_amdgcn_wave_barrier();
    const int ch = lane % PR * V;
#pragma unroll
    for (int n = 0; n < 32 / RPI; ++n) {
        const int row = n * RPI + lane / PR;
        const uint4 x = *reinterpret_cast<const uint4 *>(lds + row * RB + lane % PR * 16);
        if (row < rows && ch < D) *reinterpret_cast<uint4 *>(out + row * stride + ch) = x;
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// Hides what the lane does not see among the 32 rows from j0 on in its C/D registers: x[r] = fill unless row j = j0 + at_drow(r, h)
// has lo <= j <= hi, or j < far (FAR: the sinks the lane sees).  One unsigned comparison per element for the window (hi >= lo - 1).
template <bool FAR, class X> __device__ __forceinline__ void wa_mask(int j0, int h, int lo, int hi, int far, float fill, X &x)
{
    asm volatile("");                                 // keeps the branch around it: as selects the mask cost every tile its arithmetic
    const int base = j0 + 4 * h - lo, fb = far - j0 - 4 * h;
    const unsigned n = (unsigned)(hi - lo + 1);
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        float y = (unsigned)(base + at_drow(r, 0)) < n ? x[r] : fill;
        if (FAR) y = at_drow(r, 0) < fb ? x[r] : y;
        x[r] = y;
    }
}

// ------------------------------------------------------------------ forward
// 32 keys of the staged tile, from Kc / Vc on (keys j0 ..): scores, running softmax, products.  `whole`: every key is seen.  The
// running maximum follows only when a row's has grown by WA_LAZY (in base 2): most tiles then leave the accumulators alone
template <class T, int DP, int KT>
__device__ __forceinline__ void wa_fwd_tile(const unsigned char *Kc, const unsigned char *Vc, int j0, int lane, float c, float thr, bool whole,
                                            int lo, int hi, int far, const uint4 (&qp)[DP / 16][Mx<WaT<T>::PF>::NP], float &m, float &mc,
                                            float &l, f32x16 (&O)[DP / 32])
{
    constexpr int PREC = WaT<T>::PF, NP = Mx<PREC>::NP, ND = DP / 32;
    const int j = lane & 31, h = lane >> 5;
    f32x16 acc;
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[r] = 0.f;
#pragma unroll
    for (int kb = 0; kb < DP / 16; ++kb) {
        uint4 ak[NP];
        wa_rowfrag<PREC, DP, KT>(Kc, j, h, kb, ak);
        mm_mac<PREC>(ak, qp[kb], acc);
    }
    if (!whole) {
        if (j0 >= far) wa_mask<false>(j0, h, lo, hi, 0, -__builtin_inff(), acc);
        else wa_mask<true>(j0, h, lo, hi, min(far, hi + 1), -__builtin_inff(), acc);
    }
    float tmax = acc[0];
#pragma unroll
    for (int r = 0; r < 16; ++r) tmax = fmaxf(tmax, acc[r]);
    tmax = wa_max32(tmax);
    if (__ballot(tmax > m + thr) != 0ull) {
        const float m_new = fmaxf(m, tmax), mc_new = m_new == -__builtin_inff() ? 0.f : m_new * c;
        const float sc = m == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(mc - mc_new);
        m = m_new;
        mc = mc_new;
        l *= sc;
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r) O[d][r] *= sc;
    }
    float pd[16];
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        pd[r] = __builtin_amdgcn_exp2f(fmaf(acc[r], c, -mc));
        l += pd[r];
    }
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
        uint4 pp[NP], av[NP];
        at_regfrag<PREC>(pd, ks, pp);
#pragma unroll
        for (int d = 0; d < ND; ++d) {
            wa_trfrag<PREC, DP, KT>(Vc, lane, d, ks, av);
            mm_mac<PREC>(av, pp, O[d]);
        }
    }
}
template <class T, int DP, int NW>
__global__ void __launch_bounds__(64 * NW, DP == 128 ? (sizeof(T) == 4 ? 1 : 2) : sizeof(T) == 4 ? 3 : 4) wa_fwd_kernel(const WaArgs g, T *__restrict__ out)
{
    constexpr int PREC = WaT<T>::PF, NP = Mx<PREC>::NP, KT = (WA_KT<T, DP, NW>), SUB = KT / 32, IMG = NP * KT * WaImg<DP>::ROWB;
    constexpr int ROWB = WaImg<DP>::ROWB, ND = DP / 32;
    extern __shared__ __attribute__((aligned(16))) unsigned char at_smem[];
    unsigned char *Kimg = at_smem, *Vimg = at_smem + 2 * IMG;
    const int t = threadIdx.x, lane = t & 63, wv = __builtin_amdgcn_readfirstlane(t >> 6), j = lane & 31, h = lane >> 5;
    const unsigned bid = wa_order(blockIdx.x, gridDim.x);
    const int blk = bid % g.nblk, bg = bid / g.nblk, b = bg / g.G, gi = bg % g.G;
    const int len = wa_length(g.lengths, b, g.N), nqt = (g.N + 31) / 32;
    const int u = blk * NW + wv, qt = u / g.HG, head = gi * g.HG + u % g.HG, q0 = qt * 32, qi = q0 + j;
    const bool live = q0 < len;                         // this wave has rows (qt < nqt follows)
    const int qa = blk * NW / g.HG * 32, qb = min((blk * NW + NW - 1) / g.HG, nqt - 1) * 32 + 31;       // the workgroup's rows
    const T *kb_ = (const T *)g.k + b * g.ks.b + gi * g.ks.h, *vb = (const T *)g.v + b * g.vs.b + gi * g.vs.h;

    uint4 qp[DP / 16][NP];
    wa_colfrags<T, PREC, DP>((const T *)g.q + b * g.qs.b + (long long)qi * g.qs.r + head * g.qs.h, qi < len, g.D, h, qp);
    float m = -__builtin_inff(), mc = 0.f, l = 0.f;      // running maximum (raw scores), c m (0 while there is none), this half's sum
    f32x16 O[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) O[d][r] = 0.f;

    const int tlo = max(0, qa - g.left) / KT, thi = min(len - 1, qb + g.right) / KT;
    const int nsink = min((min(g.sinks, len) + KT - 1) / KT, tlo);
    const int nt = qa < len ? nsink + thi - tlo + 1 : 0;
    const int wlo = max(0, q0 - g.left), whi = min(len - 1, q0 + 31 + g.right), far = min(g.sinks, len);
    const int hi = min(len - 1, qi + g.right), lo = min(qi - g.left, hi + 1);
    const float thr = WA_LAZY / g.c;
    WaStage<T, DP, KT, 64 * NW> sk, sv;
    sk.init(g.ks.r, t);
    sv.init(g.vs.r, t);
    auto row0 = [&](int tt) { return (tt < nsink ? tt : tlo + tt - nsink) * KT; };
    auto load = [&](int tt) {
        const int r0 = row0(tt);
        sk.load(kb_ + (long long)r0 * g.ks.r, len - r0, g.D, t);
        sv.load(vb + (long long)r0 * g.vs.r, len - r0, g.D, t);
    };
    if (nt > 0) {
        load(0);
        sk.template put<PREC>(Kimg, t);
        sv.template put<PREC>(Vimg, t);
    }
    wa_settle(qp);
    __syncthreads();
    for (int tt = 0; tt < nt; ++tt) {
        const int cur = tt & 1, j0 = row0(tt);
        const unsigned char *Kc = Kimg + cur * IMG, *Vc = Vimg + cur * IMG;
        if (tt + 1 < nt) load(tt + 1);
        if (live) {
            // the subtiles that hold a key of this wave's window, or a sink
            auto holds = [&](int jj) { return jj <= whi && (jj + 32 > wlo || jj < far); };
            auto whole = [&](int jj, int n) { return jj + n <= len && jj + n - 1 <= q0 + g.right && (jj >= q0 + 31 - g.left || jj + n <= g.sinks); };
#pragma unroll
            for (int s = 0; s < 32 * SUB; s += 32)
                if (holds(j0 + s))
                    wa_fwd_tile<T, DP, KT>(Kc + s * ROWB, Vc + s * ROWB, j0 + s, lane, g.c, thr, whole(j0 + s, 32), lo, hi, far, qp, m, mc, l, O);
        }
        if (tt + 1 < nt) { sk.template put<PREC>(Kimg + (cur ^ 1) * IMG, t); sv.template put<PREC>(Vimg + (cur ^ 1) * IMG, t); }
        __syncthreads();
    }
    const float lt = wa_sum32(l), inv = lt > 0.f && qi < len ? 1.f / lt : (lt != lt ? lt : 0.f);
    if (qt < nqt) {
        const size_t o = (((size_t)b * g.N + q0) * g.H + head) * g.D;
        wa_store_rows<T, DP>(at_smem + wv * WA_OUT<T, DP>, O, inv, lane, out + o, (size_t)g.H * g.D, g.N - q0, g.D);
        if constexpr (sizeof(T) == 2) {
            if (g.low) {
#pragma unroll
                for (int d = 0; d < ND; ++d)
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        const float x = O[d][r] * inv;
                        O[d][r] = x - (float)(T)x;
                    }
                wa_store_rows<T, DP>(at_smem + wv * WA_OUT<T, DP>, O, 1.f, lane, (T *)g.low + o, (size_t)g.H * g.D, g.N - q0, g.D);
            }
        }
        if (qi < g.N && g.lse && h == 0) g.lse[((size_t)b * g.H + head) * g.N + qi] = lt > 0.f && qi < len ? mc + __builtin_amdgcn_logf(lt) : __builtin_inff();
    }
}

// ------------------------------------------------------------------ backward, query side: dQ and delta
template <class T, int DP>
__global__ void __launch_bounds__(256, DP == 128 && sizeof(T) == 4 ? 1 : 2) wa_bwd_dq_kernel(const WaArgs g, T *__restrict__ dq)
{
    constexpr int NW = 4;
    constexpr int PREC = WaT<T>::PB, NP = Mx<PREC>::NP, KT = 32, IMG = NP * KT * WaImg<DP>::ROWB, ND = DP / 32;
    extern __shared__ __attribute__((aligned(16))) unsigned char at_smem[];
    unsigned char *Kimg = at_smem, *Vimg = at_smem + 2 * IMG;
    const int t = threadIdx.x, lane = t & 63, wv = __builtin_amdgcn_readfirstlane(t >> 6), j = lane & 31, h = lane >> 5;
    const unsigned bid = wa_order(blockIdx.x, gridDim.x);
    const int blk = bid % g.nblk, bg = bid / g.nblk, b = bg / g.G, gi = bg % g.G;
    const int len = wa_length(g.lengths, b, g.N), nqt = (g.N + 31) / 32;
    const int u = blk * NW + wv, qt = u / g.HG, head = gi * g.HG + u % g.HG, q0 = qt * 32, qi = q0 + j;
    const bool live = q0 < len, mine = qi < len;
    const int qa = blk * NW / g.HG * 32, qb = min((blk * NW + NW - 1) / g.HG, nqt - 1) * 32 + 31;
    const T *kb_ = (const T *)g.k + b * g.ks.b + gi * g.ks.h, *vb = (const T *)g.v + b * g.vs.b + gi * g.vs.h;

    uint4 qp[DP / 16][NP], gp[DP / 16][NP];
    wa_colfrags<T, PREC, DP>((const T *)g.q + b * g.qs.b + (long long)qi * g.qs.r + head * g.qs.h, mine, g.D, h, qp);
    float dl = 0.f;
    {
        const T *grow = (const T *)g.dout + b * g.gs.b + (long long)qi * g.gs.r + head * g.gs.h;
        const T *orow = (const T *)g.out + (((size_t)b * g.N + qi) * g.H + head) * g.D, *lrow = (const T *)g.low + (((size_t)b * g.N + qi) * g.H + head) * g.D;
#pragma unroll
        for (int kb = 0; kb < DP / 16; ++kb) {
            const int ch = 16 * kb + 8 * h;
            WaRaw<T> rg = wa_zero<T>(), ro = wa_zero<T>();
            if (mine && ch < g.D) { rg = wa_load8<T>(grow + ch); ro = wa_load8<T>(orow + ch); }
            float fg[8], fo[8];
            wa_floats<T>(rg, fg);
            wa_floats<T>(ro, fo);
            if constexpr (sizeof(T) == 2) {
                if (g.low) {
                    WaRaw<T> rl = wa_zero<T>();
                    if (mine && ch < g.D) rl = wa_load8<T>(lrow + ch);
                    float fl[8];
                    wa_floats<T>(rl, fl);
#pragma unroll
                    for (int e = 0; e < 8; ++e) fo[e] += fl[e];
                }
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) dl = fmaf(fg[e], fo[e], dl);
            wa_pieces<T, PREC>(rg, gp[kb]);
        }
        dl = wa_sum32(dl);
    }
    const size_t row = ((size_t)b * g.H + head) * g.N + qi;
    const float Lq = mine ? g.lse[row] : __builtin_inff();
    if (qi < g.N && qt < nqt && h == 0) g.delta[row] = dl;
    f32x16 A[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) A[d][r] = 0.f;

    const int tlo = max(0, qa - g.left) / KT, thi = min(len - 1, qb + g.right) / KT;
    const int nsink = min((min(g.sinks, len) + KT - 1) / KT, tlo);
    const int nt = qa < len ? nsink + thi - tlo + 1 : 0;
    const int wlo = max(0, q0 - g.left), whi = min(len - 1, q0 + 31 + g.right), far = min(g.sinks, len);
    const int hi = mine ? min(len - 1, qi + g.right) : -1, lo = mine ? min(qi - g.left, hi + 1) : 0;      // rows behind the length see nothing
    WaStage<T, DP, KT, 64 * NW> sk, sv;
    sk.init(g.ks.r, t);
    sv.init(g.vs.r, t);
    auto row0 = [&](int tt) { return (tt < nsink ? tt : tlo + tt - nsink) * KT; };
    auto load = [&](int tt) {
        const int r0 = row0(tt);
        sk.load(kb_ + (long long)r0 * g.ks.r, len - r0, g.D, t);
        sv.load(vb + (long long)r0 * g.vs.r, len - r0, g.D, t);
    };
    if (nt > 0) {
        load(0);
        sk.template put<PREC>(Kimg, t);
        sv.template put<PREC>(Vimg, t);
    }
    wa_settle(qp);
    wa_settle(gp);
    float Lw = Lq;
    asm volatile("" : "+v"(Lw));
    __syncthreads();
    for (int tt = 0; tt < nt; ++tt) {
        const int cur = tt & 1, j0 = row0(tt);
        const unsigned char *Kc = Kimg + cur * IMG, *Vc = Vimg + cur * IMG;
        if (tt + 1 < nt) load(tt + 1);
        if (live && j0 <= whi && (j0 + KT > wlo || j0 < g.sinks)) {
            f32x16 acc, dp;
#pragma unroll
            for (int r = 0; r < 16; ++r) { acc[r] = 0.f; dp[r] = 0.f; }
#pragma unroll
            for (int kb = 0; kb < DP / 16; ++kb) {
                uint4 ak[NP], av[NP];
                wa_rowfrag<PREC, DP, KT>(Kc, j, h, kb, ak);
                wa_rowfrag<PREC, DP, KT>(Vc, j, h, kb, av);
                mm_mac<PREC>(ak, qp[kb], acc);
                mm_mac<PREC>(av, gp[kb], dp);
            }
            float ds[16];
#pragma unroll
            for (int r = 0; r < 16; ++r) ds[r] = __builtin_amdgcn_exp2f(fmaf(acc[r], g.c, -Lw)) * (dp[r] - dl);
            if (!(j0 + KT <= len && q0 + 32 <= len && j0 + KT - 1 <= q0 + g.right && (j0 >= q0 + 31 - g.left || j0 + KT <= g.sinks)))
            {
                if (j0 >= far) wa_mask<false>(j0, h, lo, hi, 0, 0.f, ds);
                else wa_mask<true>(j0, h, lo, hi, min(far, hi + 1), 0.f, ds);
            }
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                uint4 dsp[NP], ak[NP];
                at_regfrag<PREC>(ds, s, dsp);
#pragma unroll
                for (int d = 0; d < ND; ++d) {
                    wa_trfrag<PREC, DP, KT>(Kc, lane, d, s, ak);
                    mm_mac<PREC>(ak, dsp, A[d]);
                }
            }
        }
        if (tt + 1 < nt) { sk.template put<PREC>(Kimg + (cur ^ 1) * IMG, t); sv.template put<PREC>(Vimg + (cur ^ 1) * IMG, t); }
        __syncthreads();
    }
    if (qt < nqt)
        wa_store_rows<T, DP>(at_smem + wv * WA_OUT<T, DP>, A, g.scale, lane, dq + (((size_t)b * g.N + q0) * g.H + head) * g.D, (size_t)g.H * g.D, g.N - q0, g.D);
}


// one 32-query tile against the wave's 32 keys: K += dS^T q, V += P^T dout (unscaled).  SINK: pairs beyond the window (j < sinks,
// j < i - left), otherwise the window's
template <class T, int PREC, int DP, int R, bool SINK>
__device__ __forceinline__ void wa_dkv_tile(const WaArgs &g, const unsigned char *Qc, const unsigned char *Gc, const float *Ls, const float *Ds,
                                            int p0, int k0, int len, int lane, const uint4 (&kp)[DP / 16][Mx<PREC>::NP],
                                            const uint4 (&vp)[DP / 16][Mx<PREC>::NP], f32x16 (&AK)[DP / 32], f32x16 (&AV)[DP / 32])
{
    constexpr int NP = Mx<PREC>::NP, ND = DP / 32;
    const int j = lane & 31, h = lane >> 5, ki = k0 + j;
    f32x16 acc, dp;
#pragma unroll
    for (int r = 0; r < 16; ++r) { acc[r] = 0.f; dp[r] = 0.f; }
#pragma unroll
    for (int kb = 0; kb < DP / 16; ++kb) {
        uint4 aq[NP], ag[NP];
        wa_rowfrag<PREC, DP, R>(Qc, j, h, kb, aq);
        wa_rowfrag<PREC, DP, R>(Gc, j, h, kb, ag);
        mm_mac<PREC>(aq, kp[kb], acc);
        mm_mac<PREC>(ag, vp[kb], dp);
    }
    float pd[16], ds[16];
#pragma unroll
    for (int r4 = 0; r4 < 16; r4 += 4) {
        const float4 L4 = *reinterpret_cast<const float4 *>(Ls + at_drow(r4, h)), D4 = *reinterpret_cast<const float4 *>(Ds + at_drow(r4, h));
        const float lv[4] = {L4.x, L4.y, L4.z, L4.w}, dv[4] = {D4.x, D4.y, D4.z, D4.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            pd[r4 + e] = __builtin_amdgcn_exp2f(fmaf(acc[r4 + e], g.c, -lv[e]));
            ds[r4 + e] = pd[r4 + e] * (dp[r4 + e] - dv[e]);
        }
    }
    const bool whole = SINK ? p0 + 32 <= len && k0 + 32 <= min(g.sinks, len) && k0 + 31 < p0 - g.left
                            : p0 + 32 <= len && k0 + 32 <= len && k0 + 31 <= p0 + g.right && k0 >= p0 + 31 - g.left;
    if (!whole) {
        // rows that see the lane's key: ki - right <= i <= ki + left, or those beyond the window of a sink
        const bool on = ki < len && (!SINK || ki < g.sinks);
        const int hi = !on ? -1 : SINK ? len - 1 : min(len - 1, ki + g.left), lo = !on ? 0 : min(SINK ? ki + g.left + 1 : ki - g.right, hi + 1);
        wa_mask<false>(p0, h, lo, hi, 0, 0.f, pd);
        wa_mask<false>(p0, h, lo, hi, 0, 0.f, ds);
    }
#pragma unroll
    for (int s = 0; s < 2; ++s) {
        uint4 bp[NP], bs[NP], af[NP];
        at_regfrag<PREC>(pd, s, bp);
        at_regfrag<PREC>(ds, s, bs);
#pragma unroll
        for (int d = 0; d < ND; ++d) {
            wa_trfrag<PREC, DP, R>(Gc, lane, d, s, af);
            mm_mac<PREC>(af, bp, AV[d]);
            wa_trfrag<PREC, DP, R>(Qc, lane, d, s, af);
            mm_mac<PREC>(af, bs, AK[d]);
        }
    }
}

// ------------------------------------------------------------------ backward, key side: dK, dV
// The turns of a workgroup - (head of the key head, QT rows), heads outermost - are dealt to nsplit workgroups where there would be too
// few; they leave fp32 sums in part2[chunk][dK | dV][B N G D] for wa_bwd_join_kernel.
template <class T, int DP> constexpr int WA_QT = Mx<WaT<T>::PB>::NP == 1 ? 64 : 32;      // query rows staged per turn
template <class T, int DP>
__global__ void __launch_bounds__(256, DP == 128 ? 1 : 2) wa_bwd_dkv_kernel(const WaArgs g, T *__restrict__ dk, T *__restrict__ dv)
{
    constexpr int PREC = WaT<T>::PB, NP = Mx<PREC>::NP, QT = WA_QT<T, DP>, IMG = NP * QT * WaImg<DP>::ROWB, ND = DP / 32, ROWB = WaImg<DP>::ROWB;
    extern __shared__ __attribute__((aligned(16))) unsigned char at_smem[];
    unsigned char *Qimg = at_smem, *Gimg = at_smem + 2 * IMG;
    float (*Ls)[QT] = reinterpret_cast<float (*)[QT]>(at_smem + 4 * IMG), (*Ds)[QT] = Ls + 2;       // [2][QT] each
    const int t = threadIdx.x, lane = t & 63, wv = __builtin_amdgcn_readfirstlane(t >> 6), j = lane & 31, h = lane >> 5;
    const unsigned bid = wa_order(blockIdx.x, gridDim.x);
    const int chunk = bid % g.nsplit, blk = bid / g.nsplit % g.nblk, bg = bid / g.nsplit / g.nblk, b = bg / g.G, gi = bg % g.G;
    const int len = wa_length(g.lengths, b, g.N), kt = blk * 4 + wv, k0 = kt * 32, ki = k0 + j;
    const int ka = blk * 128, kz = min(ka + 127, len - 1);

    uint4 kp[DP / 16][NP], vp[DP / 16][NP];
    wa_colfrags<T, PREC, DP>((const T *)g.k + b * g.ks.b + (long long)ki * g.ks.r + gi * g.ks.h, ki < len, g.D, h, kp);
    wa_colfrags<T, PREC, DP>((const T *)g.v + b * g.vs.b + (long long)ki * g.vs.r + gi * g.vs.h, ki < len, g.D, h, vp);
    f32x16 AK[ND], AV[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) { AK[d][r] = 0.f; AV[d][r] = 0.f; }

    const int tlo = max(0, ka - g.right) / QT, thi = min(len - 1, kz + g.left) / QT, per = thi - tlo + 1, all = ka < len ? per * g.HG : 0;
    const int t0 = (int)((long long)all * chunk / g.nsplit), nt = (int)((long long)all * (chunk + 1) / g.nsplit) - t0;
    int hd = nt > 0 ? t0 / per : 0, rt = nt > 0 ? tlo + t0 % per : 0, p0 = rt * QT;       // hd, rt: of the turn to be loaded next
    WaStage<T, DP, QT, 256> sq, sg;
    sq.init(g.qs.r, t);
    sg.init(g.gs.r, t);
    float l1 = 0.f;
    auto load = [&]() {
        const int head = gi * g.HG + hd, r0 = rt * QT;
        sq.load((const T *)g.q + b * g.qs.b + (long long)r0 * g.qs.r + head * g.qs.h, len - r0, g.D, t);
        sg.load((const T *)g.dout + b * g.gs.b + (long long)r0 * g.gs.r + head * g.gs.h, len - r0, g.D, t);
        if (t < 2 * QT) l1 = r0 + t % QT < len ? (t < QT ? g.lse : g.delta)[((size_t)b * g.H + head) * g.N + r0 + t % QT] : 0.f;
        if (++rt > thi) { rt = tlo; ++hd; }
    };
    auto put = [&](int buf) {
        sq.template put<PREC>(Qimg + buf * IMG, t);
        sg.template put<PREC>(Gimg + buf * IMG, t);
        if (t < 2 * QT) (t < QT ? Ls : Ds)[buf][t % QT] = l1;
    };
    if (nt > 0) { load(); put(0); }
    wa_settle(kp);
    wa_settle(vp);
    __syncthreads();
    for (int tt = 0; tt < nt; ++tt) {
        const int cur = tt & 1, pn = rt * QT;
        if (tt + 1 < nt) load();
#pragma unroll
        for (int s = 0; s < QT; s += 32)
            if (k0 < len && p0 + s < len && p0 + s + 31 >= k0 - g.right && p0 + s <= k0 + 31 + g.left)
                wa_dkv_tile<T, PREC, DP, QT, false>(g, Qimg + cur * IMG + s * ROWB, Gimg + cur * IMG + s * ROWB, Ls[cur] + s, Ds[cur] + s, p0 + s, k0, len,
                                                    lane, kp, vp, AK, AV);
        if (tt + 1 < nt) put(cur ^ 1);
        p0 = pn;
        __syncthreads();
    }
    if (g.nsplit == 1 && kt < g.nst) {                        // the sinks' share from rows beyond their window
        const float *pt = g.part + ((size_t)bg * g.nst + kt) * g.nchunk * (2 * DP * 32) + j;
#pragma unroll
        for (int d = 0; d < ND; ++d) {
            float x[32];
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                x[r] = pt[(32 * d + at_drow(r, h)) * 32];
                x[16 + r] = pt[(DP + 32 * d + at_drow(r, h)) * 32];
            }
#pragma unroll
            for (int r = 0; r < 16; ++r) { AK[d][r] += x[r]; AV[d][r] += x[16 + r]; }
        }
    }
    if (k0 < g.N) {
        const size_t o = (((size_t)b * g.N + k0) * g.G + gi) * g.D, row = (size_t)g.G * g.D, all_ = (size_t)g.B * g.N * g.G * g.D;
        unsigned char *lds = at_smem + wv * WA_OUT<float, DP>;
        if (g.nsplit > 1) {
            float *pk = g.part2 + (size_t)chunk * 2 * all_ + o;
            wa_store_rows<float, DP>(lds, AK, 1.f, lane, pk, row, g.N - k0, g.D);
            wa_store_rows<float, DP>(lds, AV, 1.f, lane, pk + all_, row, g.N - k0, g.D);
        } else {
            wa_store_rows<T, DP>(lds, AK, g.scale, lane, dk + o, row, g.N - k0, g.D);
            wa_store_rows<T, DP>(lds, AV, 1.f, lane, dv + o, row, g.N - k0, g.D);
        }
    }
}
// dK, dV = the chunks' sums in order, then the sinks' share; a thread takes four channels
template <class T, int DP>
__global__ void __launch_bounds__(256) wa_bwd_join_kernel(const WaArgs g, T *__restrict__ dk, T *__restrict__ dv)
{
    const size_t all = (size_t)g.B * g.N * g.G * g.D, e = ((size_t)blockIdx.x * 256 + threadIdx.x) * 4;
    if (e >= all) return;
    const int ch = (int)(e % g.D);
    const size_t row = e / g.D;
    const int gi = (int)(row % g.G), ki = (int)(row / g.G % g.N), b = (int)(row / g.G / g.N);
#pragma unroll
    for (int w = 0; w < 2; ++w) {
        float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int c = 0; c < g.nsplit; ++c) {
            const float4 x = *reinterpret_cast<const float4 *>(g.part2 + ((size_t)2 * c + w) * all + e);
            a.x += x.x; a.y += x.y; a.z += x.z; a.w += x.w;
        }
        if (ki < 32 * g.nst) {
            const float *pt = g.part + ((size_t)(b * g.G + gi) * g.nst + ki / 32) * g.nchunk * (2 * DP * 32) + (w * DP + ch) * 32 + ki % 32;
            a.x += pt[0]; a.y += pt[32]; a.z += pt[64]; a.w += pt[96];
        }
        const float f = w ? 1.f : g.scale;
        wa_store4<T>((w ? dv : dk) + e, a.x * f, a.y * f, a.z * f, a.w * f);
    }
}

// what 32 sink keys receive from the rows of one chunk that lie beyond their window: part[bg][tile][chunk][dK | dV][channel][key]
template <class T, int DP> constexpr int WA_SINK_NW = DP == 128 && Mx<WaT<T>::PB>::NP == 3 ? 2 : 4;       // waves: what LDS holds
template <class T, int DP>
__global__ void __launch_bounds__(64 * (WA_SINK_NW<T, DP>), 1) wa_bwd_sink_kernel(const WaArgs g)
{
    constexpr int PREC = WaT<T>::PB, NP = Mx<PREC>::NP, IMG = NP * 32 * WaImg<DP>::ROWB, ND = DP / 32, NW = (WA_SINK_NW<T, DP>);
    extern __shared__ __attribute__((aligned(16))) unsigned char at_smem[];
    const int t = threadIdx.x, lane = t & 63, wv = __builtin_amdgcn_readfirstlane(t >> 6), j = lane & 31, h = lane >> 5;
    unsigned char *Qimg = at_smem + wv * (2 * IMG + 256), *Gimg = Qimg + IMG;                     // a wave's own images
    float *Ls = reinterpret_cast<float *>(Gimg + IMG), *Ds = Ls + 32;
    const int chunk = blockIdx.x % g.nchunk, st = blockIdx.x / g.nchunk % g.nst, bg = blockIdx.x / g.nchunk / g.nst, b = bg / g.G, gi = bg % g.G;
    const int len = wa_length(g.lengths, b, g.N), k0 = st * 32, ki = k0 + j;

    uint4 kp[DP / 16][NP], vp[DP / 16][NP];
    wa_colfrags<T, PREC, DP>((const T *)g.k + b * g.ks.b + (long long)ki * g.ks.r + gi * g.ks.h, ki < len, g.D, h, kp);
    wa_colfrags<T, PREC, DP>((const T *)g.v + b * g.vs.b + (long long)ki * g.vs.r + gi * g.vs.h, ki < len, g.D, h, vp);
    f32x16 AK[ND], AV[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) { AK[d][r] = 0.f; AV[d][r] = 0.f; }

    const int tlo = min(len, k0 + g.left + 1) / 32, per = (len + 31) / 32 - tlo;               // row tiles that hold i > k0 + left
    const int total = max(per, 0) * g.HG, each = (total + g.nchunk - 1) / g.nchunk, f0 = chunk * each, f1 = min(total, f0 + each);
    wa_settle(kp);
    wa_settle(vp);
    for (int f = f0; f < f1; f += NW) {                                                         // trip count is the workgroup's
        const int ff = f + wv;
        const bool on = ff < f1;
        const int head = gi * g.HG + (on ? ff / per : 0), p0 = on ? (tlo + ff % per) * 32 : 0;
        if (on) {
            WaStage<T, DP, 32, 64> sq, sg;
            sq.init(g.qs.r, lane);
            sg.init(g.gs.r, lane);
            sq.load((const T *)g.q + b * g.qs.b + (long long)p0 * g.qs.r + head * g.qs.h, len - p0, g.D, lane);
            sg.load((const T *)g.dout + b * g.gs.b + (long long)p0 * g.gs.r + head * g.gs.h, len - p0, g.D, lane);
            sq.template put<PREC>(Qimg, lane);
            sg.template put<PREC>(Gimg, lane);
            (lane < 32 ? Ls : Ds)[j] = p0 + j < len ? (lane < 32 ? g.lse : g.delta)[((size_t)b * g.H + head) * g.N + p0 + j] : 0.f;
        }
        __syncthreads();
        if (on) wa_dkv_tile<T, PREC, DP, 32, true>(g, Qimg, Gimg, Ls, Ds, p0, k0, len, lane, kp, vp, AK, AV);
        __syncthreads();
    }
    float *sum = reinterpret_cast<float *>(at_smem);                                            // [wave][dK | dV][channel][key]
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            float *a = sum + (wv * 2 * DP + 32 * d + at_drow(r, h)) * 32 + j;
            a[0] = AK[d][r];
            a[DP * 32] = AV[d][r];
        }
    __syncthreads();
    float *o = g.part + (size_t)blockIdx.x * (2 * DP * 32);
    for (int e = 4 * t; e < 2 * DP * 32; e += 256 * NW) {
        float4 x = *reinterpret_cast<const float4 *>(sum + e);
#pragma unroll
        for (int w = 1; w < NW; ++w) {
            const float4 y = *reinterpret_cast<const float4 *>(sum + w * 2 * DP * 32 + e);
            x.x += y.x; x.y += y.y; x.z += y.z; x.w += y.w;
        }
        *reinterpret_cast<float4 *>(o + e) = x;
    }
}

// the chunks of a sink tile added, in order, into the first: thread = 4 values, grid (values / 1024, tiles)
template <int DP> __global__ void __launch_bounds__(256) wa_sink_sum_kernel(float *__restrict__ part, int nchunk)
{
    constexpr int PER = 2 * DP * 32;
    float4 *p = reinterpret_cast<float4 *>(part + (size_t)blockIdx.y * nchunk * PER) + blockIdx.x * 256 + threadIdx.x;
    float4 a = p[0];
#pragma unroll 8
    for (int c = 1; c < nchunk; ++c) {
        const float4 x = p[(size_t)c * (PER / 4)];
        a.x += x.x; a.y += x.y; a.z += x.z; a.w += x.w;
    }
    p[0] = a;
}

// ------------------------------------------------------------------ the last T positions of cached sequences
// Columns of a wave's tile = up to 32 (head of the key head, row) pairs, so that a cached key is read once for all of them.  The
// visible key tiles of a sequence are dealt to the waves of its nchunk workgroups in turn; each wave keeps its own running
// softmax, the waves of a workgroup join through LDS, the workgroups (nchunk > 1) through part[..][m | l | O] and a second kernel.
// HBM-bound: a wave has a tile of K and V in flight (32 keys x 128 channels: 16 KB) beside the one it computes.  64 sequences x 4112 keys
// x 4 key heads x 128 bf16: 122 us, 4.4 TB/s; with lane masks around the loads of every tile 26 us more.  WIDE: eight waves instead of
// four, for few small caches that are not split (see wa_step_plan).
template <class T, int DP, bool WIDE> constexpr int WA_STEP_NW = WIDE ? 8 : 4;
template <class T, int DP, bool WIDE>
__global__ void __launch_bounds__(64 * (WA_STEP_NW<T, DP, WIDE>), sizeof(T) == 4 && DP == 128 ? 1 : 2) wa_step_kernel(const WaArgs g, T *__restrict__ out)
{
    constexpr int PREC = WaT<T>::PF, NP = Mx<PREC>::NP, IMG = NP * 32 * WaImg<DP>::ROWB, ND = DP / 32, NK = DP / 16, NW = (WA_STEP_NW<T, DP, WIDE>);
    extern __shared__ __attribute__((aligned(16))) unsigned char at_smem[];
    const int t = threadIdx.x, lane = t & 63, wv = __builtin_amdgcn_readfirstlane(t >> 6), j = lane & 31, h = lane >> 5;
    unsigned char *Vimg = at_smem + wv * IMG;
    const unsigned bid = wa_order(blockIdx.x, gridDim.x);        // the heads of a sequence lie side by side: on one XCD
    const int sp = bid % g.nchunk, cb = bid / g.nchunk % g.nblk, bg = bid / g.nchunk / g.nblk, b = bg / g.G, gi = bg % g.G;
    const int len = wa_length(g.lengths, b, g.S), col = cb * 32 + j, hs = col / g.N, head = gi * g.HG + hs, tq = col % g.N, qi = len - g.N + tq;
    const bool mine = hs < g.HG && qi >= 0;
    const T *kb_ = (const T *)g.k + b * g.ks.b + gi * g.ks.h, *vb = (const T *)g.v + b * g.vs.b + gi * g.vs.h;

    uint4 qp[NK][NP];
    wa_colfrags<T, PREC, DP>((const T *)g.q + b * g.qs.b + tq * g.qs.r + head * g.qs.h, mine, g.D, h, qp);
    float m = -__builtin_inff(), mc = 0.f, l = 0.f;
    f32x16 O[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) O[d][r] = 0.f;

    const int first = max(0, len - g.N - g.left), tlo = first / 32, thi = (len - 1) / 32;
    const int nsink = min((min(g.sinks, len) + 31) / 32, tlo), nt = len > 0 ? nsink + thi - tlo + 1 : 0;
    const float thr = WA_LAZY / g.c;
    WaRaw<T> rk[NK], rv[NK];                             // lane (row j, half h): channels 16 kb + 8 h ..
    auto row0 = [&](int tt) { return (tt < nsink ? tt : tlo + tt - nsink) * 32; };
    auto load = [&](int tt) {
        const int r0 = row0(tt);
        const T *kr = kb_ + (long long)(r0 + j) * g.ks.r, *vr = vb + (long long)(r0 + j) * g.vs.r;
        if (r0 >= first && r0 + 32 <= len && g.D == DP) {                  // (not masked: see above)
#pragma unroll
            for (int kb = 0; kb < NK; ++kb) {
                rk[kb] = wa_load8<T>(kr + 16 * kb + 8 * h);
                rv[kb] = wa_load8<T>(vr + 16 * kb + 8 * h);
            }
        } else {
            asm volatile("");
            const bool seen = r0 + j < len && (r0 + j >= first || r0 + j < g.sinks);        // what no row sees may be overwritten
#pragma unroll
            for (int kb = 0; kb < NK; ++kb) {
                const int ch = 16 * kb + 8 * h;
                rk[kb] = wa_zero<T>();
                rv[kb] = wa_zero<T>();
                if (seen && ch < g.D) {
                    rk[kb] = wa_load8<T>(kr + ch);
                    rv[kb] = wa_load8<T>(vr + ch);
                }
            }
        }
    };
    const int step = NW * g.nchunk;
    int tt = sp * NW + wv;
    if (tt < nt) load(tt);
    for (; tt < nt; tt += step) {
        const int j0 = row0(tt);
        f32x16 acc;
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[r] = 0.f;
#pragma unroll
        for (int kb = 0; kb < NK; ++kb) {
            uint4 ak[NP], pv[NP];
            wa_pieces<T, PREC>(rk[kb], ak);
            mm_mac<PREC>(ak, qp[kb], acc);
            wa_pieces<T, PREC>(rv[kb], pv);
#pragma unroll
            for (int p = 0; p < NP; ++p) *reinterpret_cast<uint4 *>(Vimg + p * WaImg<DP>::template plane<32>() + j * WaImg<DP>::ROWB + 32 * kb + 16 * h) = pv[p];
        }
        if (tt + step < nt) load(tt + step);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");       // the image is the wave's own: LDS serves a wave in order
        __builtin_amdgcn_wave_barrier();
        float tmax = -__builtin_inff();
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const int jj = j0 + at_drow(r, h);
            const bool ok = jj < len && jj <= qi && (jj >= qi - g.left || jj < g.sinks);
            acc[r] = ok ? acc[r] : -__builtin_inff();
            tmax = fmaxf(tmax, acc[r]);
        }
        tmax = wa_max32(tmax);
        if (__ballot(tmax > m + thr) != 0ull) {
            const float m_new = fmaxf(m, tmax), mc_new = m_new == -__builtin_inff() ? 0.f : m_new * g.c;
            const float sc = m == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(mc - mc_new);
            m = m_new;
            mc = mc_new;
            l *= sc;
#pragma unroll
            for (int d = 0; d < ND; ++d)
#pragma unroll
                for (int r = 0; r < 16; ++r) O[d][r] *= sc;
        }
        float pd[16];
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            pd[r] = __builtin_amdgcn_exp2f(fmaf(acc[r], g.c, -mc));
            l += pd[r];
        }
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
            uint4 pp[NP], av[NP];
            at_regfrag<PREC>(pd, ks, pp);
#pragma unroll
            for (int d = 0; d < ND; ++d) {
                wa_trfrag<PREC, DP, 32>(Vimg, lane, d, ks, av);
                mm_mac<PREC>(av, pp, O[d]);
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
    // join the waves: ml[wave][m, l][32], o[wave][channel][32]; every thread sums its values over the waves in order
    l = wa_sum32(l);
    const float mb = m == -__builtin_inff() ? -__builtin_inff() : mc;      // maximum in base-2 units
    __syncthreads();
    float *ml = reinterpret_cast<float *>(at_smem), *osum = ml + NW * 64;
    if (h == 0) { ml[wv * 64 + j] = mb; ml[wv * 64 + 32 + j] = l; }
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) osum[(wv * DP + 32 * d + at_drow(r, h)) * 32 + j] = O[d][r];
    __syncthreads();
    float M = -__builtin_inff(), Lt = 0.f, f[NW];                          // (thread t's column is j as well: t & 31)
#pragma unroll
    for (int w = 0; w < NW; ++w) M = fmaxf(M, ml[w * 64 + j]);
#pragma unroll
    for (int w = 0; w < NW; ++w) {
        const float mw = ml[w * 64 + j];
        f[w] = mw == -__builtin_inff() ? 1.f : __builtin_amdgcn_exp2f(mw - M);      // a wave without keys holds zeros
        Lt = fmaf(ml[w * 64 + 32 + j], f[w], Lt);
    }
    const float inv = Lt > 0.f ? 1.f / Lt : (Lt != Lt ? Lt : 0.f);
    float *po = g.part + (size_t)bid * (64 + DP * 32);
    if (g.nchunk > 1 && t < 32) { po[j] = M; po[32 + j] = Lt; }
    for (int ch = 4 * (t >> 5); ch < DP; ch += 8 * NW) {
        float o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < NW; ++w)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = fmaf(osum[(w * DP + ch + e) * 32 + j], f[w], o[e]);
        if (g.nchunk > 1) {
#pragma unroll
            for (int e = 0; e < 4; ++e) po[64 + (ch + e) * 32 + j] = o[e];
        } else if (hs < g.HG && ch < g.D)
            wa_store4<T>(out + (((size_t)b * g.N + tq) * g.H + head) * g.D + ch, o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv);
    }
}

// joins the nchunk partial softmaxes of one (sequence, key head, 32 columns): thread = (column, 4 channels), all of it at once
template <class T, int DP>
__global__ void __launch_bounds__(8 * DP) wa_join_kernel(const WaArgs g, T *__restrict__ out)
{
    constexpr int PER = 64 + DP * 32;
    const int t = threadIdx.x, j = t & 31, ch = 4 * (t >> 5);
    const int cb = blockIdx.x % g.nblk, bg = blockIdx.x / g.nblk, b = bg / g.G, gi = bg % g.G;
    const int col = cb * 32 + j, hs = col / g.N, head = gi * g.HG + hs, tq = col % g.N;
    if (hs >= g.HG || ch >= g.D) return;
    const float *pt = g.part + (size_t)blockIdx.x * g.nchunk * PER;
    float M = -__builtin_inff(), Lt = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int s = 0; s < g.nchunk; ++s) M = fmaxf(M, pt[(size_t)s * PER + j]);
#pragma unroll 4
    for (int s = 0; s < g.nchunk; ++s) {
        const float *p = pt + (size_t)s * PER, ms = p[j];
        const float f = ms == -__builtin_inff() ? 1.f : __builtin_amdgcn_exp2f(ms - M);
        Lt = fmaf(p[32 + j], f, Lt);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = fmaf(p[64 + (ch + e) * 32 + j], f, o[e]);
    }
    const float inv = Lt > 0.f ? 1.f / Lt : (Lt != Lt ? Lt : 0.f);
    wa_store4<T>(out + (((size_t)b * g.N + tq) * g.H + head) * g.D + ch, o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv);
}

// ------------------------------------------------------------------ host side
int wa_check(const char *who, const gfs3d_window_attn_args *a)
{
    GFS3D_REQUIRE(a, "%s: NULL args", who);
    GFS3D_REQUIRE(a->type == GFS3D_COMPUTE_F32 || a->type == GFS3D_COMPUTE_BF16 || a->type == GFS3D_COMPUTE_F16,
                  "%s: type must be one of GFS3D_COMPUTE_*", who);
    GFS3D_REQUIRE(a->B >= 1 && a->N >= 1 && a->S >= 1 && a->S <= (1 << 29) && a->N <= (1 << 29), "%s: bad shape B=%d N=%d S=%d", who, a->B, a->N, a->S);
    GFS3D_REQUIRE(a->G >= 1 && a->H >= a->G && a->H % a->G == 0, "%s: %d heads over %d key heads", who, a->H, a->G);
    GFS3D_REQUIRE(a->D >= 8 && a->D <= 128 && a->D % 8 == 0, "%s: head size %d unsupported (a multiple of 8 up to 128)", who, a->D);
    GFS3D_REQUIRE(a->left >= 0 && a->right >= 0 && a->sinks >= 0, "%s: left=%d right=%d sinks=%d", who, a->left, a->right, a->sinks);
    GFS3D_REQUIRE(a->scale > 0.f && a->scale < 3e38f, "%s: scale %g must be positive and finite", who, (double)a->scale);
    GFS3D_REQUIRE(a->q && a->k && a->v && a->out, "%s: NULL buffer", who);
    const int gran = 16 / (a->type == GFS3D_COMPUTE_F32 ? 4 : 2);
    const void *written[6] = {a->out, a->out_low, a->dq, a->dk, a->dv, a->workspace};
    for (const void *w : written) GFS3D_REQUIRE(((uintptr_t)w & 15) == 0, "%s: an output or the workspace is not aligned to 16 bytes", who);
    const long long *st[4] = {a->q_stride, a->k_stride, a->v_stride, a->dout_stride};
    const void *pt[4] = {a->q, a->k, a->v, a->dout};
    for (int n = 0; n < 4; ++n) {
        if (!pt[n]) continue;
        GFS3D_REQUIRE(((uintptr_t)pt[n] & 15) == 0, "%s: a tensor is not aligned to 16 bytes", who);
        GFS3D_REQUIRE(st[n][1] <= (1 << 23), "%s: rows more than 2^23 elements apart", who);        // 32-bit offsets within a tile
        for (int e = 0; e < 3; ++e) GFS3D_REQUIRE(st[n][e] >= 0 && st[n][e] % gran == 0, "%s: a stride is negative or not a multiple of 16 bytes", who);
    }
    return GFS3D_OK;
}
int wa_dp(int D) { return D <= 32 ? 32 : D <= 64 ? 64 : 128; }
WaArgs wa_args(const gfs3d_window_attn_args *a)
{
    WaArgs g{};
    g.q = a->q; g.k = a->k; g.v = a->v; g.out = a->out; g.dout = a->dout; g.low = a->type == GFS3D_COMPUTE_F32 ? nullptr : a->out_low;
    g.qs = {a->q_stride[0], a->q_stride[1], a->q_stride[2]};
    g.ks = {a->k_stride[0], a->k_stride[1], a->k_stride[2]};
    g.vs = {a->v_stride[0], a->v_stride[1], a->v_stride[2]};
    g.gs = {a->dout_stride[0], a->dout_stride[1], a->dout_stride[2]};
    g.lengths = a->lengths; g.lse = a->lse;
    g.B = a->B; g.N = a->N; g.S = a->S; g.H = a->H; g.G = a->G; g.HG = a->H / a->G; g.D = a->D;
    g.left = a->left < a->S ? a->left : a->S; g.right = a->right < a->S ? a->right : a->S; g.sinks = a->sinks < a->S ? a->sinks : a->S;
    g.scale = a->scale; g.c = a->scale * 1.4426950408889634f;
    return g;
}
// the sinks' gradient kernel runs where some row lies beyond the first key's window; at most 32 chunks of at least 8 row tiles, and
// only until every CU has four workgroups: each chunk leaves fp32 sums of its 32 keys, which otherwise outgrow the tensors
void wa_sink_plan(WaArgs &g)
{
    g.nst = g.sinks > 0 && g.N > g.left + 1 ? (g.sinks + 31) / 32 : 0;
    const long long tiles = (long long)((g.N + 31) / 32) * g.HG, keys = (long long)g.B * g.G * g.nst;
    long long n = tiles / 8 > 32 ? 32 : tiles / 8;
    if (keys > 0 && n > (1023 + keys) / keys) n = (1023 + keys) / keys;
    g.nchunk = (int)(n < 1 ? 1 : n);
}
// dK, dV: workgroups of 128 keys, their turns split until every CU has two workgroups (at most 8 ways, 4 turns at least; 196 workgroups of 7 x
// 1777 rows x 6 / 2 heads x 40, three ways: 116 us + 6 for the join, unsplit 157)
void wa_dkv_plan(WaArgs &g, bool most = false)       // most: the bound over all types and reaches
{
    const long long blocks = (long long)g.B * g.G * ((g.N + 127) / 128);
    const long long reach = g.N < 127ll + g.left + g.right ? g.N : 127ll + g.left + g.right, turns = (reach + 63) / 64 * g.HG;
    long long n = (512 + blocks - 1) / blocks;
    if (!most && n > turns / 4) n = turns / 4;
    g.nsplit = (int)(n < 1 ? 1 : n > 8 ? 8 : n);
}
size_t wa_split_floats(const WaArgs &g) { return g.nsplit > 1 ? (size_t)g.nsplit * 2 * g.B * g.N * g.G * g.D : 0; }
size_t wa_sink_floats(const WaArgs &g) { return (size_t)g.B * g.G * g.nst * g.nchunk * 2 * wa_dp(g.D) * 32; }
// Long caches (more than 64 tiles): four waves to a workgroup, the keys split until every CU has four, four tiles to a wave at least.  Lengths
// differ in earnest, and the longest sequence must not be one workgroup's (kernels, 64 sequences x 4 key heads x 128 bf16: lengths spread over
// 400 .. 8192 153 us, unsplit 204; one of 8192 beside 409 48 for 128; all of 8192 223 for 244.  256 x 2 x 64, all of 8192: 237 for 209).
// Short caches: split until every CU has one workgroup, two tiles to a wave at least (16 x 2 key heads x 1028 x 128 bf16: 15.0 us, with twice the
// tiles per wave 18.5; 256 x 2 x 1028 x 64: unsplit 29.7, in two 38.9).  A split costs a second launch, 4 us of the caller's time: caches of
// up to 320 KB take one workgroup of eight waves instead (whole calls, 4 x 2 key heads, 1028 keys x 64 bf16: 13.3 us for 17.7; the sides meet
// near 400 KB: 1028 x 128 bf16 20.7 for 17.6, 1028 x 64 fp32 22.0 for 17.7, 1540 x 32 fp32 17.7 for 18.0).  With a workgroup for every CU
// nothing is split, and eight waves serve a long sequence beside short ones better (256 x 2 key heads of up to 1900 x 64 bf16, every eighth full:
// 24 us for 33; all full: 56 for 53) unless they have fewer than two tiles each and a CU has two workgroups (260 keys, 512 workgroups x 64 bf16:
// 14.7 for 10.0; 256 x 64 fp32: 12.4 for 14.2).  Eight waves of fp32 at 128 channels do not fit a CU's LDS.
constexpr long long WA_WIDE_BYTES = 320 * 1024;
void wa_step_plan(WaArgs &g, bool fp32, bool &wide)
{
    g.nblk = (int)(((long long)g.HG * g.N + 31) / 32);
    const long long keys = (long long)g.left + g.N < g.S ? (long long)g.left + g.N : g.S;
    const long long tiles = keys / 32 + 2 + (g.sinks + 31) / 32, blocks = (long long)g.B * g.G * g.nblk, dp = wa_dp(g.D);
    const bool longs = tiles > 64;
    wide = !longs && !(fp32 && dp == 128) && (blocks < 256 ? tiles * 32 * dp * 2 * (fp32 ? 4 : 2) <= WA_WIDE_BYTES : tiles > 16 || blocks < 512);
    long long n = wide ? 1 : ((longs ? 1023 : 255) + blocks) / blocks;
    if (n > tiles / (longs ? 16 : 8)) n = tiles / (longs ? 16 : 8);
    g.nchunk = (int)(n < 1 ? 1 : n > 64 ? 64 : n);
}
// Waves of a workgroup in the forward: eight share every staged key tile where that leaves four workgroups to a CU (rooms of 2 x 65536 x
// 8 heads x 64: 409 us, with four waves 418; 128 channels, causal: 568, with four 600; dQ in eight waves spills at four waves per SIMD and
// was 17 % slower), four otherwise
template <class T, int DP> bool wa_wide(const WaArgs &g)
{
    return sizeof(T) == 2 && (long long)g.B * g.G * (((g.N + 31) / 32 * (long long)g.HG + 7) / 8) >= 1024;
}
// a launch holds fewer than 2^32 threads
#define WA_REQUIRE_GRID(blocks, threads, who) GFS3D_REQUIRE((size_t)(blocks) * (threads) < (1ull << 32), "%s: %zu workgroups", who, (size_t)(blocks))
// workgroups of NW waves per (sequence, key head): a wave takes 32 rows of one head
size_t wa_query_blocks(const WaArgs &g, int NW) { return ((size_t)((g.N + 31) / 32) * g.HG + NW - 1) / NW; }
template <class T, int DP, int NW> int wa_forward_queries(WaArgs g, void *out, hipStream_t st, const char *who)
{
    constexpr size_t im = 4ull * Mx<WaT<T>::PF>::NP * (WA_KT<T, DP, NW>) * WaImg<DP>::ROWB, ou = (size_t)NW * WA_OUT<T, DP>, lds = im > ou ? im : ou;
    const size_t blocks = (size_t)g.B * g.G * wa_query_blocks(g, NW);
    WA_REQUIRE_GRID(blocks, 64 * NW, who);
    g.nblk = (int)wa_query_blocks(g, NW);
    GFS3D_ENSURE_LDS((wa_fwd_kernel<T, DP, NW>), lds, who);
    hipLaunchKernelGGL((wa_fwd_kernel<T, DP, NW>), dim3((unsigned)blocks), dim3(64 * NW), lds, st, g, (T *)out);
    GFS3D_LAUNCH_CHECK("wa_fwd_kernel");
    return GFS3D_OK;
}
template <class T, int DP> int wa_forward(const WaArgs &g, void *out, hipStream_t st, const char *who)
{
    if constexpr (sizeof(T) == 2) {
        if (wa_wide<T, DP>(g)) return wa_forward_queries<T, DP, 8>(g, out, st, who);
    }
    return wa_forward_queries<T, DP, 4>(g, out, st, who);
}
template <class T, int DP> int wa_backward_queries(WaArgs g, void *dq, hipStream_t st, const char *who)
{
    constexpr int NW = 4;
    constexpr size_t im = 4ull * Mx<WaT<T>::PB>::NP * 32 * WaImg<DP>::ROWB, ou = (size_t)NW * WA_OUT<T, DP>, lds = im > ou ? im : ou;
    g.nblk = (int)wa_query_blocks(g, NW);
    const size_t blocks = (size_t)g.B * g.G * g.nblk;
    GFS3D_ENSURE_LDS((wa_bwd_dq_kernel<T, DP>), lds, who);
    hipLaunchKernelGGL((wa_bwd_dq_kernel<T, DP>), dim3((unsigned)blocks), dim3(64 * NW), lds, st, g, (T *)dq);
    GFS3D_LAUNCH_CHECK("wa_bwd_dq_kernel");
    return GFS3D_OK;
}
template <class T, int DP> int wa_backward_keys(WaArgs g, void *dk, void *dv, hipStream_t st, const char *who)
{
    constexpr int QT = WA_QT<T, DP>;
    constexpr size_t im = 4 * ((size_t)Mx<WaT<T>::PB>::NP * QT * WaImg<DP>::ROWB + QT * sizeof(float)), ou = 4ull * WA_OUT<float, DP>, lds = im > ou ? im : ou;
    g.nblk = (g.N + 127) / 128;
    const size_t blocks = (size_t)g.nblk * g.B * g.G * g.nsplit;
    GFS3D_ENSURE_LDS((wa_bwd_dkv_kernel<T, DP>), lds, who);
    hipLaunchKernelGGL((wa_bwd_dkv_kernel<T, DP>), dim3((unsigned)blocks), dim3(256), lds, st, g, (T *)dk, (T *)dv);
    GFS3D_LAUNCH_CHECK("wa_bwd_dkv_kernel");
    if (g.nsplit > 1) {
        const size_t threads = (size_t)g.B * g.N * g.G * g.D / 4;
        hipLaunchKernelGGL((wa_bwd_join_kernel<T, DP>), dim3((unsigned)((threads + 255) / 256)), dim3(256), 0, st, g, (T *)dk, (T *)dv);
        GFS3D_LAUNCH_CHECK("wa_bwd_join_kernel");
    }
    return GFS3D_OK;
}
template <class T, int DP> int wa_backward(WaArgs g, void *dq, void *dk, void *dv, hipStream_t st, const char *who)
{
    constexpr size_t img = (size_t)Mx<WaT<T>::PB>::NP * 32 * WaImg<DP>::ROWB;
    const size_t pairs = (size_t)g.B * g.G, sinks = pairs * g.nst * g.nchunk;
    WA_REQUIRE_GRID(pairs * wa_query_blocks(g, 4), 256, who);                // all refusals before the first launch
    WA_REQUIRE_GRID(sinks, 64 * (WA_SINK_NW<T, DP>), who);
    WA_REQUIRE_GRID(pairs * ((g.N + 127) / 128) * g.nsplit, 256, who);
    if (int rc = wa_backward_queries<T, DP>(g, dq, st, who)) return rc;
    if (g.nst > 0) {
        constexpr int NW = (WA_SINK_NW<T, DP>);
        constexpr size_t ws = (size_t)NW * (2 * img + 256), sum = 2ull * NW * DP * 32 * sizeof(float), lsk = ws > sum ? ws : sum;
        GFS3D_ENSURE_LDS((wa_bwd_sink_kernel<T, DP>), lsk, who);
        hipLaunchKernelGGL((wa_bwd_sink_kernel<T, DP>), dim3((unsigned)sinks), dim3(64 * NW), lsk, st, g);
        GFS3D_LAUNCH_CHECK("wa_bwd_sink_kernel");
        if (g.nchunk > 1) {                                  // (then there are fewer than 1024 tiles)
            hipLaunchKernelGGL((wa_sink_sum_kernel<DP>), dim3(2 * DP * 32 / 1024, (unsigned)(g.B * g.G * g.nst)), dim3(256), 0, st, g.part, g.nchunk);
            GFS3D_LAUNCH_CHECK("wa_sink_sum_kernel");
        }
    }
    return wa_backward_keys<T, DP>(g, dk, dv, st, who);
}
template <class T, int DP, bool WIDE> int wa_step_go(const WaArgs &g, void *out, hipStream_t st, const char *who)
{
    constexpr int NW = (WA_STEP_NW<T, DP, WIDE>);
    constexpr size_t im = (size_t)NW * Mx<WaT<T>::PF>::NP * 32 * WaImg<DP>::ROWB, js = (size_t)NW * (64 + DP * 32) * sizeof(float), lds = im > js ? im : js;
    static_assert(lds <= 160 * 1024, "LDS");
    const size_t groups = (size_t)g.B * g.G * g.nblk, blocks = groups * g.nchunk;
    WA_REQUIRE_GRID(blocks, 64 * NW, who);
    if (g.nchunk > 1) WA_REQUIRE_GRID(groups, 8 * DP, who);
    GFS3D_ENSURE_LDS((wa_step_kernel<T, DP, WIDE>), lds, who);
    hipLaunchKernelGGL((wa_step_kernel<T, DP, WIDE>), dim3((unsigned)blocks), dim3(64 * NW), lds, st, g, (T *)out);
    GFS3D_LAUNCH_CHECK("wa_step_kernel");
    if (g.nchunk > 1) {
        hipLaunchKernelGGL((wa_join_kernel<T, DP>), dim3((unsigned)groups), dim3(8 * DP), 0, st, g, (T *)out);
        GFS3D_LAUNCH_CHECK("wa_join_kernel");
    }
    return GFS3D_OK;
}
template <class T, int DP> int wa_step(const WaArgs &g, bool wide, void *out, hipStream_t st, const char *who)
{
    if constexpr (!(sizeof(T) == 4 && DP == 128)) {
        if (wide) return wa_step_go<T, DP, true>(g, out, st, who);
    }
    return wa_step_go<T, DP, false>(g, out, st, who);
}

// one call per (type, padded head size)
#define WA_DISPATCH(call)                                                                                                            \
    switch (wa_dp(a->D) * 4 + a->type) {                                                                                             \
    case 32 * 4 + GFS3D_COMPUTE_F32: { using T = float; constexpr int DP = 32; return call; }                                        \
    case 64 * 4 + GFS3D_COMPUTE_F32: { using T = float; constexpr int DP = 64; return call; }                                        \
    case 128 * 4 + GFS3D_COMPUTE_F32: { using T = float; constexpr int DP = 128; return call; }                                      \
    case 32 * 4 + GFS3D_COMPUTE_BF16: { using T = __bf16; constexpr int DP = 32; return call; }                                      \
    case 64 * 4 + GFS3D_COMPUTE_BF16: { using T = __bf16; constexpr int DP = 64; return call; }                                      \
    case 128 * 4 + GFS3D_COMPUTE_BF16: { using T = __bf16; constexpr int DP = 128; return call; }                                    \
    case 32 * 4 + GFS3D_COMPUTE_F16: { using T = _Float16; constexpr int DP = 32; return call; }                                     \
    case 64 * 4 + GFS3D_COMPUTE_F16: { using T = _Float16; constexpr int DP = 64; return call; }                                     \
    default: { using T = _Float16; constexpr int DP = 128; return call; }                                                            \
    }

}  // namespace
}  // namespace gfs3d

extern "C" size_t gfs3d_window_attn_workspace_bytes(int B, int N, int S, int H, int G, int D, int left, int sinks, int step)
{
    if (B < 1 || N < 1 || S < 1 || G < 1 || H < G || H % G || D < 8 || D > 128 || left < 0 || sinks < 0) return 0;
    WaArgs g{};
    g.B = B; g.N = N; g.S = S; g.H = H; g.G = G; g.HG = H / G; g.D = D;
    g.left = left < S ? left : S; g.sinks = sinks < S ? sinks : S;
    if (step) {
        bool wide;
        wa_step_plan(g, step == 1 + GFS3D_COMPUTE_F32, wide);
        return g.nchunk > 1 ? (size_t)B * G * g.nblk * g.nchunk * (64 + wa_dp(D) * 32) * sizeof(float) : 0;
    }
    wa_sink_plan(g);
    wa_dkv_plan(g, true);
    return (align_up((size_t)B * H * N, 64) + wa_sink_floats(g) + wa_split_floats(g)) * sizeof(float);
}

extern "C" int gfs3d_window_attn_forward(const gfs3d_window_attn_args *a, void *stream)
{
    const char *who = "gfs3d_window_attn_forward";
    if (int rc = wa_check(who, a)) return rc;
    GFS3D_REQUIRE(a->S == a->N, "%s: S=%d differs from N=%d", who, a->S, a->N);
    const WaArgs g = wa_args(a);
    hipStream_t st = static_cast<hipStream_t>(stream);
    WA_DISPATCH((wa_forward<T, DP>(g, a->out, st, who)))
}

extern "C" int gfs3d_window_attn_backward(const gfs3d_window_attn_args *a, void *stream)
{
    const char *who = "gfs3d_window_attn_backward";
    if (int rc = wa_check(who, a)) return rc;
    GFS3D_REQUIRE(a->S == a->N, "%s: S=%d differs from N=%d", who, a->S, a->N);
    GFS3D_REQUIRE(a->lse && a->dout && a->dq && a->dk && a->dv && a->workspace, "%s: NULL buffer", who);
    WaArgs g = wa_args(a);
    wa_sink_plan(g);
    wa_dkv_plan(g);
    const size_t need = gfs3d_window_attn_workspace_bytes(a->B, a->N, a->S, a->H, a->G, a->D, a->left, a->sinks, 0);
    if (a->workspace_bytes < need) {
        set_error("%s: workspace too small (%zu, needs %zu)", who, a->workspace_bytes, need);
        return GFS3D_ERR_WORKSPACE;
    }
    g.delta = (float *)a->workspace;
    g.part = g.delta + align_up((size_t)a->B * a->H * a->N, 64);
    g.part2 = g.part + wa_sink_floats(g);
    hipStream_t st = static_cast<hipStream_t>(stream);
    WA_DISPATCH((wa_backward<T, DP>(g, a->dq, a->dk, a->dv, st, who)))
}

extern "C" int gfs3d_window_attn_step(const gfs3d_window_attn_args *a, void *stream)
{
    const char *who = "gfs3d_window_attn_step";
    if (int rc = wa_check(who, a)) return rc;
    GFS3D_REQUIRE(a->lengths, "%s: NULL lengths", who);
    WaArgs g = wa_args(a);
    bool wide;
    wa_step_plan(g, a->type == GFS3D_COMPUTE_F32, wide);
    const size_t need = gfs3d_window_attn_workspace_bytes(a->B, a->N, a->S, a->H, a->G, a->D, a->left, a->sinks, 1 + a->type);
    if (need > 0 && (!a->workspace || a->workspace_bytes < need)) {
        set_error("%s: workspace too small (%zu, needs %zu)", who, a->workspace_bytes, need);
        return GFS3D_ERR_WORKSPACE;
    }
    g.part = (float *)a->workspace;
    hipStream_t st = static_cast<hipStream_t>(stream);
    WA_DISPATCH((wa_step<T, DP>(g, wide, a->out, st, who)))
}
