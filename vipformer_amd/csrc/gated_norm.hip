// gated_norm.hip -- h = alpha x + beta gate * post(y), n = pre(h), and its gradient (gfx950).
//
// A row is held in the registers of TPR threads (8 values each), so each tensor crosses HBM once: forward reads x, y and writes h, n;
// backward reads dh, dn, x, y and writes dx, dy.  Backward rebuilds h from x and y with the statistics that forward kept (four floats a
// row): the bytes are the same as reading h, and h's rounding to x's type does not enter the gradient of the second norm.
// Above D = 4096 a row takes 1024 threads and a thread has 128 registers; backward needs about 230 and spills 300 - 488 bytes a thread
// (bf16, 8192 rows, us: D = 4096 95, 4104 678, 8192 754).
// Variances are sums of squared differences from the mean (two passes over registers), all sums fp32.
// Parameters and a broadcast gate stay in registers while a workgroup walks consecutive rows.
//   backward, per row:   e = dn w_pre            dH = dh + rstd_h (e - mean(e) - hh mean(e hh))        (RMS: without the plain means)
//                        dx = alpha dH           dgate += beta dH u
//                        f = beta gate dH w_post  dy = rstd_y (f - mean(f) - yh mean(f yh))
//   column sums over rows: registers -> one partial row per workgroup -> gn_fold_kernel in a fixed order (no atomics).
#include "vpf_elem.h"

#define GN_E 8                  // values of a row in one thread
#define GN_FOLD_SLICES 16

template <int TPR> struct GnGeom { static constexpr int NT = TPR <= 256 ? 256 : TPR, G = NT / TPR, W = (TPR + 63) / 64; };

// `single`: a gate row serves so few rows that its gradient goes row by row to scratch and is summed from there
struct GnArgs { VpfGatedNorm a; int rows_per_wg, nwg, want, single; };
enum { GN_WANT_WPOST = 1, GN_WANT_BPOST = 2, GN_WANT_WPRE = 4, GN_WANT_BPRE = 8, GN_WANT_GATE = 16 };

// this thread's columns of a row: 8 t .. 8 t + 7 (V = 8: D a multiple of 8, 16-byte aligned) or t, t + TPR, .. (V = 1)
template <int TPR, int V> __device__ __forceinline__ int gn_col(int t, int e) { return V == 8 ? 8 * t + e : t + e * TPR; }
template <typename T, int TPR, int V> __device__ __forceinline__ void gn_store(T* p, const float* v, int t, int D)
{
    if constexpr (V == 8) { if (8 * t < D) vpf_store<T, 8>(p + 8 * t, v); }
    else {
#pragma unroll
        for (int e = 0; e < GN_E; ++e) { const int c = gn_col<TPR, V>(t, e); if (c < D) p[c] = (T)v[e]; }
    }
}
// a thread's part of a row as it lies in memory: the next row's tensors wait in these registers while this row is worked on.  Columns behind D
// are fetched from column 0; they read as 0 (V = 1) or the thread's share of every row sum is dropped (V = 8: whole threads are behind D).
template <typename T, int TPR, int V> struct GnRaw {
    VpfRaw<T, V> r[GN_E / V];
    __device__ __forceinline__ void fetch(const T* p, int t, int D)
    {
#pragma unroll
        for (int e = 0; e < GN_E; e += V) { const int c = gn_col<TPR, V>(t, e); r[e / V].load(p + (c < D ? c : 0)); }
    }
    __device__ __forceinline__ void get(float* v, int t, int D) const
    {
#pragma unroll
        for (int e = 0; e < GN_E; ++e) { const float x = r[e / V].get(e % V); v[e] = V == 8 || gn_col<TPR, V>(t, e) < D ? x : 0.f; }
    }
};
template <int TPR, int V> __device__ __forceinline__ void gn_param(float* v, const float* p, int t, int D, float none)
{
    if (p) { GnRaw<float, TPR, V> r; r.fetch(p, t, D); r.get(v, t, D); }
    else {
#pragma unroll
        for (int e = 0; e < GN_E; ++e) v[e] = none;
    }
}
// sums of a and b over the TPR threads of a row, in every one of them.  More than one wave: through LDS; `buf` alternates, so one barrier
// a call is enough (a wave writes buffer i again two barriers later).
template <int TPR> __device__ __forceinline__ void gn_sum2(float& a, float& b, float2 (*red)[16], int& buf)
{
    auto step = [](float v) {
        v += dpp_f<VPF_DPP_QUAD_1032, 0xF>(0.f, v);
        v += dpp_f<VPF_DPP_QUAD_2301, 0xF>(0.f, v);
        v += dpp_f<VPF_DPP_ROW_HALF_MIRROR, 0xF>(0.f, v);
        v += dpp_f<VPF_DPP_ROW_MIRROR, 0xF>(0.f, v);
        if constexpr (TPR >= 32) { const auto w = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false); v = __uint_as_float(w[0]) + __uint_as_float(w[1]); }
        if constexpr (TPR >= 64) { const auto w = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false); v = __uint_as_float(w[0]) + __uint_as_float(w[1]); }
        return v;
    };
    a = step(a); b = step(b);
    if constexpr (TPR > 64) {
        constexpr int W = GnGeom<TPR>::W;
        const int wave = threadIdx.x >> 6;
        if ((threadIdx.x & 63) == 0) red[buf][wave] = make_float2(a, b);
        __syncthreads();
        const int w0 = wave / W * W;
        a = b = 0.f;
#pragma unroll
        for (int i = 0; i < W; ++i) { const float2 p = red[buf][w0 + i]; a += p.x; b += p.y; }
        buf ^= 1;
    }
}

// mean and 1 / sqrt(variance + eps) of a row (RMS: 0 and 1 / sqrt(mean square + eps))
template <int TPR, int V>
__device__ __forceinline__ void gn_stats(const float* v, int t, int D, int rms, float eps, float& mean, float& rstd, float2 (*red)[16], int& buf)
{
    const float inv = 1.f / (float)D, live = V == 8 && 8 * t >= D ? 0.f : 1.f;
    float s = 0.f, q = 0.f;
    mean = 0.f;
    if (!rms) {
#pragma unroll
        for (int e = 0; e < GN_E; ++e) s += v[e];
        s *= live;
        gn_sum2<TPR>(s, q, red, buf);
        mean = s * inv;
    }
    q = 0.f; s = 0.f;
#pragma unroll
    for (int e = 0; e < GN_E; ++e) { const float d = V == 8 || gn_col<TPR, V>(t, e) < D ? v[e] - mean : 0.f; q = fmaf(d, d, q); }
    q *= live;
    gn_sum2<TPR>(q, s, red, buf);
    rstd = rsqrtf(q * inv + eps);
}

template <typename TX, typename TY, int TPR, int V>
__global__ void __launch_bounds__(GnGeom<TPR>::NT) gn_fwd_kernel(GnArgs g)
{
    constexpr int G = GnGeom<TPR>::G;
    __shared__ float2 red[2][16];
    int buf = 0;
    const VpfGatedNorm& a = g.a;
    const int t = threadIdx.x % TPR, grp = threadIdx.x / TPR, D = a.D;
    const long r0 = (long)blockIdx.x * g.rows_per_wg, r1 = min(a.rows, r0 + g.rows_per_wg);
    float wp[GN_E], bp[GN_E], wn[GN_E], bn[GN_E], gt[GN_E];
    gn_param<TPR, V>(wp, a.has_post ? a.w_post : nullptr, t, D, 1.f);
    gn_param<TPR, V>(bp, a.has_post ? a.b_post : nullptr, t, D, 0.f);
    gn_param<TPR, V>(wn, a.w_pre, t, D, 1.f);
    gn_param<TPR, V>(bn, a.b_pre, t, D, 0.f);
#pragma unroll
    for (int e = 0; e < GN_E; ++e) gt[e] = 1.f;
    GnRaw<TX, TPR, V> rx;
    GnRaw<TY, TPR, V> ry_, rg;
    auto fetch = [&](long i) {
        const long r = min(i + grp, r1 - 1);                              // the last rows may be taken twice: every wave meets every barrier
        rx.fetch((const TX*)a.x + r * D, t, D);
        ry_.fetch((const TY*)a.y + r * D, t, D);
        if (a.gate_mode == VPF_GATE_FULL) rg.fetch((const TY*)a.gate + r * D, t, D);
    };
    fetch(r0);
    int sample = -1;
    for (long i = r0; i < r1; i += G) {
        const long r = min(i + grp, r1 - 1);
        const bool mine = i + grp < r1;
        float x[GN_E], y[GN_E];
        rx.get(x, t, D); ry_.get(y, t, D);
        if (a.gate_mode == VPF_GATE_FULL) rg.get(gt, t, D);
        else if (a.gate_mode == VPF_GATE_ROWS) {
            const int s = (int)((uint32_t)r / (uint32_t)a.gate_rows);
            if (s != sample) { gn_param<TPR, V>(gt, (const float*)a.gate + (long)s * D, t, D, 1.f); sample = s; }
        }
        fetch(i + G < r1 ? i + G : i);                                    // (unconditional: behind a branch its values would be awaited at the join)
        float my = 0.f, ry = 1.f, mh = 0.f, rh = 1.f;
        if (a.has_post) {
            gn_stats<TPR, V>(y, t, D, a.kind, a.eps_post, my, ry, red, buf);
#pragma unroll
            for (int e = 0; e < GN_E; ++e) y[e] = (y[e] - my) * ry * wp[e] + bp[e];
        }
#pragma unroll
        for (int e = 0; e < GN_E; ++e) {
            x[e] = a.alpha * x[e] + a.beta * gt[e] * y[e];
            if (V == 1 && gn_col<TPR, V>(t, e) >= D) x[e] = 0.f;
        }
        if (mine) gn_store<TX, TPR, V>((TX*)a.h + r * D, x, t, D);
        if (a.has_pre) {
            gn_stats<TPR, V>(x, t, D, a.kind, a.eps_pre, mh, rh, red, buf);
#pragma unroll
            for (int e = 0; e < GN_E; ++e) x[e] = (x[e] - mh) * rh * wn[e] + bn[e];
            if (mine) gn_store<TY, TPR, V>((TY*)a.n + r * D, x, t, D);
        }
        if (a.stats && mine && t == 0) {
            a.stats[r] = my; a.stats[a.rows + r] = ry; a.stats[2 * a.rows + r] = mh; a.stats[3 * a.rows + r] = rh;
        }
    }
}

// one accumulator of every thread -> one row of D column sums (over the workgroup's G row groups)
template <int TPR, int V>
__device__ __forceinline__ void gn_partial(const float* acc, float* dst, int t, int grp, int D, float* lds)
{
    constexpr int G = GnGeom<TPR>::G, NT = GnGeom<TPR>::NT;
    if constexpr (G == 1) { gn_store<float, TPR, V>(dst, acc, t, D); return; }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < GN_E; ++e) lds[grp * (TPR * GN_E) + gn_col<TPR, V>(t, e)] = acc[e];
    __syncthreads();
    for (int c = threadIdx.x; c < D; c += NT) {
        float s = 0.f;
#pragma unroll
        for (int k = 0; k < G; ++k) s += lds[k * (TPR * GN_E) + c];
        dst[c] = s;
    }
}

// ws: [4][nwg][D] partials of dw_post, db_post, dw_pre, db_pre, then [nwg + samples][D] of the gate: workgroup w's rows of sample s go to
// row w + s (unique: along consecutive rows at least one of the two rises from one (w, s) to the next).  g.single: [rows][D] of the gate instead.
template <typename TX, typename TY, int TPR, int V>
__global__ void __launch_bounds__(GnGeom<TPR>::NT) gn_bwd_kernel(GnArgs g)
{
    constexpr int G = GnGeom<TPR>::G;
    __shared__ float2 red[2][16];
    __shared__ float cols[G > 1 ? GnGeom<TPR>::NT * GN_E : 1];
    int buf = 0;
    const VpfGatedNorm& a = g.a;
    const int t = threadIdx.x % TPR, grp = threadIdx.x / TPR, D = a.D;
    const long r0 = (long)blockIdx.x * g.rows_per_wg, r1 = min(a.rows, r0 + g.rows_per_wg);
    const float inv = 1.f / (float)D, plain = a.kind == 0 ? 1.f : 0.f;    // RMS has no mean to take out
    const float live = V == 8 && 8 * t >= D ? 0.f : 1.f;
    float wp[GN_E], bp[GN_E], wn[GN_E], gt[GN_E], bg[GN_E], awp[GN_E], abp[GN_E], awn[GN_E], abn[GN_E], ag[GN_E];
    gn_param<TPR, V>(wp, a.has_post ? a.w_post : nullptr, t, D, 1.f);
    gn_param<TPR, V>(bp, a.has_post ? a.b_post : nullptr, t, D, 0.f);
    gn_param<TPR, V>(wn, a.w_pre, t, D, 1.f);
#pragma unroll
    for (int e = 0; e < GN_E; ++e) { gt[e] = 1.f; awp[e] = abp[e] = awn[e] = abn[e] = ag[e] = 0.f; }
    float* wsg = a.ws + 4L * g.nwg * D;
    for (long seg = r0; seg < r1;) {
        long end = r1;
        int s = 0;
        if (a.gate_mode == VPF_GATE_ROWS && !g.single) {
            s = (int)((uint32_t)seg / (uint32_t)a.gate_rows);
            end = min(r1, (long)(s + 1) * a.gate_rows);
            gn_param<TPR, V>(gt, (const float*)a.gate + (long)s * D, t, D, 1.f);
        }
        GnRaw<TX, TPR, V> rdh, rx;
        GnRaw<TY, TPR, V> rdn, ry_, rg;
        GnRaw<float, TPR, V> rgs;
        float s0, s1_, s2_, s3;
        auto fetch = [&](long i) {
            const long r = min(i + grp, end - 1);
            rdh.fetch((const TX*)a.dh + r * D, t, D);
            if (a.has_pre) rdn.fetch((const TY*)a.dn + r * D, t, D);
            rx.fetch((const TX*)a.x + r * D, t, D);
            ry_.fetch((const TY*)a.y + r * D, t, D);
            if (a.gate_mode == VPF_GATE_FULL) rg.fetch((const TY*)a.gate + r * D, t, D);
            if (g.single) rgs.fetch((const float*)a.gate + (long)((uint32_t)r / (uint32_t)a.gate_rows) * D, t, D);
            s0 = a.stats[r]; s1_ = a.stats[a.rows + r]; s2_ = a.stats[2 * a.rows + r]; s3 = a.stats[3 * a.rows + r];
        };
        fetch(seg);
        for (long i = seg; i < end; i += G) {
            const long r = min(i + grp, end - 1);
            const bool mine = i + grp < end;
            float x[GN_E], y[GN_E], dh[GN_E], dn[GN_E], u[GN_E];
            rdh.get(dh, t, D); rx.get(x, t, D); ry_.get(y, t, D);
            if (a.has_pre) rdn.get(dn, t, D);
            if (a.gate_mode == VPF_GATE_FULL) rg.get(gt, t, D);
            if (g.single) rgs.get(gt, t, D);
            const float ry = s1_, cy = -s0 * s1_, rh = s3, ch = -s2_ * s3;
            fetch(i + G < end ? i + G : i);                               // (unconditional: behind a branch its values would be awaited at the join)
            if (G > 1 && !mine) {                                         // a row taken twice: its gradients count once
#pragma unroll
                for (int e = 0; e < GN_E; ++e) dh[e] = dn[e] = 0.f;
            }
            if (a.gate_mode == VPF_GATE_FULL || g.single || i == seg) {
#pragma unroll
                for (int e = 0; e < GN_E; ++e) bg[e] = a.beta * gt[e];
            }
#pragma unroll
            for (int e = 0; e < GN_E; ++e) {
                y[e] = fmaf(y[e], ry, cy);                                // no post norm: mean 0, rstd 1
                u[e] = fmaf(y[e], wp[e], bp[e]);
            }
            if (a.has_pre) {
                float s1 = 0.f, s2 = 0.f;
#pragma unroll
                for (int e = 0; e < GN_E; ++e) {
                    x[e] = fmaf(fmaf(a.alpha, x[e], bg[e] * u[e]), rh, ch);
                    if (V == 1 && gn_col<TPR, V>(t, e) >= D) x[e] = 0.f;
                    awn[e] = fmaf(dn[e], x[e], awn[e]);
                }
                if (g.want & GN_WANT_BPRE) {
#pragma unroll
                    for (int e = 0; e < GN_E; ++e) abn[e] += dn[e];
                }
#pragma unroll
                for (int e = 0; e < GN_E; ++e) { dn[e] *= wn[e]; s1 += dn[e]; s2 = fmaf(dn[e], x[e], s2); }
                s1 *= live; s2 *= live;
                gn_sum2<TPR>(s1, s2, red, buf);
                s1 *= inv * plain; s2 *= inv;
#pragma unroll
                for (int e = 0; e < GN_E; ++e) dh[e] = fmaf(rh, fmaf(-x[e], s2, dn[e] - s1), dh[e]);
            }
            if (a.dx && mine) {
#pragma unroll
                for (int e = 0; e < GN_E; ++e) x[e] = a.alpha * dh[e];
                gn_store<TX, TPR, V>((TX*)a.dx + r * D, x, t, D);
            }
            if (a.gate_mode == VPF_GATE_FULL) {
                if (a.dgate && mine) {
#pragma unroll
                    for (int e = 0; e < GN_E; ++e) x[e] = a.beta * dh[e] * u[e];
                    gn_store<TY, TPR, V>((TY*)a.dgate + r * D, x, t, D);
                }
            } else if (g.single) {
                if ((g.want & GN_WANT_GATE) && mine) {
#pragma unroll
                    for (int e = 0; e < GN_E; ++e) x[e] = a.beta * dh[e] * u[e];
                    gn_store<float, TPR, V>(wsg + r * D, x, t, D);
                }
            } else if (g.want & GN_WANT_GATE) {
#pragma unroll
                for (int e = 0; e < GN_E; ++e) ag[e] = fmaf(dh[e], u[e], ag[e]);      // (times beta when it is written)
            }
            float f1 = 0.f, f2 = 0.f;
#pragma unroll
            for (int e = 0; e < GN_E; ++e) {
                if (V == 1 && gn_col<TPR, V>(t, e) >= D) dh[e] = 0.f;
                dh[e] *= bg[e];
                awp[e] = fmaf(dh[e], y[e], awp[e]);
            }
            if (g.want & GN_WANT_BPOST) {
#pragma unroll
                for (int e = 0; e < GN_E; ++e) abp[e] += dh[e];
            }
#pragma unroll
            for (int e = 0; e < GN_E; ++e) { dh[e] *= wp[e]; f1 += dh[e]; f2 = fmaf(dh[e], y[e], f2); }
            if (a.has_post) {
                f1 *= live; f2 *= live;
                gn_sum2<TPR>(f1, f2, red, buf);
                f1 *= inv * plain; f2 *= inv;
#pragma unroll
                for (int e = 0; e < GN_E; ++e) dh[e] = ry * fmaf(-y[e], f2, dh[e] - f1);
            }
            if (a.dy && mine) gn_store<TY, TPR, V>((TY*)a.dy + r * D, dh, t, D);
        }
        if ((g.want & GN_WANT_GATE) && !g.single) {
#pragma unroll
            for (int e = 0; e < GN_E; ++e) ag[e] *= a.beta;
            gn_partial<TPR, V>(ag, wsg + ((long)blockIdx.x + s) * D, t, grp, D, cols);
#pragma unroll
            for (int e = 0; e < GN_E; ++e) ag[e] = 0.f;
        }
        seg = end;
    }
    auto slot = [&](int k) { return a.ws + ((long)k * g.nwg + blockIdx.x) * D; };
    if (g.want & GN_WANT_WPOST) gn_partial<TPR, V>(awp, slot(0), t, grp, D, cols);
    if (g.want & GN_WANT_BPOST) gn_partial<TPR, V>(abp, slot(1), t, grp, D, cols);
    if (g.want & GN_WANT_WPRE) gn_partial<TPR, V>(awn, slot(2), t, grp, D, cols);
    if (g.want & GN_WANT_BPRE) gn_partial<TPR, V>(abn, slot(3), t, grp, D, cols);
}

// Partial rows -> sums: workgroup = 64 columns of one result (the four parameters, then the gate of every sample), 16 slices of the partial
// rows in parallel, joined in LDS in a fixed order.
__global__ void __launch_bounds__(64 * GN_FOLD_SLICES) gn_fold_kernel(GnArgs g, int col_blocks, long items)
{
    __shared__ float part[GN_FOLD_SLICES][64];
    const VpfGatedNorm& a = g.a;
    const int lane = threadIdx.x & 63, sl = threadIdx.x >> 6;
    for (long item = blockIdx.x; item < items; item += gridDim.x) {
        const long k = item / col_blocks;
        const int c = (int)(item % col_blocks) * 64 + lane;
        if (k < 4 && !(g.want & (1 << k))) continue;
        const float* src;
        long n;
        if (k < 4) { src = a.ws + k * g.nwg * a.D; n = g.nwg; }
        else if (g.single) { src = a.ws + (4L * g.nwg + (k - 4) * a.gate_rows) * a.D; n = a.gate_rows; }
        else {
            const long s = k - 4, w0 = s * a.gate_rows / g.rows_per_wg, w1 = ((s + 1) * a.gate_rows - 1) / g.rows_per_wg;
            src = a.ws + (4L * g.nwg + w0 + s) * a.D; n = w1 - w0 + 1;
        }
        const long per = (n + GN_FOLD_SLICES - 1) / GN_FOLD_SLICES, b = min(n, sl * per), e = min(n, b + per);
        float s0 = 0.f, s1 = 0.f, s2 = 0.f, s3 = 0.f;
        if (c < a.D) {
            long i = b;
            for (; i + 3 < e; i += 4) {
                s0 += src[i * a.D + c]; s1 += src[(i + 1) * a.D + c]; s2 += src[(i + 2) * a.D + c]; s3 += src[(i + 3) * a.D + c];
            }
            for (; i < e; ++i) s0 += src[i * a.D + c];
        }
        part[sl][lane] = (s0 + s1) + (s2 + s3);
        __syncthreads();
        if (sl == 0 && c < a.D) {
            float s = 0.f;
#pragma unroll
            for (int j = 0; j < GN_FOLD_SLICES; ++j) s += part[j][lane];
            switch (k) {
                case 0: a.dw_post[c] = s; break;
                case 1: a.db_post[c] = s; break;
                case 2: a.dw_pre[c] = s; break;
                case 3: a.db_pre[c] = s; break;
                default: ((float*)a.dgate)[(k - 4) * a.D + c] = s;
            }
        }
        __syncthreads();
    }
}

// threads of a row: the smallest power of two whose 8 values each cover it
static int gn_tpr(int D) { int t = 16; while (t * GN_E < D) t *= 2; return t; }
static int gn_groups(int D) { const int t = gn_tpr(D); return t <= 256 ? 256 / t : 1; }
static void gn_plan(GnArgs& g, int want_wgs)
{
    const int G = gn_groups(g.a.D);
    long per = (g.a.rows + want_wgs - 1) / want_wgs;
    per = (per + G - 1) / G * G;
    g.rows_per_wg = (int)per;
    g.nwg = vpf_cdiv(g.a.rows, per);
}
// Backward: a workgroup walks at least 4 row groups, so that its partial rows (5 D floats) stay small beside what it reads, and the
// partials are at most 512 rows (two workgroups per CU, the next row of each in flight).  Measured on 32768 x 2048 in bf16, kernel + fold:
// 512 177 + 6 us, 768 215 + 10, 1024 177 + 14, 1536 189 + 19.
static void gn_plan_bwd(GnArgs& g)
{
    const long want = g.a.rows / (4L * gn_groups(g.a.D)) + 1;
    gn_plan(g, want < 512 ? (int)want : 512);
    const VpfGatedNorm& a = g.a;
    g.want = (a.has_post && a.dw_post ? GN_WANT_WPOST : 0) | (a.has_post && a.db_post ? GN_WANT_BPOST : 0) | (a.has_pre && a.dw_pre ? GN_WANT_WPRE : 0) |
             (a.has_pre && a.db_pre ? GN_WANT_BPRE : 0) | (a.gate_mode == VPF_GATE_ROWS && a.dgate ? GN_WANT_GATE : 0);
    // a gate row that serves fewer rows than two walks of a workgroup's row groups: segments of its own would leave most groups idle
    g.single = a.gate_mode == VPF_GATE_ROWS && a.gate_rows < 2 * gn_groups(a.D);
}
static long gn_samples(const VpfGatedNorm& a) { return a.gate_mode == VPF_GATE_ROWS ? a.rows / a.gate_rows : 0; }

static long gn_ws_floats(const GnArgs& g) { return (4L * g.nwg + (g.single ? g.a.rows : g.nwg + gn_samples(g.a))) * g.a.D; }

static int gn_check(const VpfGatedNorm& a)
{
    if (a.rows < 0 || a.rows > 0x7fffffffL || a.D < 1 || a.D > VPF_GATED_NORM_MAX_D || a.kind < 0 || a.kind > 1) return VPF_ERR_BADSHAPE;
    if (a.gate_mode < VPF_GATE_NONE || a.gate_mode > VPF_GATE_FULL) return VPF_ERR_UNSUPPORTED;
    if (a.gate_mode == VPF_GATE_ROWS && (a.gate_rows < 1 || a.rows % a.gate_rows)) return VPF_ERR_BADSHAPE;
    if (!vpf_elem_ok(a.x_type) || !vpf_elem_ok(a.y_type) || (a.x_type != VPF_T_F32 && a.x_type != a.y_type)) return VPF_ERR_UNSUPPORTED;
    return VPF_OK;
}
// 16-byte accesses: whole chunks of 8 columns and aligned bases
static bool gn_vec(const VpfGatedNorm& a, bool bwd)
{
    if (a.D % 8) return false;
    const void* p[] = {a.x, a.y, a.gate, a.w_post, a.b_post, a.w_pre, a.b_pre, a.h, a.n};
    const void* q[] = {a.dh, a.dn, a.dx, a.dy, a.dgate, a.ws};
    for (const void* i : p) if (!vpf_aligned(i, 16)) return false;
    if (bwd) for (const void* i : q) if (!vpf_aligned(i, 16)) return false;
    return true;
}

template <typename TX, typename TY, int V, bool BWD>
static int gn_launch(const GnArgs& g, hipStream_t st)
{
    switch (gn_tpr(g.a.D)) {
#define GN_CASE(T) case T: \
        if (BWD) hipLaunchKernelGGL((gn_bwd_kernel<TX, TY, T, V>), dim3(g.nwg), dim3(GnGeom<T>::NT), 0, st, g); \
        else hipLaunchKernelGGL((gn_fwd_kernel<TX, TY, T, V>), dim3(g.nwg), dim3(GnGeom<T>::NT), 0, st, g); \
        break;
        GN_CASE(16) GN_CASE(32) GN_CASE(64) GN_CASE(128) GN_CASE(256) GN_CASE(512) GN_CASE(1024)
#undef GN_CASE
        default: return VPF_ERR_BADSHAPE;
    }
    VPF_CHECK_LAUNCH();
    return VPF_OK;
}
template <bool BWD>
static int gn_pick(const GnArgs& g, hipStream_t st)
{
    const VpfGatedNorm& a = g.a;
    const bool v = gn_vec(a, BWD);
#define GN_TYPES(X, Y) return v ? gn_launch<X, Y, 8, BWD>(g, st) : gn_launch<X, Y, 1, BWD>(g, st)
    if (a.x_type == VPF_T_F32) {
        if (a.y_type == VPF_T_F32) GN_TYPES(float, float);
        if (a.y_type == VPF_T_F16) GN_TYPES(float, vpf_f16);
        GN_TYPES(float, vpf_bf16);
    }
    if (a.x_type == VPF_T_F16) GN_TYPES(vpf_f16, vpf_f16);
    GN_TYPES(vpf_bf16, vpf_bf16);
#undef GN_TYPES
}

extern "C" int vpf_gated_norm_fwd(const VpfGatedNorm* args, void* stream)
{
    (void)hipGetLastError();
    if (!args) return VPF_ERR_NULL;
    GnArgs g = {*args, 0, 0, 0, 0};
    const VpfGatedNorm& a = g.a;
    if (const int rc = gn_check(a)) return rc;
    if (a.rows == 0) return VPF_OK;
    if (!a.x || !a.y || !a.h || (a.has_pre && !a.n) || (a.gate_mode != VPF_GATE_NONE && !a.gate)) return VPF_ERR_NULL;
    gn_plan(g, 2048);
    return gn_pick<false>(g, (hipStream_t)stream);
}

extern "C" long vpf_gated_norm_ws(const VpfGatedNorm* args)
{
    if (!args) return VPF_ERR_NULL;
    GnArgs g = {*args, 0, 0, 0, 0};
    if (const int rc = gn_check(g.a)) return rc;
    if (g.a.rows == 0) return 0;
    gn_plan_bwd(g);
    return gn_ws_floats(g);
}

extern "C" int vpf_gated_norm_bwd(const VpfGatedNorm* args, void* stream)
{
    (void)hipGetLastError();
    if (!args) return VPF_ERR_NULL;
    GnArgs g = {*args, 0, 0, 0, 0};
    const VpfGatedNorm& a = g.a;
    if (const int rc = gn_check(a)) return rc;
    if (a.rows == 0) return VPF_OK;
    if (!a.x || !a.y || !a.dh || !a.stats || (a.has_pre && !a.dn) || (a.gate_mode != VPF_GATE_NONE && !a.gate) || !a.ws) return VPF_ERR_NULL;
    gn_plan_bwd(g);
    const long samples = gn_samples(a);
    if (a.ws_floats < gn_ws_floats(g)) return VPF_ERR_BADSHAPE;
    if (const int rc = gn_pick<true>(g, (hipStream_t)stream)) return rc;
    if (!g.want) return VPF_OK;
    const int cb = vpf_cdiv(a.D, 64);
    const long items = cb * (4 + (g.want & GN_WANT_GATE ? samples : 0));
    hipLaunchKernelGGL(gn_fold_kernel, dim3((unsigned)(items < 65536 ? items : 65536)), dim3(64 * GN_FOLD_SLICES), 0, (hipStream_t)stream, g, cb, items);
    VPF_CHECK_LAUNCH();
    return VPF_OK;
}
