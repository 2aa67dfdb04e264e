// rotary.hip -- rotary positions with several axes on queries and keys (gfx950).
//
// Pair p of a head's channels belongs to one axis a(p) of the token's position and turns by the angle pos[a(p)] * freq[p]:
//   (x0, x1) -> (x0 cos - x1 sin, x1 cos + x0 sin)
// The gradient is the same rotation by the negative angle, so one kernel does both directions.
// The angle is formed in fp64 and reduced to a fraction of a turn before it becomes fp32: at position 10^6 an fp32 product has lost
// 0.06 rad.  An angle serves every head of its token, so a workgroup puts cos / sin of its tokens into LDS once (one fp64 product and
// one sincospi per angle) while its first q / k loads are in flight; what remains is one read and one write of q and k: HBM bound.
#include "vpf_elem.h"

#define ROT_THREADS 256
#define ROT_ITEMS 4             // chunks a thread has in flight: loads of all of them are issued in front of the angle table
#define ROT_TOKENS 64           // tokens a workgroup takes at most

struct RotArgs {
    VpfRotary a;
    int tok;                    // tokens per workgroup
    int blocks;                 // workgroups per sample
    int rot_chunks, chunks;     // chunks of a head: rotated ones, all of them (the rest is copied)
};

__device__ __forceinline__ double rot_pos(const VpfRotary& a, size_t i)
{
    switch (a.pos_type) {
        case VPF_POS_F32: return (double)((const float*)a.pos)[i];
        case VPF_POS_F64: return ((const double*)a.pos)[i];
        case VPF_POS_I32: return (double)((const int*)a.pos)[i];
        default: return (double)((const long long*)a.pos)[i];
    }
}

// A chunk is what one thread rotates at a time: HALF: V channels at c and the V partners at c + P; otherwise: V pairs side by side
// (2 V channels).  Chunks behind rot_chunks are copied: V (HALF) or 2 V channels each.
template <typename T, int V, bool HALF>
__global__ void __launch_bounds__(ROT_THREADS) rotary_kernel(RotArgs r)
{
    extern __shared__ float2 rot_table[];                       // [tok][P]
    const VpfRotary& a = r.a;
    const int b = blockIdx.x / r.blocks, t0 = (blockIdx.x % r.blocks) * r.tok;
    const int nt = min(r.tok, a.L - t0), H = a.Hq + a.Hk;
    const int per = H * r.chunks, n = nt * per;

    struct Item { const T* src; T* dst; int t, c; };
    auto locate = [&](int i) {
        Item it;
        it.t = i / per;
        const int rest = i - it.t * per, head = rest / r.chunks;
        it.c = rest - head * r.chunks;
        const long tok = t0 + it.t;
        if (head < a.Hq) {
            it.src = (const T*)a.q + b * a.q_sb + tok * a.q_sl + head * a.q_sh;
            it.dst = (T*)a.oq + b * a.oq_sb + tok * a.oq_sl + head * a.oq_sh;
        } else {
            const int hk = head - a.Hq;
            it.src = (const T*)a.k + b * a.k_sb + tok * a.k_sl + hk * a.k_sh;
            it.dst = (T*)a.ok + b * a.ok_sb + tok * a.ok_sl + hk * a.ok_sh;
        }
        return it;
    };
    bool table = false;
    for (int base = 0; base < n; base += ROT_THREADS * ROT_ITEMS) {
        float x[ROT_ITEMS][2 * V];
#pragma unroll
        for (int j = 0; j < ROT_ITEMS; ++j) {
            const int i = base + j * ROT_THREADS + threadIdx.x;
            if (i >= n) continue;
            const Item it = locate(i);
            if (it.c < r.rot_chunks) {
                if (HALF) { vpf_load<T, V>(x[j], it.src + it.c * V); vpf_load<T, V>(x[j] + V, it.src + a.P + it.c * V); }
                else vpf_load<T, 2 * V>(x[j], it.src + it.c * 2 * V);
            } else if (HALF) vpf_load<T, V>(x[j], it.src + 2 * a.P + (it.c - r.rot_chunks) * V);
            else vpf_load<T, 2 * V>(x[j], it.src + it.c * 2 * V);
        }
        if (!table) {
            for (int i = threadIdx.x; i < nt * a.P; i += ROT_THREADS) {
                const int t = i / a.P, p = i - t * a.P;
                const double turns = rot_pos(a, (size_t)b * a.pos_sb + (size_t)(t0 + t) * a.axes + a.axis[p]) * a.freq[p];
                float s, c;
                sincospif(2.0f * (float)(turns - rint(turns)), &s, &c);
                rot_table[i] = make_float2(c, a.inverse ? -s : s);
            }
            __syncthreads();
            table = true;
        }
#pragma unroll
        for (int j = 0; j < ROT_ITEMS; ++j) {
            const int i = base + j * ROT_THREADS + threadIdx.x;
            if (i >= n) continue;
            const Item it = locate(i);
            if (it.c < r.rot_chunks) {
                const float2* cs = rot_table + it.t * a.P + it.c * V;
                float y[2 * V];
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const float2 w = cs[e];
                    const float x0 = HALF ? x[j][e] : x[j][2 * e], x1 = HALF ? x[j][V + e] : x[j][2 * e + 1];
                    y[HALF ? e : 2 * e] = x0 * w.x - x1 * w.y;
                    y[HALF ? V + e : 2 * e + 1] = x1 * w.x + x0 * w.y;
                }
                if (HALF) { vpf_store<T, V>(it.dst + it.c * V, y); vpf_store<T, V>(it.dst + a.P + it.c * V, y + V); }
                else vpf_store<T, 2 * V>(it.dst + it.c * 2 * V, y);
            } else if (HALF) vpf_store<T, V>(it.dst + 2 * a.P + (it.c - r.rot_chunks) * V, x[j]);
            else vpf_store<T, 2 * V>(it.dst + it.c * 2 * V, x[j]);
        }
    }
}

template <typename T, int V, bool HALF>
static int rotary_launch(const VpfRotary& a, hipStream_t st)
{
    RotArgs r;
    r.a = a;
    r.rot_chunks = a.P / V;
    r.chunks = r.rot_chunks + (a.head_dim - 2 * a.P) / (HALF ? V : 2 * V);
    // Tokens per workgroup: enough that every thread holds ROT_ITEMS chunks and the angle table is shared by them, but no fewer than
    // about 1024 workgroups (four per CU) where the call has that many tokens.
    const long per = (long)(a.Hq + a.Hk) * r.chunks, tokens = (long)a.B * a.L;
    long tok = (ROT_THREADS * ROT_ITEMS + per - 1) / per;
    tok = tok < tokens / 1024 + 1 ? tok : tokens / 1024 + 1;
    tok = tok < ROT_TOKENS ? tok : ROT_TOKENS;
    const long fits = 65536 / (long)sizeof(float2) / a.P;
    tok = tok < fits ? tok : fits;
    r.tok = (int)(tok < a.L ? tok : a.L);
    r.blocks = vpf_cdiv(a.L, r.tok);
    const long grid = (long)a.B * r.blocks;
    if (grid > 0x7fffffffL) return VPF_ERR_BADSHAPE;
    hipLaunchKernelGGL((rotary_kernel<T, V, HALF>), dim3((unsigned)grid), dim3(ROT_THREADS), sizeof(float2) * r.tok * a.P, st, r);
    VPF_CHECK_LAUNCH();
    return VPF_OK;
}

template <typename T>
static int rotary_pick(const VpfRotary& a, hipStream_t st)
{
    // widest access that divides the rotated and the copied part of a head and every base address and stride
    const long strides[12] = {a.q_sb, a.q_sl, a.q_sh, a.oq_sb, a.oq_sl, a.oq_sh, a.Hk ? a.k_sb : 0, a.Hk ? a.k_sl : 0, a.Hk ? a.k_sh : 0,
                              a.Hk ? a.ok_sb : 0, a.Hk ? a.ok_sl : 0, a.Hk ? a.ok_sh : 0};
    auto fits = [&](int v, bool half) {
        const int w = half ? v : 2 * v;                        // channels of one access
        if (a.P % v || (a.head_dim - 2 * a.P) % w) return false;
        for (long s : strides) if (s % w) return false;
        const size_t by = sizeof(T) * w < 16 ? sizeof(T) * w : 16;
        return vpf_aligned(a.q, by) && vpf_aligned(a.oq, by) && vpf_aligned(a.k, by) && vpf_aligned(a.ok, by);
    };
    if (a.layout == VPF_ROTARY_HALF) {
        constexpr int V = sizeof(T) == 4 ? 4 : 8;
        if (fits(V, true)) return rotary_launch<T, V, true>(a, st);
        if (fits(V / 2, true)) return rotary_launch<T, V / 2, true>(a, st);
        if (fits(2, true)) return rotary_launch<T, 2, true>(a, st);
        return rotary_launch<T, 1, true>(a, st);
    }
    constexpr int V = sizeof(T) == 4 ? 2 : 4;
    if (fits(V, false)) return rotary_launch<T, V, false>(a, st);
    if (fits(1, false)) return rotary_launch<T, 1, false>(a, st);
    return VPF_ERR_BADALIGN;
}

extern "C" int vpf_rotary_axes(const VpfRotary* args, void* stream)
{
    (void)hipGetLastError();
    if (!args) return VPF_ERR_NULL;
    const VpfRotary& a = *args;
    if (a.B < 0 || a.L < 0 || a.Hq < 0 || a.Hk < 0 || a.head_dim <= 0 || a.P <= 0 || 2 * a.P > a.head_dim || a.head_dim > VPF_ROTARY_MAX_DIM ||
        a.axes < 1 || a.axes > VPF_ROTARY_MAX_AXES || a.Hq > 4096 || a.Hk > 4096) return VPF_ERR_BADSHAPE;
    if (a.layout != VPF_ROTARY_HALF && a.layout != VPF_ROTARY_PAIR) return VPF_ERR_UNSUPPORTED;
    if (a.pos_type < VPF_POS_F32 || a.pos_type > VPF_POS_I64 || !vpf_elem_ok(a.dtype)) return VPF_ERR_UNSUPPORTED;
    if ((long)a.B * a.L * (a.Hq + a.Hk) == 0) return VPF_OK;
    if (!a.pos || !a.freq || !a.axis || (a.Hq && (!a.q || !a.oq)) || (a.Hk && (!a.k || !a.ok))) return VPF_ERR_NULL;
    hipStream_t st = (hipStream_t)stream;
    if (a.dtype == VPF_T_F32) return rotary_pick<float>(a, st);
    if (a.dtype == VPF_T_F16) return rotary_pick<vpf_f16>(a, st);
    return rotary_pick<vpf_bf16>(a, st);
}
