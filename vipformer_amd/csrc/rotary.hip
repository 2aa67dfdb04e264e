// rotary.hip -- rotary positions with several axes on queries and keys (gfx950).
//
// Pair p of a head's channels belongs to one axis a(p) of the token's position and turns by the angle pos[a(p)] * freq[p]:
//   (x0, x1) -> (x0 cos - x1 sin, x1 cos + x0 sin)
// The gradient is the same rotation by the negative angle, so one kernel does both directions.
// The angle is formed in fp64 and reduced to a fraction of a turn before it becomes fp32: at position 10^6 an fp32 product has lost
// 0.06 rad.  An angle serves every head of its token, so a workgroup puts cos / sin of its tokens into LDS once (one fp64 product and
// one sincospi per angle) while its first q / k loads are in flight; what remains is one read and one write of q and k: HBM bound.
#include "vpf_elem.h"

#define ROT_BYTES 64            // bytes a thread has in flight (32, 64, 128, 256: 43, 45, 48, 51 us with 2 x 16 bytes an access, 71, 64, 67, 67 with 16)
#define ROT_MAX_THREADS 1024

struct RotArgs {
    VpfRotary a;
    int tok;                    // tokens per workgroup
    int blocks;                 // workgroups per sample
    int rot_chunks, chunks;     // chunks of a head: rotated ones, all of them (the rest is copied)
    int side;                   // tokens side by side in a workgroup
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
// A thread keeps its head and chunk and walks over tokens, ITEMS of them in flight: the divisions and the pointers are made once.
template <typename T, int V, bool HALF>
__global__ void __launch_bounds__(ROT_MAX_THREADS) rotary_kernel(RotArgs r)
{
    constexpr int N = 2 * V * (int)sizeof(T), ITEMS = ROT_BYTES / N < 1 ? 1 : ROT_BYTES / N > 8 ? 8 : ROT_BYTES / N;
    extern __shared__ float2 rot_table[];                       // [tok][P]
    const VpfRotary& a = r.a;
    const int b = blockIdx.x / r.blocks, t0 = (blockIdx.x % r.blocks) * r.tok, nt = min(r.tok, a.L - t0);
    const int H = a.Hq + a.Hk, per = H * r.chunks, sub = (int)threadIdx.x / per;
    bool table = false;
    // (one turn of the outer loop unless a token has more chunks than the workgroup threads)
    for (int base = 0; base < per; base += blockDim.x) {
        const bool mine = sub < r.side && base + (int)threadIdx.x - sub * per < per;
        const int item = mine ? base + threadIdx.x - sub * per : 0, head = item / r.chunks, c = item - head * r.chunks;
        const bool isq = head < a.Hq, turned = c < r.rot_chunks;
        const int h = isq ? head : head - a.Hq;
        const long sl = isq ? a.q_sl : a.k_sl, ol = isq ? a.oq_sl : a.ok_sl;
        const int at = HALF ? (turned ? c * V : 2 * a.P + (c - r.rot_chunks) * V) : c * 2 * V;
        const T* src = (isq ? (const T*)a.q + b * a.q_sb + h * a.q_sh : (const T*)a.k + b * a.k_sb + h * a.k_sh) + t0 * sl + at;
        T* dst = (isq ? (T*)a.oq + b * a.oq_sb + h * a.oq_sh : (T*)a.ok + b * a.ok_sb + h * a.ok_sh) + t0 * ol + at;
        const int partner = turned ? a.P : 0;
        for (int first = 0; first < nt; first += ITEMS * r.side) {
            VpfRaw<T, HALF ? V : 2 * V> x[ITEMS], z[HALF ? ITEMS : 1];
#pragma unroll
            for (int j = 0; j < ITEMS; ++j) {                   // (tokens behind the last one: the last one again, dropped below)
                const T* p = src + min(first + j * r.side + sub, nt - 1) * sl;
                x[j].load(p);
                if (HALF) z[j].load(p + partner);
            }
            if (!table) {
                for (int i = threadIdx.x; i < nt * a.P; i += blockDim.x) {
                    const int t = i / a.P, p = i - t * a.P;
                    const double turns = rot_pos(a, (size_t)b * a.pos_sb + (size_t)(t0 + t) * a.axes + a.axis[p]) * a.freq[p];
                    float s, co;
                    sincospif(2.0f * (float)(turns - rint(turns)), &s, &co);
                    rot_table[i] = make_float2(co, a.inverse ? -s : s);
                }
                __syncthreads();
                table = true;
            }
#pragma unroll
            for (int j = 0; j < ITEMS; ++j) {
                const int t = first + j * r.side + sub;
                if (!mine || t >= nt) continue;
                T* p = dst + t * ol;
                float y[2 * V];
                if (turned) {
                    const float2* cs = rot_table + t * a.P + c * V;
#pragma unroll
                    for (int e = 0; e < V; ++e) {
                        const float2 w = cs[e];
                        const float x0 = HALF ? x[j].get(e) : x[j].get(2 * e), x1 = HALF ? z[j].get(e) : x[j].get(2 * e + 1);
                        y[HALF ? e : 2 * e] = x0 * w.x - x1 * w.y;
                        y[HALF ? V + e : 2 * e + 1] = x1 * w.x + x0 * w.y;
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < (HALF ? V : 2 * V); ++e) y[e] = x[j].get(e);
                }
                if (!HALF) vpf_store<T, 2 * V>(p, y);
                else { vpf_store<T, V>(p, y); if (turned) vpf_store<T, V>(p + a.P, y + V); }
            }
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
    // A workgroup is as many whole tokens side by side as 256 threads hold (one, with up to 1024 threads, where a token has more chunks).
    const int per = (a.Hq + a.Hk) * r.chunks;
    r.side = per <= 256 ? 256 / per : 1;
    const int threads = vpf_cdiv((long)r.side * per < ROT_MAX_THREADS ? (long)r.side * per : ROT_MAX_THREADS, 64) * 64;
    // Its tokens: one full set in flight, fewer where the call would not leave about 1024 workgroups (four per CU).
    constexpr int N = 2 * V * (int)sizeof(T), ITEMS = ROT_BYTES / N < 1 ? 1 : ROT_BYTES / N > 8 ? 8 : ROT_BYTES / N;
    const long tokens = (long)a.B * a.L, fits = 65536 / (long)sizeof(float2) / a.P;
    long deep = tokens / (1024L * r.side);
    deep = deep < 1 ? 1 : deep < ITEMS ? deep : ITEMS;
    long tok = deep * r.side;
    tok = tok < fits ? tok : fits;
    r.tok = (int)(tok < a.L ? tok : a.L);
    r.blocks = vpf_cdiv(a.L, r.tok);
    const long grid = (long)a.B * r.blocks;
    if (grid * threads >= 1L << 32) return VPF_ERR_BADSHAPE;          // (a launch counts its threads in 32 bits)
    hipLaunchKernelGGL((rotary_kernel<T, V, HALF>), dim3((unsigned)grid), dim3(threads), sizeof(float2) * r.tok * a.P, st, r);
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
