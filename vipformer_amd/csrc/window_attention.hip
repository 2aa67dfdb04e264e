// window_attention.hip -- attention inside a sliding window with first tokens that stay visible (gfx950), fp16 and bf16.
//
// Query i of a sample stands at position p = n - Lq + i (n keys in use) and sees key j where
//   j < n,  j <= p + right,  (j >= p - left  or  j < sinks),  and j is not padding.
// out = softmax(scale q k^T over the visible keys) v; a query that sees nothing gets zeros.
//
// Shared key heads: the g = Hq / Hk query heads of a key head are rows of ONE matrix, row r = query r / g, head r % g, so a tile of K and V
// serves all of them and a single token over a cache still fills a matrix tile.
//
// Layout of the products (key index in registers, row on the lane), as in attention.hip:
//   S^T[key, row] = K[key, :] . Q[row, :]        A = K rows (LDS), B = Q (registers)
//   O^T[d, row] += V^T[d, key] . P^T[key, row]   A = V columns (LDS, transposing reads), B = P straight from the accumulators of S^T
// Statistics are per-lane scalars in fp32, in units of log2; P is rounded to the tensors' type for the second product (at most 2^-8 / 2^-11
// relative for each weight, the size of the output's own rounding).  fp16 has that precision down to 2^-14 only, and behind a first token that
// takes nearly all the weight the others can lie far below: forward's weights are lifted by WaMma::LIFT powers of two (their sum with them).
//
// LDS tiles hold rows of NC 16-byte chunks without padding; chunk c of row r sits at c ^ swz(r).  Over 64 banks of 4 bytes a fragment read
// takes the same chunk of 16 consecutive rows (they must differ modulo 16 chunks) and a transposing read takes 4 chunks side by side of 4
// consecutive rows (they must fall into the 4 groups of 4 chunks): swz does both.
#include "vpf_elem.h"

typedef __attribute__((ext_vector_type(4))) short wa_s16x4;
typedef __attribute__((ext_vector_type(8))) short wa_s16x8;
typedef __attribute__((ext_vector_type(16))) float wa_f32x16;
#define WA_LOG2E 1.4426950408889634f
#define WA_THREADS 256
#define WA_MAX_GRID (1L << 23)          // workgroups of up to 512 threads: a launch counts its threads in 32 bits
#define WA_FAR (1 << 30)                // an open side of the window; positions and lengths stay below it

template <typename T> struct WaMma;
template <> struct WaMma<vpf_f16> {
    static constexpr bool NARROW = true;    // 5 bits of exponent: what is rounded to it for a product is scaled first
    static constexpr float GROW = 4.f, LIFT = 11.f;     // weights up to 2^(GROW + LIFT) = 32768; full precision down to 2^-25 of the largest
    typedef __attribute__((ext_vector_type(8))) vpf_f16 v8;
    static __device__ __forceinline__ wa_f32x16 mma(v8 a, v8 b, wa_f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
};
template <> struct WaMma<vpf_bf16> {
    static constexpr bool NARROW = false;
    static constexpr float GROW = 8.f, LIFT = 0.f;
    typedef __attribute__((ext_vector_type(8))) vpf_bf16 v8;
    static __device__ __forceinline__ wa_f32x16 mma(v8 a, v8 b, wa_f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
};

struct WaArgs {
    VpfWindowAttn a;
    int g, rows;                // query heads per key head; rows of one (sample, key head)
    uint32_t magic;             // r / g == umulhi(r, magic) for r < 2^32 / g (g > 1)
    int tiles, splits, runs;    // row tiles; parts of a row tile's keys; order of the workgroups (wa_item)
    float c;                    // scale * log2(e)
    int key_tile, ktiles, sink_tiles, chunks, chunk_rows;      // backward: keys of a tile, tiles, those with sinks, pieces of the rows far behind those and their size
    int cycle;                  // row blocks between two common starting points of the key tiles' walks
};
// backward scratch: delta of every row (whole 16-byte pieces), in fp16 also its lse - WA_LIFT, then the pieces
#define WA_LIFT 15              // backward's weights are at most 1: fp16 takes them times 2^15 (full precision down to 2^-29)
__host__ __device__ static inline size_t wa_delta_floats(const WaArgs& w) { return ((size_t)w.a.B * w.a.Hk * w.rows + 3) / 4 * 4; }
__host__ __device__ static inline size_t wa_row_floats(const WaArgs& w) { return wa_delta_floats(w) * (w.a.dtype == VPF_T_F16 ? 2 : 1); }

__device__ __forceinline__ int wa_query(const WaArgs& w, int r) { return w.g == 1 ? r : (int)__umulhi((uint32_t)r, w.magic); }
__device__ __forceinline__ float wa_exp2(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float wa_half_max(float v)
{
    const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(s[0]), __uint_as_float(s[1]));
}
__device__ __forceinline__ float wa_half_sum(float v)
{
    const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(s[0]) + __uint_as_float(s[1]);
}
__device__ __forceinline__ wa_f32x16 wa_zero16()
{
    wa_f32x16 z;
#pragma unroll
    for (int r = 0; r < 16; ++r) z[r] = 0.f;
    return z;
}
template <typename T> __device__ __forceinline__ typename WaMma<T>::v8 wa_pack8(const float* f)
{
    typename WaMma<T>::v8 v;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (T)f[i];
    return v;
}

// ------------------------------------------------------------------ LDS tiles
template <int DP> struct WaTile {
    static constexpr int CH = DP / 8;                                       // 16-byte chunks of a row that hold data
    static constexpr int NC = DP <= 32 ? 4 : DP <= 64 ? 8 : 16;             // chunks of a row in LDS
    static constexpr int PITCH = NC * 16;
    static __device__ __forceinline__ int swz(int r)
    {
        return NC == 16 ? ((r & 3) << 2) | ((r >> 2) & 3) : NC == 8 ? (((r >> 1) & 1) << 2) | ((r >> 2) & 3) : (r >> 2) & 3;
    }
    static __device__ __forceinline__ int at(int r, int c) { return r * PITCH + ((c ^ swz(r)) << 4); }
};
// Fragment addresses are LDS bytes.  The chunk number is XORed into bits that the row leaves zero, so ONE base per tile and lane reaches every
// fragment: base ^ (a constant of the fragment) + (a constant of the row block).
__device__ __forceinline__ uint32_t wa_lds_byte(const void* p) { return (uint32_t)(size_t)(__attribute__((address_space(3))) const char*)p; }
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Wint-to-pointer-cast"      // (LDS pointers are 32 bits wide)
// operand from rows: element (row0 + (lane & 31), 16 s + 8 (lane >> 5) + j); `base` of wa_row_base, `at` = the bytes of row0 (a multiple of 16 rows)
template <int DP> __device__ __forceinline__ uint32_t wa_row_base()
{
    const int lane = threadIdx.x & 63;
    return WaTile<DP>::at(lane & 31, lane >> 5);
}
template <typename T> __device__ __forceinline__ typename WaMma<T>::v8 wa_frag_row(uint32_t base, int s, uint32_t at)
{
    typedef typename WaMma<T>::v8 __attribute__((address_space(3)))* lds_p;
    return *(lds_p)((base ^ (uint32_t)(s << 5)) + at);
}
// operand from columns: element (k, 32 dt + (lane & 31)), k in the order of an accumulator used as operand: slot (h, j) <-> k = row0 + 8 (j >> 2) + 4 h + (j & 3)
template <int DP> __device__ __forceinline__ uint32_t wa_col_base()
{
    const int lane = threadIdx.x & 63, g = lane >> 4, q = (lane >> 2) & 3, p = lane & 3;
    return WaTile<DP>::at(4 * (g >> 1) + q, 2 * (g & 1) + (p >> 1)) + 8 * (p & 1);
}
template <typename T, int DP> __device__ __forceinline__ typename WaMma<T>::v8 wa_frag_col(uint32_t base, int dt, uint32_t at)
{
    typedef wa_s16x4 __attribute__((address_space(3)))* lds_p;
    const wa_s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_p)((base ^ (uint32_t)(dt << 6)) + at));
    // eight rows on, the swizzle has turned chunk bit 1
    const wa_s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_p)((base ^ (uint32_t)(dt << 6) ^ 32u) + at + 8 * WaTile<DP>::PITCH));
    const wa_s16x8 v = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    return __builtin_bit_cast(typename WaMma<T>::v8, v);
}
#pragma clang diagnostic pop
// keeps the optimiser from holding every XORed address of a loop in a register of its own
__device__ __forceinline__ uint32_t wa_opaque(uint32_t v) { asm volatile("" : "+v"(v)); return v; }

// ------------------------------------------------------------------ what a sample's rows see
struct WaSeen { int n, off; };                                              // keys in use; position of query 0
__device__ __forceinline__ WaSeen wa_seen(const WaArgs& w, int b)
{
    WaSeen s;
    s.n = w.a.Lkv;
    if (w.a.lens) s.n = (int)max(0L, min(w.a.lens64 ? (long)((const long long*)w.a.lens)[b] : (long)((const int*)w.a.lens)[b], (long)w.a.Lkv));
    s.off = s.n - w.a.Lq;
    return s;
}
// The keys a block of rows at positions pmin .. pmax can see, as one list: the `first` first ones, then lo .. hi.  Entry x is key x, or
// x + shift from `first` on; a stage is a run of entries, so the first tokens share a stage with the window instead of having their own.
struct WaSpan { int first, shift, total; };
__device__ __forceinline__ WaSpan wa_span(const WaArgs& w, const WaSeen& s, int pmin, int pmax)
{
    WaSpan k;
    const int hi = max(0, min(pmax + w.a.right + 1, s.n)), lo = min(max(0, pmin - w.a.left), hi);
    k.first = min(w.a.sinks, lo);
    k.shift = lo - k.first;
    k.total = hi - k.shift;
    return k;
}

// Order of the workgroups; consecutive ones go round the 8 XCDs, each with an L2 of its own.  The (sample, key head) pairs run fastest, so each
// XCD keeps few of them, and within a pair the longest walks start first.  With fewer than 8 pairs XCDs share one, and where all walks are
// about as long (w.runs) each then takes a run of consecutive tiles, whose rows share their keys.  Measured, runs against pairs first: 4 pairs of
// 256 tiles dQ 237 / 283 us, 1024 tiles forward 1362 / 1387 us; 96 pairs of 9 tiles forward 41.6 / 33.5 us, dQ 46 / 38 us.
__device__ __forceinline__ void wa_item(const WaArgs& w, int& bh, int& tile, int& split)
{
    const int pairs = w.a.B * w.a.Hk;
    int id = blockIdx.x;
    if (w.runs) {
        const int per = gridDim.x / 8, cut = per * 8;
        if (id < cut) id = (id & 7) * per + (id >> 3);
        bh = id / w.tiles; tile = id % w.tiles; split = 0;
        return;
    }
    bh = id % pairs; split = id / pairs % w.splits; tile = w.tiles - 1 - id / pairs / w.splits;
}

// Stages travel memory -> LDS without registers (global_load_lds, 16 bytes a lane): a wave instruction fills 1 KB of the tile, lane i its 16
// bytes at + 16 i, so the swizzle is made on the global side: the lane fetches the chunk whose place it fills.  The rows a lane serves in
// its instructions are STEP apart, a multiple of the swizzle's period, so row0 and the chunk are the same for all of them.
// The instruction is issued from inline asm (through the builtin the compiler waits for it in front of every LDS read); a stage is awaited by
// wa_stage_wait in front of the barrier that opens it.  Rows and chunks that do not exist are replaced by ones that do (finite where the
// product takes a zero weight); keys that are padding come from wa_zeros.
__device__ const uint4 wa_zeros[WA_THREADS / 64] = {};
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"          // (m0 is reserved: it is what the instruction takes its LDS address from)
__device__ __forceinline__ void wa_dma(const void* base, uint32_t off, uint32_t lds_byte)
{
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" :: "s"(lds_byte), "v"(off), "s"(base) : "memory", "m0");
}
__device__ __forceinline__ void wa_dma4(const void* base, uint32_t off, uint32_t lds_byte)      // 4 bytes a lane
{
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2" :: "s"(lds_byte), "v"(off), "s"(base) : "memory", "m0");
}
__device__ __forceinline__ void wa_dma_any(const void* p, uint32_t lds_byte)
{
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" :: "s"(lds_byte), "v"(p) : "memory", "m0");
}
#pragma clang diagnostic pop
// waits for this wave's loads but the N youngest (they retire in order)
template <int N> __device__ __forceinline__ void wa_stage_wait() { asm volatile("s_waitcnt vmcnt(%0)" :: "n"(N) : "memory"); }
template <int DP, int ROWS, int NW = 4> struct WaStage {
    static constexpr int PITCH = WaTile<DP>::PITCH, ALL = NW * 1024, PER = ROWS * PITCH / ALL, STEP = ALL / PITCH;      // wave instructions of one tile per wave
    static_assert(ROWS * PITCH % ALL == 0 && STEP % 16 == 0, "a stage is whole instructions of all waves, whole periods of the swizzle apart");
    int row0;                   // this lane's row in the wave's first instruction
    uint32_t col;               // its chunk, in bytes
    uint32_t wave_byte;
    __device__ __forceinline__ WaStage(int dh)
    {
        const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), at = wave * 1024 + (threadIdx.x & 63) * 16;
        row0 = at / PITCH;
        const int c = (at % PITCH / 16) ^ WaTile<DP>::swz(row0);
        col = 8 * c < dh ? 16 * c : 0;
        wave_byte = wave * 1024;
    }
    // rows 0 .. last (the others repeat the last one) of a matrix with `stride` bytes from row to row
    __device__ __forceinline__ void rows(const char* base, uint32_t stride, int last, uint32_t tile) const
    {
#pragma unroll
        for (int i = 0; i < PER; ++i) wa_dma(base, (uint32_t)min(row0 + i * STEP, last) * stride + col, tile + wave_byte + i * ALL);
    }
    // rows key(0) .. key(last) of it, with zeros where pad[key] is set (pad may be null)
    template <typename F> __device__ __forceinline__ void rows_of(const char* base, long stride, int last, F key, const uint8_t* pad, uint32_t tile) const
    {
        const char* p[PER];
#pragma unroll
        for (int i = 0; i < PER; ++i) {                         // all padding bytes are on their way before the first is looked at
            const int k = key(min(row0 + i * STEP, last));
            p[i] = base + k * stride + col;
            if (pad) p[i] = pad[k] ? (const char*)wa_zeros : p[i];
        }
#pragma unroll
        for (int i = 0; i < PER; ++i) wa_dma_any(p[i], tile + wave_byte + i * ALL);
    }
};

// Does a wave with rows at positions wmin .. wmax see nothing / all of the n list entries from x on?  (A block across the list's seam: neither.)
__device__ __forceinline__ bool wa_none(const WaArgs& w, const WaSpan& s, int x, int n, int wmin, int wmax)
{
    if (x >= s.total) return true;
    if (x < s.first && x + n > s.first) return false;
    const int k = x < s.first ? x : x + s.shift;
    return k > wmax + w.a.right || (k + n <= wmin - w.a.left && k >= w.a.sinks);
}
__device__ __forceinline__ bool wa_all(const WaArgs& w, const WaSpan& s, int x, int n, int wmin, int wmax)
{
    if (x + n > s.total || (x < s.first && x + n > s.first)) return false;
    const int k = x < s.first ? x : x + s.shift;
    return k + n - 1 <= wmin + w.a.right && (k >= wmax - w.a.left || k + n <= w.a.sinks);
}

// Which of the 32 list entries from x on the lane's row sees, as bits: key in low .. top, or a first token up to top
__device__ __forceinline__ uint32_t wa_below(int n) { return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1u; }      // the n lowest bits
__device__ __forceinline__ uint32_t wa_window(int k, int top, int low, int sinks) { return wa_below(top + 1 - k) & (~wa_below(low - k) | wa_below(sinks - k)); }
__device__ __forceinline__ uint32_t wa_visible(const WaSpan& s, int x, int top, int low, int sinks)
{
    uint32_t m = wa_window(x + s.shift, top, low, sinks);
    if (x < s.first) {                                           // (uniform) in front of the list's seam: entry = key
        const uint32_t f = wa_below(s.first - x);
        m = (m & ~f) | (wa_window(x, top, low, sinks) & f);
    }
    return m & wa_below(s.total - x);
}
// hidden scores -> -inf (accumulator order: entry (r & 3) + 8 (r >> 2) + 4 hl)
__device__ __forceinline__ void wa_hide(wa_f32x16& s, uint32_t visible, int hl)
{
    visible >>= 4 * hl;
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = visible & (1u << ((r & 3) + 8 * (r >> 2))) ? s[r] : -INFINITY;
}

// ------------------------------------------------------------------ forward
// Workgroup = 4 waves = RB groups of RW blocks of 32 rows x KS parts of a stage's keys (SUBK each); K and V are double-buffered in LDS, the loads of
// the next stage are in flight during the products of this one.  At RW = 1 every fragment of K and V that comes from LDS serves one matrix
// instruction, which keeps the LDS as busy as the matrix cores; at RW = 2 it serves two.  The priority is up around the products, so that the two
// waves of a SIMD fall out of step and one's softmax runs beside the other's products (4 - 5 %).  splits > 1: the stages of a row tile are divided over workgroups, whose
// (maximum, sum, unnormalised output) wa_join_kernel joins.
template <typename T, int DP, int RB, int RW, int KS, int SUBK>
__global__ void __launch_bounds__(WA_THREADS, 2) wa_fwd_kernel(WaArgs w)
{
    using Tile = WaTile<DP>;
    constexpr int STAGE = SUBK * KS, KST = DP / 16, DT = DP / 32, NB = SUBK / 32, KG = RW == 1 ? NB : 1, BUF = STAGE * Tile::PITCH, WR = 32 * RW;
    constexpr bool DEEP = KS == 4;                                           // few rows: the loads are what takes time
    extern __shared__ __attribute__((aligned(1024))) char lds[];               // [2][K, V][STAGE rows], pads
    const VpfWindowAttn& a = w.a;
    uint32_t* const pads = reinterpret_cast<uint32_t*>(lds + 4 * BUF);     // [2][STAGE / 32]: a bit for every key that is not padding
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), hl = lane >> 5, rb = wave % RB, ks = wave / RB;
    int bh, tile, split;
    wa_item(w, bh, tile, split);
    const int b = bh / a.Hk, hk = bh % a.Hk;
    const WaSeen seen = wa_seen(w, b);
    const int r0 = tile * WR * RB, rend = min(r0 + WR * RB, w.rows);
    const WaSpan span = wa_span(w, seen, seen.off + wa_query(w, r0), seen.off + wa_query(w, rend - 1));
    const int stages = (span.total + STAGE - 1) / STAGE, t0 = (int)((long)stages * split / w.splits), t1 = (int)((long)stages * (split + 1) / w.splits);

    const char* kp = (const char*)((const T*)a.k + b * a.k_sb + hk * a.k_sh);
    const char* vp = (const char*)((const T*)a.v + b * a.v_sb + hk * a.v_sh);
    const uint8_t* pad = a.pad ? (const uint8_t*)a.pad + (size_t)b * a.Lkv : nullptr;

    const WaStage<DP, STAGE> stage(a.head_dim);
    const uint32_t tiles_at = wa_lds_byte(lds), row_base = wa_row_base<DP>(), col_base = wa_col_base<DP>();
    auto load = [&](int t) {
        const int x0 = t * STAGE, last = min(STAGE, span.total - x0) - 1;
        const uint32_t at = tiles_at + (t & 1) * 2 * BUF;
        const long kst = a.k_sl * (long)sizeof(T), vst = a.v_sl * (long)sizeof(T);
        if (pad || x0 < span.first) {
            auto key = [&](int r) { return (long)(x0 + r < span.first ? x0 + r : x0 + r + span.shift); };
            if (pad) {
                const uint64_t kept = __ballot((int)threadIdx.x <= last && !pad[key(min((int)threadIdx.x, last))]);      // threads 64 i ..: entries 64 i ..
                if (lane < 2 && wave * 2 + lane < STAGE / 32) pads[(t & 1) * (STAGE / 32) + wave * 2 + lane] = (uint32_t)(kept >> (32 * lane));
            }
            // a key that nobody here sees must not reach the product with V: 0 * NaN is NaN
            stage.rows_of(kp, kst, last, key, nullptr, at);
            stage.rows_of(vp, vst, last, key, pad, at + BUF);
        } else {
            stage.rows(kp + (x0 + span.shift) * kst, (uint32_t)kst, last, at);
            stage.rows(vp + (x0 + span.shift) * vst, (uint32_t)vst, last, at + BUF);
        }
    };
    if (t0 < t1) load(t0);
    if (DEEP && t0 + 1 < t1) load(t0 + 1);
    // this lane's rows: one of each of the wave's RW blocks
    const int wrow = r0 + rb * WR;
    const bool live = wrow < w.rows;
    const int wmin = seen.off + wa_query(w, min(wrow, w.rows - 1)), wmax = seen.off + wa_query(w, min(wrow + WR - 1, w.rows - 1));
    auto row_of = [&](int j) { return wrow + 32 * j + (lane & 31); };
    int pos[RW];
    typename WaMma<T>::v8 qf[RW][KST];
#pragma unroll
    for (int j = 0; j < RW; ++j) {
        const int rq = min(row_of(j), w.rows - 1), qi = wa_query(w, rq);
        pos[j] = seen.off + qi;
        const T* qp = (const T*)a.q + b * a.q_sb + qi * a.q_sl + (hk * w.g + (rq - qi * w.g)) * a.q_sh;
#pragma unroll
        for (int s = 0; s < KST; ++s) {
            const int d = 16 * s + 8 * hl;
            uint4 u = make_uint4(0, 0, 0, 0);
            if (d < a.head_dim) u = *reinterpret_cast<const uint4*>(qp + d);
            qf[j][s] = __builtin_bit_cast(typename WaMma<T>::v8, u);
        }
    }
    wa_f32x16 o[RW][DT];
    float m[RW], l[RW];
#pragma unroll
    for (int j = 0; j < RW; ++j) {
        m[j] = -INFINITY; l[j] = 0.f;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) o[j][dt] = wa_zero16();
    }

    if (!DEEP) { wa_stage_wait<0>(); __syncthreads(); }
    for (int t = t0; t < t1; ++t) {
        if (DEEP) {                                                          // two stages in flight; this one's loads are the older ones
            if (t + 1 < t1) wa_stage_wait<2 * WaStage<DP, STAGE>::PER>();
            else wa_stage_wait<0>();
            __syncthreads();
        } else if (t + 1 < t1) load(t + 1);
        const int x0 = t * STAGE + ks * SUBK;
        const uint32_t sk = tiles_at + (t & 1) * 2 * BUF + ks * SUBK * Tile::PITCH, krow = wa_opaque(row_base + sk), vcol = wa_opaque(col_base + sk + BUF);
#pragma unroll
        for (int k0 = 0; k0 < NB; k0 += KG) {
            const int xg = x0 + 32 * k0;
            if (!live || wa_none(w, span, xg, 32 * KG, wmin, wmax)) continue;
            wa_f32x16 s[RW][KG];
            __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int kb = 0; kb < KG; ++kb) {
#pragma unroll
                for (int j = 0; j < RW; ++j) s[j][kb] = wa_zero16();
#pragma unroll
                for (int i = 0; i < KST; ++i) {
                    const typename WaMma<T>::v8 kf = wa_frag_row<T>(krow, i, 32 * (k0 + kb) * Tile::PITCH);
#pragma unroll
                    for (int j = 0; j < RW; ++j) s[j][kb] = WaMma<T>::mma(kf, qf[j][i], s[j][kb]);
                }
            }
            __builtin_amdgcn_s_setprio(0);
            if (pad || !wa_all(w, span, xg, 32 * KG, wmin, wmax)) {
#pragma unroll
                for (int j = 0; j < RW; ++j)
#pragma unroll
                    for (int kb = 0; kb < KG; ++kb) {
                        uint32_t see = wa_visible(span, xg + 32 * kb, pos[j] + a.right, pos[j] - a.left, a.sinks);
                        if (pad) see &= pads[(t & 1) * (STAGE / 32) + ks * NB + k0 + kb];
                        wa_hide(s[j][kb], see, hl);
                    }
            }
            float mx[RW];
            bool grown = false;
#pragma unroll
            for (int j = 0; j < RW; ++j) {
                mx[j] = s[j][0][0];
#pragma unroll
                for (int kb = 0; kb < KG; ++kb)
#pragma unroll
                    for (int r = 0; r < 16; ++r) mx[j] = fmaxf(mx[j], s[j][kb][r]);
                mx[j] = wa_half_max(mx[j]) * w.c;
                grown = grown || mx[j] > m[j] + WaMma<T>::GROW;
            }
            // The running maximum only has to keep exp2 in range: it moves when a row has outgrown it by 2^GROW
            if (__any(grown)) {
#pragma unroll
                for (int j = 0; j < RW; ++j) {
                    const float mn = fmaxf(m[j], mx[j]), f = m[j] == -INFINITY ? 0.f : wa_exp2(m[j] - mn);
                    m[j] = mn;
                    l[j] *= f;
#pragma unroll
                    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                        for (int r = 0; r < 16; ++r) o[j][dt][r] *= f;
                }
            }
            __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int kb = 0; kb < KG; ++kb) {
                typename WaMma<T>::v8 pf[RW][2];
#pragma unroll
                for (int j = 0; j < RW; ++j) {
                    const float base = m[j] == -INFINITY ? 0.f : m[j] - WaMma<T>::LIFT;      // a row that has seen nothing yet: every weight is exp2(-inf)
                    float p[16];
#pragma unroll
                    for (int r = 0; r < 16; ++r) { p[r] = wa_exp2(fmaf(s[j][kb][r], w.c, -base)); l[j] += p[r]; }
                    pf[j][0] = wa_pack8<T>(p); pf[j][1] = wa_pack8<T>(p + 8);
                }
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int dt = 0; dt < DT; ++dt) {
                        const typename WaMma<T>::v8 vf = wa_frag_col<T, DP>(vcol, dt, (32 * (k0 + kb) + 16 * i) * Tile::PITCH);
#pragma unroll
                        for (int j = 0; j < RW; ++j) o[j][dt] = WaMma<T>::mma(vf, pf[j][i], o[j][dt]);
                    }
            }
            __builtin_amdgcn_s_setprio(0);
        }
        if (!DEEP) { wa_stage_wait<0>(); __syncthreads(); }
        else if (t + 2 < t1) { __syncthreads(); load(t + 2); }
    }
    if (DEEP) __syncthreads();
    static_assert(KS == 1 || RW == 1, "parts of the keys are joined for one row block");
    if constexpr (KS > 1) {                                                            // join the key parts through LDS (the stages are done with)
        float* slots = reinterpret_cast<float*>(lds);
        constexpr int SLOT = (DT * 16 + 2) * 64;
        static_assert((KS / 2) * RB * SLOT * 4 <= 4 * BUF, "the partial results fit the stage buffers");
#pragma unroll
        for (int step = KS / 2; step >= 1; step >>= 1) {
            if (ks >= step && ks < 2 * step) {
                float* slot = slots + ((ks - step) * RB + rb) * SLOT + lane;
#pragma unroll
                for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                    for (int r = 0; r < 16; ++r) slot[(dt * 16 + r) * 64] = o[0][dt][r];
                slot[DT * 16 * 64] = m[0]; slot[(DT * 16 + 1) * 64] = l[0];
            }
            __syncthreads();
            if (ks < step) {
                const float* slot = slots + (ks * RB + rb) * SLOT + lane;
                const float m2 = slot[DT * 16 * 64], mn = fmaxf(m[0], m2);
                const float f1 = m[0] == -INFINITY ? 0.f : wa_exp2(m[0] - mn), f2 = m2 == -INFINITY ? 0.f : wa_exp2(m2 - mn);
                l[0] = l[0] * f1 + slot[(DT * 16 + 1) * 64] * f2;
                m[0] = mn;
#pragma unroll
                for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                    for (int r = 0; r < 16; ++r) o[0][dt][r] = o[0][dt][r] * f1 + slot[(dt * 16 + r) * 64] * f2;
            }
            if (step > 1) __syncthreads();
        }
    }
    if (ks != 0) return;
#pragma unroll
    for (int jr = 0; jr < RW; ++jr) {
    const int row = row_of(jr);
    if (row >= w.rows) return;
    const int qi = wa_query(w, row);
    const float lr = wa_half_sum(l[jr]), mr = m[jr];
    if (w.splits > 1) {
        const size_t at = ((size_t)split * a.B * a.Hk + bh) * w.rows + row;
        float* part = a.ws + at * DP;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                *reinterpret_cast<float4*>(part + 32 * dt + 8 * j + 4 * hl) = make_float4(o[jr][dt][4 * j], o[jr][dt][4 * j + 1], o[jr][dt][4 * j + 2], o[jr][dt][4 * j + 3]);
        if (hl == 0) reinterpret_cast<float2*>(a.ws + (size_t)w.splits * a.B * a.Hk * w.rows * DP)[at] = make_float2(mr, lr);
        continue;
    }
    const float inv = lr == 0.f ? 0.f : 1.f / lr;
    T* op = (T*)a.out + b * a.o_sb + qi * a.o_sl + (hk * w.g + (row - qi * w.g)) * a.o_sh;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int d = 32 * dt + 8 * j + 4 * hl;
            const float v[4] = {o[jr][dt][4 * j] * inv, o[jr][dt][4 * j + 1] * inv, o[jr][dt][4 * j + 2] * inv, o[jr][dt][4 * j + 3] * inv};
            if (d < a.head_dim) {
                vpf_store<T, 4>(op + d, v);
                if (a.out_lo) {
                    const float e[4] = {v[0] - (float)(T)v[0], v[1] - (float)(T)v[1], v[2] - (float)(T)v[2], v[3] - (float)(T)v[3]};
                    vpf_store<T, 4>((T*)a.out_lo + ((size_t)bh * w.rows + row) * a.head_dim + d, e);
                }
            }
        }
    if (a.lse && hl == 0) a.lse[(size_t)bh * w.rows + row] = lr == 0.f ? INFINITY : (mr - WaMma<T>::LIFT) + log2f(lr);
    }
}

// parts of the keys -> output: one wave per row.  Lane i holds maximum and sum of part i (splits <= 64); the channels' loads of 4 parts are in
// flight together.
template <typename T, int DP>
__global__ void __launch_bounds__(WA_THREADS) wa_join_kernel(WaArgs w)
{
    const VpfWindowAttn& a = w.a;
    const size_t all = (size_t)a.B * a.Hk * w.rows, at = (size_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    if (at >= all) return;
    const float2* ml = reinterpret_cast<const float2*>(a.ws + (size_t)w.splits * all * DP);
    const float2 mine = lane < w.splits ? ml[lane * all + at] : make_float2(-INFINITY, 0.f);
    const float m = wave_max(mine.x), f = mine.x == -INFINITY ? 0.f : wa_exp2(mine.x - m), l = wave_sum(mine.y * f);
    constexpr int N = (DP + 63) / 64;
    float o[N];
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] = 0.f;
#pragma unroll 4
    for (int s = 0; s < w.splits; ++s) {
        const float fs = __shfl(f, s);
#pragma unroll
        for (int i = 0; i < N; ++i) if (lane + 64 * i < DP) o[i] += a.ws[(s * all + at) * DP + lane + 64 * i] * fs;
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const int bh = (int)(at / w.rows), row = (int)(at % w.rows), qi = wa_query(w, row);
    T* op = (T*)a.out + bh / a.Hk * a.o_sb + qi * a.o_sl + (bh % a.Hk * w.g + (row - qi * w.g)) * a.o_sh;
#pragma unroll
    for (int i = 0; i < N; ++i) if (lane + 64 * i < a.head_dim) {
        const T v = (T)(o[i] * inv);
        op[lane + 64 * i] = v;
        if (a.out_lo) ((T*)a.out_lo)[at * a.head_dim + lane + 64 * i] = (T)(o[i] * inv - (float)v);
    }
    if (a.lse && lane == 0) a.lse[at] = l == 0.f ? INFINITY : (m - WaMma<T>::LIFT) + log2f(l);
}

// ------------------------------------------------------------------ backward: queries
// dS = P (dP - delta), dP = dO V^T, delta = sum of P dP = rowsum(dO . O);  dQ = scale dS K.  The walk over the keys is the forward kernel's.  dS is
// rounded to the tensors' type for its product, as P is.
// fp16 does not hold dS as it is: with gradients of 10^-4 over 2048 keys most of it lies below 2^-24, and |dP - delta| can pass 65504 where dq does
// not.  A row here (a key in the kernel of the keys) carries a power of two for its dS, which starts at 2^WA_UP and falls whenever the row's largest
// |dS| would pass 2^15 of it, to bring that to 2^10 .. 2^11; its sums fall with it, so nothing is rounded by it.  What then lies below fp16's
// smallest numbers is 2^-35 of the row's largest.  It costs (fp16, us, dQ and dK / dV kernel without / with): 16 x 1025, 6 heads of 64, window 257
// 39.8 / 41.1 and 40.7 / 43.3; 8192 queries, 16 + 4 heads of 128, window 2048 264 / 270 and 312 / 343.
#define WA_UP 64
#define WA_TOP 32768.f
__device__ __forceinline__ int wa_fall(float largest) { return largest > WA_TOP ? min(0, 11 - __builtin_amdgcn_frexp_expf(largest)) : 0; }
__device__ __forceinline__ float wa_largest(const float* v)                  // |v| of 16 values of the lane and of its partner
{
    float m = fabsf(v[0]);
#pragma unroll
    for (int r = 1; r < 16; ++r) m = fmaxf(m, fabsf(v[r]));
    return wa_half_max(m);
}
template <int N> __device__ __forceinline__ void wa_scale(wa_f32x16* acc, int e)
{
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[i][r] = __builtin_ldexpf(acc[i][r], e);
}
// delta comes in three qualities.  rowsum(dO . O) is there before the walk, with O as forward had it before rounding (out + out_lo; with the
// rounded O the error of dq against 64 bits was 1.6 instead of 1.4 times the output's own rounding); what is left in it is the rounding of
// forward's weights, 1 / sqrt(keys) of dS's own rounding.  Where rows see few keys (WA_FEW) the walk is therefore made twice, first for
// the sum of P dP in fp32.  That sum is also what a single walk leaves behind for the kernel of the keys.
#define WA_FEW 64
template <typename T, int DP, int RB, int KS>
__global__ void __launch_bounds__(WA_THREADS, 2) wa_dq_kernel(WaArgs w)
{
    using Tile = WaTile<DP>;
    constexpr int SUBK = KS == 1 ? 64 : 32, STAGE = SUBK * KS, KST = DP / 16, DT = DP / 32, NB = SUBK / 32, BUF = STAGE * Tile::PITCH;
    constexpr bool NARROW = WaMma<T>::NARROW;
    extern __shared__ __attribute__((aligned(1024))) char lds[];
    const VpfWindowAttn& a = w.a;
    uint32_t* const pads = reinterpret_cast<uint32_t*>(lds + 4 * BUF);     // [2][STAGE / 32]: a bit for every key that is not padding
    float* const sums = reinterpret_cast<float*>(pads + 2 * (STAGE / 32));  // [KS][RB][32]: the key parts' sums of P dP
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), hl = lane >> 5, rb = wave % RB, ks = wave / RB;
    int bh, tile, split;
    wa_item(w, bh, tile, split);
    const int b = bh / a.Hk, hk = bh % a.Hk;
    const WaSeen seen = wa_seen(w, b);
    const int r0 = tile * 32 * RB, rend = min(r0 + 32 * RB, w.rows);
    const WaSpan span = wa_span(w, seen, seen.off + wa_query(w, r0), seen.off + wa_query(w, rend - 1));
    const int stages = (span.total + STAGE - 1) / STAGE;
    const int row = r0 + rb * 32 + (lane & 31), rq = min(row, w.rows - 1), qi = wa_query(w, rq), head = hk * w.g + (rq - qi * w.g);
    const int pos = seen.off + qi, wlast = min(r0 + rb * 32 + 31, w.rows - 1);
    const bool live = r0 + rb * 32 < w.rows;
    const int wmin = seen.off + wa_query(w, min(r0 + rb * 32, w.rows - 1)), wmax = seen.off + wa_query(w, wlast);
    typename WaMma<T>::v8 qf[KST], gf[KST];
    float delta = 0.f;
    {
        const T* qp = (const T*)a.q + b * a.q_sb + qi * a.q_sl + head * a.q_sh;
        const T* gp = (const T*)a.dout + b * a.do_sb + qi * a.do_sl + head * a.do_sh;
        const T* op = (const T*)a.out + b * a.o_sb + qi * a.o_sl + head * a.o_sh;
        const T* lp = (const T*)a.out_lo + ((size_t)bh * w.rows + rq) * a.head_dim;
#pragma unroll
        for (int s = 0; s < KST; ++s) {
            const int d = 16 * s + 8 * hl;
            uint4 u = make_uint4(0, 0, 0, 0), v = u, x = u, y = u;
            if (d < a.head_dim) {
                u = *reinterpret_cast<const uint4*>(qp + d); v = *reinterpret_cast<const uint4*>(gp + d);
                x = *reinterpret_cast<const uint4*>(op + d); y = *reinterpret_cast<const uint4*>(lp + d);
            }
            qf[s] = __builtin_bit_cast(typename WaMma<T>::v8, u);
            gf[s] = __builtin_bit_cast(typename WaMma<T>::v8, v);
            const typename WaMma<T>::v8 of = __builtin_bit_cast(typename WaMma<T>::v8, x), ol = __builtin_bit_cast(typename WaMma<T>::v8, y);
#pragma unroll
            for (int i = 0; i < 8; ++i) delta += (float)gf[s][i] * ((float)of[i] + (float)ol[i]);
        }
        delta = wa_half_sum(delta);
    }
    const float lse = a.lse[(size_t)bh * w.rows + rq];
    if (lse == INFINITY) delta = 0.f;                                        // a row that sees nothing: whatever its gradient holds
    const char* kp = (const char*)((const T*)a.k + b * a.k_sb + hk * a.k_sh);
    const char* vp = (const char*)((const T*)a.v + b * a.v_sb + hk * a.v_sh);
    const uint8_t* pad = a.pad ? (const uint8_t*)a.pad + (size_t)b * a.Lkv : nullptr;
    wa_f32x16 dq[DT];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) dq[dt] = wa_zero16();

    const WaStage<DP, STAGE> stage(a.head_dim);
    const uint32_t tiles_at = wa_lds_byte(lds), row_base = wa_row_base<DP>(), col_base = wa_col_base<DP>();
    auto load = [&](int t, int buf) {
        const int x0 = t * STAGE, last = min(STAGE, span.total - x0) - 1;
        const uint32_t at = tiles_at + buf * 2 * BUF;
        const long kst = a.k_sl * (long)sizeof(T), vst = a.v_sl * (long)sizeof(T);
        if (pad || x0 < span.first) {
            auto key = [&](int r) { return (long)(x0 + r < span.first ? x0 + r : x0 + r + span.shift); };
            if (pad) {
                const uint64_t kept = __ballot((int)threadIdx.x <= last && !pad[key(min((int)threadIdx.x, last))]);      // threads 64 i ..: entries 64 i ..
                if (lane < 2 && wave * 2 + lane < STAGE / 32) pads[buf * (STAGE / 32) + wave * 2 + lane] = (uint32_t)(kept >> (32 * lane));
            }
            // a key that nobody here sees must not reach the product with K: 0 * NaN is NaN
            stage.rows_of(kp, kst, last, key, pad, at);
            stage.rows_of(vp, vst, last, key, nullptr, at + BUF);
        } else {
            stage.rows(kp + (x0 + span.shift) * kst, (uint32_t)kst, last, at);
            stage.rows(vp + (x0 + span.shift) * vst, (uint32_t)vst, last, at + BUF);
        }
    };
    // the fewest keys a row here can see (padding aside): at one of the ends of the tile's positions
    auto keys_of = [&](int p) { const int lo = max(0, p - a.left); return min(p + a.right, seen.n - 1) + 1 - lo + min(a.sinks, lo); };
    const bool twice = min(keys_of(seen.off + wa_query(w, r0)), keys_of(seen.off + wa_query(w, rend - 1))) <= WA_FEW;
    const int steps = twice ? 2 * stages : stages;
    float pdp = 0.f, lsu = NARROW && !twice ? lse - WA_UP : lse;             // (exp2(.. - lsu): the weight times the row's power of two)
    int up = WA_UP;
    auto joined = [&](float v) {                                             // over the lane pair and the key parts
        v = wa_half_sum(v);
        if constexpr (KS > 1) {
            if (hl == 0) sums[(ks * RB + rb) * 32 + lane] = v;
            __syncthreads();
            v = 0.f;
#pragma unroll
            for (int i = 0; i < KS; ++i) v += sums[(i * RB + rb) * 32 + (lane & 31)];
        }
        return v;
    };
    if (stages > 0) { load(0, 0); wa_stage_wait<0>(); }
    __syncthreads();
    for (int step = 0; step < steps; ++step) {
        const int t = step < stages ? step : step - stages, next = t + 1 < stages ? t + 1 : 0;
        const bool first = twice && step < stages;                           // the walk for delta alone
        if (step + 1 < steps) load(next, (step + 1) & 1);
        const int x0 = t * STAGE + ks * SUBK;
        const uint32_t sk = tiles_at + (step & 1) * 2 * BUF + ks * SUBK * Tile::PITCH, krow = wa_opaque(row_base + sk), kcol = wa_opaque(col_base + sk);
#pragma unroll
        for (int kb = 0; kb < NB; ++kb) {
            const int xb = x0 + 32 * kb;
            if (!live || wa_none(w, span, xb, 32, wmin, wmax)) continue;
            __builtin_amdgcn_s_setprio(1);
            wa_f32x16 s = wa_zero16(), dp = wa_zero16();
#pragma unroll
            for (int i = 0; i < KST; ++i) {
                s = WaMma<T>::mma(wa_frag_row<T>(krow, i, 32 * kb * Tile::PITCH), qf[i], s);
                dp = WaMma<T>::mma(wa_frag_row<T>(krow, i, 32 * kb * Tile::PITCH + BUF), gf[i], dp);
            }
            __builtin_amdgcn_s_setprio(0);
            const bool all = !pad && wa_all(w, span, xb, 32, wmin, wmax);
            if (!all) {
                uint32_t see = wa_visible(span, xb, pos + a.right, pos - a.left, a.sinks);
                if (pad) see &= pads[(step & 1) * (STAGE / 32) + ks * NB + kb];
                wa_hide(s, see, hl);
            }
            float ds[16];
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const float p = wa_exp2(fmaf(s[r], w.c, -lsu));
                float x = p * dp[r];
                if (!all) x = s[r] == -INFINITY ? 0.f : x;                   // what a hidden key holds stays out
                pdp += x;
                ds[r] = fmaf(-p, delta, x);
            }
            if (first) continue;
            if constexpr (NARROW) {
                const float largest = wa_largest(ds);
                if (__any(largest > WA_TOP)) {
                    const int e = wa_fall(largest);
                    up += e; lsu -= (float)e;
                    pdp = __builtin_ldexpf(pdp, e);
#pragma unroll
                    for (int r = 0; r < 16; ++r) ds[r] = __builtin_ldexpf(ds[r], e);
                    wa_scale<DT>(dq, e);
                }
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const typename WaMma<T>::v8 df = wa_pack8<T>(ds + 8 * i);
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) dq[dt] = WaMma<T>::mma(wa_frag_col<T, DP>(kcol, dt, (32 * kb + 16 * i) * Tile::PITCH), df, dq[dt]);
            }
        }
        if (first && step + 1 == stages) { delta = joined(pdp); pdp = 0.f; if (NARROW) lsu = lse - WA_UP; }
        wa_stage_wait<0>();
        __syncthreads();
    }
    if (!twice) delta = joined(NARROW ? __builtin_ldexpf(pdp, -up) : pdp);
    if constexpr (NARROW) wa_scale<DT>(dq, -up);
    if (ks == 0 && hl == 0 && row < w.rows) {
        a.ws[(size_t)bh * w.rows + row] = delta;
        if (NARROW) a.ws[wa_delta_floats(w) + (size_t)bh * w.rows + row] = lse - WA_LIFT;
    }
    if (KS > 1) {
        float* slots = reinterpret_cast<float*>(lds);
        constexpr int SLOT = DT * 16 * 64;
        static_assert((KS / 2) * RB * SLOT * 4 <= 4 * BUF, "the partial results fit the stage buffers");
#pragma unroll
        for (int step = KS / 2; step >= 1; step >>= 1) {
            if (ks >= step && ks < 2 * step) {
                float* slot = slots + ((ks - step) * RB + rb) * SLOT + lane;
#pragma unroll
                for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                    for (int r = 0; r < 16; ++r) slot[(dt * 16 + r) * 64] = dq[dt][r];
            }
            __syncthreads();
            if (ks < step) {
                const float* slot = slots + (ks * RB + rb) * SLOT + lane;
#pragma unroll
                for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                    for (int r = 0; r < 16; ++r) dq[dt][r] += slot[(dt * 16 + r) * 64];
            }
            if (step > 1) __syncthreads();
        }
    }
    if (ks != 0 || row >= w.rows) return;
    T* op = (T*)a.dq + b * a.dq_sb + qi * a.dq_sl + head * a.dq_sh;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int d = 32 * dt + 8 * j + 4 * hl;
            const float v[4] = {dq[dt][4 * j] * a.scale, dq[dt][4 * j + 1] * a.scale, dq[dt][4 * j + 2] * a.scale, dq[dt][4 * j + 3] * a.scale};
            if (d < a.head_dim) vpf_store<T, 4>(op + d, v);
        }
}

// ------------------------------------------------------------------ backward: keys
// dV = P^T dO, dK = scale dS^T Q, summed over the rows (queries and heads) that see the key, in one fixed order.
// Workgroup = KB blocks of 32 keys x 2 halves of a 64-row stage of Q and dO (double-buffered in LDS); K of the wave's keys stays in registers as
// operand (key on the lane), V as well up to head dimension 96 -- at 128 the two accumulators, K and the scores leave no room for it and V is
// read from LDS (a spill would be worse than slow: its reload waits behind the DMA of the next stage).
// The row blocks are walked downwards from a block that is the same for all key tiles (w.cycle), wrapping round: tiles that run at the same
// time then read the same rows of Q and dO at the same time.  Each starting at its own first row, the tiles of a long causal window had
// their rows spread over the whole sequence and every stage came from beyond the L2.
// The first tokens are seen by every row behind them: the rows beyond their window are cut into pieces of chunk_rows, one workgroup each, and
// wa_sink_join_kernel adds the pieces.
#define WA_ROWS 64
struct WaRowRange { int lo, hi; };
__device__ __forceinline__ WaRowRange wa_rows_of(const WaArgs& w, const WaSeen& s, int k0)
{
    // positions k0 - right .. k0 + key_tile - 1 + left; queries 0 .. Lq - 1 stand at off ..
    const long lo = max((long)k0 - w.a.right - s.off, 0L), hi = min((long)k0 + w.key_tile + w.a.left - s.off, (long)w.a.Lq);
    WaRowRange r;
    r.lo = (int)min(lo, (long)w.a.Lq) * w.g;
    r.hi = max((int)max(hi, 0L) * w.g, r.lo);
    return r;
}

// BLIND: the call can have rows that see nothing (wa_blind).  They may hold anything, and 0 * NaN is NaN: their Q and dO become zeros in front of
// the products.  A variant of its own, since around that look at every stage the compiler orders the products' reads worse (us without / with it:
// 8192 queries, 16 + 4 heads of 128, window 2048 306 / 340; 5 x 777, 6 + 2 heads of 80, window 128 25.0 / 26.8).
// Up to head dimension 64 three waves fit a SIMD (168 registers); two take 47 us instead of 41 at 16 x 1025, 6 heads of 64, window 257.
template <typename T, int DP, int KB, bool BLIND>
__global__ void __launch_bounds__(KB * 128, DP <= 64 ? 3 : 2) wa_dkv_kernel(WaArgs w)
{
    using Tile = WaTile<DP>;
    constexpr int ROWS = WA_ROWS, KST = DP / 16, DT = DP / 32, BUF = ROWS * Tile::PITCH, KT = KB * 32;
    constexpr bool VREG = DP <= 96, NARROW = WaMma<T>::NARROW;
    extern __shared__ __attribute__((aligned(1024))) char lds[];               // [2][Q, dO][64 rows], V [KT] (!VREG), [2][lse, delta, position][64]
    const VpfWindowAttn& a = w.a;
    float* const stats = reinterpret_cast<float*>(lds + 4 * BUF + (VREG ? 0 : KT * Tile::PITCH));
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), hl = lane >> 5, kb = wave % KB, qs = wave / KB;
    const int pairs = a.B * a.Hk, bh = blockIdx.x % pairs, it = blockIdx.x / pairs, b = bh / a.Hk, hk = bh % a.Hk, pieces = w.sink_tiles * w.chunks;
    const bool far = it < pieces;
    const int kt = far ? it / w.chunks : it - pieces, chunk = far ? it % w.chunks : 0, kt0 = kt * KT;
    const WaSeen seen = wa_seen(w, b);
    WaRowRange rr = wa_rows_of(w, seen, kt0);
    if (kt0 >= seen.n) rr.hi = rr.lo;                                        // keys behind the ones in use
    else if (kt0 < a.sinks) {
        if (w.chunks == 0) rr.hi = max(rr.hi, w.rows);
        else if (far) { const int f = rr.hi; rr.lo = max(f, chunk * w.chunk_rows); rr.hi = min(w.rows, (chunk + 1) * w.chunk_rows); }
    }

    const int key = kt0 + 32 * kb + (lane & 31), kc = min(key, a.Lkv - 1);
    const uint8_t* pad = a.pad ? (const uint8_t*)a.pad + (size_t)b * a.Lkv : nullptr;
    const bool kok = key < seen.n && !(pad && pad[kc]);
    typename WaMma<T>::v8 kf[KST], vf[VREG ? KST : 1];
    {
        const T* kp = (const T*)a.k + b * a.k_sb + kc * a.k_sl + hk * a.k_sh;
        const T* vp = (const T*)a.v + b * a.v_sb + kc * a.v_sl + hk * a.v_sh;
#pragma unroll
        for (int s = 0; s < KST; ++s) {
            const int d = 16 * s + 8 * hl;
            uint4 u = make_uint4(0, 0, 0, 0), v = u;
            if (d < a.head_dim && kok) { u = *reinterpret_cast<const uint4*>(kp + d); v = *reinterpret_cast<const uint4*>(vp + d); }
            kf[s] = __builtin_bit_cast(typename WaMma<T>::v8, u);
            if constexpr (VREG) vf[s] = __builtin_bit_cast(typename WaMma<T>::v8, v);
            else if (qs == 0) *reinterpret_cast<uint4*>(lds + 4 * BUF + Tile::at(32 * kb + (lane & 31), 2 * s + hl)) = v;
        }
    }
    wa_f32x16 dk[DT], dv[DT];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) { dk[dt] = wa_zero16(); dv[dt] = wa_zero16(); }
    float up = __builtin_ldexpf(1.f, WA_UP - WA_LIFT);                       // fp16: the key's power of two for dS (see wa_dq_kernel), beside P's
    const float* const lse_of = NARROW ? a.ws + wa_delta_floats(w) : a.lse;
    const int kmin = kt0 + 32 * kb, kmax = kmin + 31;
    const bool whole = !pad && kmax < seen.n;
    // the positions that see the lane's key are key - right .. key + left (a first token: no upper end; a hidden key: none): one unsigned comparison
    const int see_from = kok ? key - a.right : WA_FAR + WA_FAR / 2;
    const uint32_t see_n = !kok ? 0u : key < a.sinks ? 0x7fffffffu : (uint32_t)a.left + (uint32_t)a.right;

    const WaStage<DP, ROWS, 2 * KB> stage(a.head_dim);
    const uint32_t tiles_at = wa_lds_byte(lds), stats_at = wa_lds_byte(stats), row_base = wa_row_base<DP>(), col_base = wa_col_base<DP>();
    const char* qp = (const char*)((const T*)a.q + b * a.q_sb + hk * w.g * a.q_sh);
    const char* gp = (const char*)((const T*)a.dout + b * a.do_sb + hk * w.g * a.do_sh);
    // Where the query heads of a key head divide a row block, a lane's rows have the same query offset and head in every block: with 128-key tiles
    // their offsets stay in registers, 3 % of this kernel (295 -> 285 us at 8192 queries, 16 + 4 heads of 128, window 2048); the smaller tiles
    // lost 1 - 14 % to those registers.
    constexpr bool KEEP = KB == 4;
    const bool even = KEEP && ROWS % w.g == 0;
    uint32_t qoff[KEEP ? stage.PER : 1], goff[KEEP ? stage.PER : 1];
    if constexpr (KEEP) {
#pragma unroll
        for (int i = 0; i < stage.PER; ++i) {
            const int r = stage.row0 + i * stage.STEP, qi = wa_query(w, r), h = r - qi * w.g;
            qoff[i] = (uint32_t)(qi * (int)a.q_sl + h * (int)a.q_sh) * (uint32_t)sizeof(T) + stage.col;
            goff[i] = (uint32_t)(qi * (int)a.do_sl + h * (int)a.do_sh) * (uint32_t)sizeof(T) + stage.col;
        }
    }
    auto load = [&](int r0, int buf) {
        const int q0 = wa_query(w, r0), skip = r0 - q0 * w.g, last = min(ROWS, rr.hi - r0) - 1;
        const char* qb = qp + (size_t)q0 * a.q_sl * sizeof(T);
        const char* gb = gp + (size_t)q0 * a.do_sl * sizeof(T);
        const uint32_t at = tiles_at + buf * 2 * BUF;
        bool kept = false;
        if constexpr (KEEP) {
            if (even && last == ROWS - 1) {
                kept = true;
#pragma unroll
                for (int i = 0; i < stage.PER; ++i) {
                    wa_dma(qb, qoff[i], at + stage.wave_byte + i * stage.ALL);
                    wa_dma(gb, goff[i], at + BUF + stage.wave_byte + i * stage.ALL);
                }
            }
        }
        if (!kept)
#pragma unroll
        for (int i = 0; i < stage.PER; ++i) {
            const int r = skip + min(stage.row0 + i * stage.STEP, last), qi = wa_query(w, r), h = r - qi * w.g;
            wa_dma(qb, (uint32_t)(qi * (int)a.q_sl + h * (int)a.q_sh) * (uint32_t)sizeof(T) + stage.col, at + stage.wave_byte + i * stage.ALL);
            wa_dma(gb, (uint32_t)(qi * (int)a.do_sl + h * (int)a.do_sh) * (uint32_t)sizeof(T) + stage.col, at + BUF + stage.wave_byte + i * stage.ALL);
        }
        const int rc = min(lane, last);                                      // (rows behind the range: its last one again, as in the stage)
        const uint32_t stat = stats_at + buf * 3 * ROWS * 4;
        if (wave == 0) wa_dma4(lse_of + (size_t)bh * w.rows + r0, 4 * rc, stat);
        if (wave == 1) wa_dma4(a.ws + (size_t)bh * w.rows + r0, 4 * rc, stat + 4 * ROWS);
        if (wave == 2) reinterpret_cast<int*>(stats)[buf * 3 * ROWS + 2 * ROWS + lane] = seen.off + wa_query(w, r0 + rc);
    };
    // row blocks b_lo .. b_hi - 1, whole 64-row blocks of the sample's rows: what a block holds beyond the tile's range is hidden by its position
    const int b_lo = rr.lo / ROWS, b_hi = rr.hi > rr.lo ? (rr.hi + ROWS - 1) / ROWS : b_lo, steps = b_hi - b_lo;
    int top = b_hi - 1;
    { const int c = (top + 1) / w.cycle * w.cycle - 1; if (c >= b_lo) top = c; }
    auto block = [&](int t) { const int i = top - t; return (i < b_lo ? i + steps : i) * ROWS; };
    if (steps > 0) { load(block(0), 0); wa_stage_wait<0>(); }
    __syncthreads();
    for (int t = 0; t < steps; ++t) {
        if (t + 1 < steps) load(block(t + 1), (t + 1) & 1);
        if constexpr (BLIND) {                                               // (every wave finds the same rows)
            if (const uint64_t blind = __ballot(stats[(t & 1) * 3 * ROWS + (wa_opaque(threadIdx.x) & 63)] == INFINITY)) {
                for (int i = wa_opaque(threadIdx.x); i < ROWS * Tile::NC; i += KB * 128)
                    if (blind >> (i / Tile::NC) & 1) {
                        char* const at = lds + (t & 1) * 2 * BUF + i * 16;
                        *reinterpret_cast<uint4*>(at) = *reinterpret_cast<uint4*>(at + BUF) = make_uint4(0, 0, 0, 0);
                    }
                __syncthreads();
            }
        }
        const uint32_t sq = tiles_at + (t & 1) * 2 * BUF + 32 * qs * Tile::PITCH, qrow = wa_opaque(row_base + sq), qcol = wa_opaque(col_base + sq);
        const uint32_t vrow = VREG ? 0 : wa_opaque(row_base + tiles_at + 4 * BUF + 32 * kb * Tile::PITCH);
        const float* st = stats + (t & 1) * 3 * ROWS + 32 * qs + 4 * hl;
        const int* sp = reinterpret_cast<const int*>(stats + (t & 1) * 3 * ROWS + 2 * ROWS + 32 * qs);
        const int rlo = block(t) + 32 * qs;
        const int pmin = seen.off + wa_query(w, rlo), pmax = seen.off + wa_query(w, rlo + 31);      // (rows behind the last one: no harm)
        if (rlo < rr.hi && rlo + 32 > rr.lo && !(far && kmin >= a.sinks) && pmax >= kmin - a.right && (pmin <= kmax + a.left || kmin < a.sinks)) {
            __builtin_amdgcn_s_setprio(1);
            wa_f32x16 s = wa_zero16(), dp = wa_zero16();
#pragma unroll
            for (int i = 0; i < KST; ++i) {
                s = WaMma<T>::mma(wa_frag_row<T>(qrow, i, 0), kf[i], s);
                if constexpr (VREG) dp = WaMma<T>::mma(wa_frag_row<T>(qrow, i, BUF), vf[i], dp);
                else dp = WaMma<T>::mma(wa_frag_row<T>(qrow, i, BUF), wa_frag_row<T>(vrow, i, 0), dp);
            }
            __builtin_amdgcn_s_setprio(0);
            const bool all = whole && rlo >= rr.lo && rlo + 32 <= rr.hi && kmax <= pmin + a.right && (kmin >= pmax - a.left || kmax < a.sinks);
            float p[16], ds[16];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float4 lse = *reinterpret_cast<const float4*>(st + 8 * j), dl = *reinterpret_cast<const float4*>(st + ROWS + 8 * j);
                const float ls[4] = {lse.x, lse.y, lse.z, lse.w}, de[4] = {dl.x, dl.y, dl.z, dl.w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int r = 4 * j + e;
                    p[r] = wa_exp2(fmaf(s[r], w.c, -ls[e]));
                    ds[r] = (NARROW ? p[r] * up : p[r]) * (dp[r] - de[e]);
                }
            }
            if (!all) {
                const bool cut = rlo < rr.lo || rlo + 32 > rr.hi;            // (uniform) rows outside the range: another workgroup's, or none
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int4 po = *reinterpret_cast<const int4*>(sp + 4 * hl + 8 * j);
                    const int ps[4] = {po.x, po.y, po.z, po.w};
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const bool see = (uint32_t)(ps[e] - see_from) <= see_n;
                        p[4 * j + e] = see ? p[4 * j + e] : 0.f;
                        ds[4 * j + e] = see ? ds[4 * j + e] : 0.f;
                    }
                }
                if (cut) {
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        const bool in = (uint32_t)(rlo - rr.lo + 4 * hl + 8 * (r >> 2) + (r & 3)) < (uint32_t)(rr.hi - rr.lo);
                        p[r] = in ? p[r] : 0.f;
                        ds[r] = in ? ds[r] : 0.f;
                    }
                }
            }
            if constexpr (NARROW) {
                const float largest = wa_largest(ds);
                if (__any(largest > WA_TOP)) {
                    const int e = wa_fall(largest);
                    up = __builtin_ldexpf(up, e);
#pragma unroll
                    for (int r = 0; r < 16; ++r) ds[r] = __builtin_ldexpf(ds[r], e);
                    wa_scale<DT>(dk, e);
                }
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const typename WaMma<T>::v8 pf = wa_pack8<T>(p + 8 * i), df = wa_pack8<T>(ds + 8 * i);
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) {
                    dv[dt] = WaMma<T>::mma(wa_frag_col<T, DP>(qcol, dt, 16 * i * Tile::PITCH + BUF), pf, dv[dt]);
                    dk[dt] = WaMma<T>::mma(wa_frag_col<T, DP>(qcol, dt, 16 * i * Tile::PITCH), df, dk[dt]);
                }
            }
        }
        wa_stage_wait<0>();
        __syncthreads();
    }
    if constexpr (NARROW) { wa_scale<DT>(dk, 1 - WA_LIFT - __builtin_amdgcn_frexp_expf(up)); wa_scale<DT>(dv, -WA_LIFT); }
    // the two halves of the rows: through LDS, dV first
    float* slot = reinterpret_cast<float*>(lds) + kb * (DT * 16 * 64) + lane;
    static_assert(KB * DT * 16 * 64 * 4 <= 4 * BUF, "the partial results fit the stage buffers");
#pragma unroll
    for (int pass = 0; pass < 2; ++pass) {
        wa_f32x16* acc = pass ? dk : dv;
        if (pass) __syncthreads();
        if (qs == 1) {
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                for (int r = 0; r < 16; ++r) slot[(dt * 16 + r) * 64] = acc[dt][r];
        }
        __syncthreads();
        if (qs == 0) {
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                for (int r = 0; r < 16; ++r) acc[dt][r] += slot[(dt * 16 + r) * 64];
        }
    }
    if (qs != 0) return;
    if (w.chunks > 0 && key < a.sinks) {                                     // a first token: one of the pieces of its sum
        const size_t piece = (size_t)bh * (w.chunks + 1) + (far ? chunk + 1 : 0);
        float* part = a.ws + wa_row_floats(w) + (piece * a.sinks + key) * 2 * DP;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int d = 32 * dt + 8 * j + 4 * hl;
                *reinterpret_cast<float4*>(part + d) = make_float4(dk[dt][4 * j], dk[dt][4 * j + 1], dk[dt][4 * j + 2], dk[dt][4 * j + 3]);
                *reinterpret_cast<float4*>(part + DP + d) = make_float4(dv[dt][4 * j], dv[dt][4 * j + 1], dv[dt][4 * j + 2], dv[dt][4 * j + 3]);
            }
        return;
    }
    if (far) return;
    if (key >= a.Lkv) return;
    T* okp = (T*)a.dk + b * a.dk_sb + key * a.dk_sl + hk * a.dk_sh;
    T* ovp = (T*)a.dv + b * a.dv_sb + key * a.dv_sl + hk * a.dv_sh;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int d = 32 * dt + 8 * j + 4 * hl;
            const float x[4] = {dk[dt][4 * j] * a.scale, dk[dt][4 * j + 1] * a.scale, dk[dt][4 * j + 2] * a.scale, dk[dt][4 * j + 3] * a.scale};
            const float y[4] = {dv[dt][4 * j], dv[dt][4 * j + 1], dv[dt][4 * j + 2], dv[dt][4 * j + 3]};
            if (d < a.head_dim) { vpf_store<T, 4>(okp + d, x); vpf_store<T, 4>(ovp + d, y); }
        }
}

// pieces of the first tokens' sums -> dk, dv: one workgroup per first token and (sample, key head)
template <typename T, int DP>
__global__ void __launch_bounds__(2 * DP) wa_sink_join_kernel(WaArgs w)
{
    const VpfWindowAttn& a = w.a;
    const int bh = blockIdx.x / a.sinks, key = blockIdx.x % a.sinks, d = threadIdx.x % DP;
    const bool is_v = threadIdx.x >= DP;
    const float* p = a.ws + wa_row_floats(w) + ((size_t)bh * (w.chunks + 1) * a.sinks + key) * 2 * DP + threadIdx.x;
    float s = 0.f;
#pragma unroll 4
    for (int c = 0; c <= w.chunks; ++c) s += p[(size_t)c * a.sinks * 2 * DP];
    if (d >= a.head_dim) return;
    const int b = bh / a.Hk, hk = bh % a.Hk;
    if (is_v) ((T*)a.dv)[b * a.dv_sb + key * a.dv_sl + hk * a.dv_sh + d] = (T)s;
    else ((T*)a.dk)[b * a.dk_sb + key * a.dk_sl + hk * a.dk_sh + d] = (T)(s * a.scale);
}

// ------------------------------------------------------------------ host
static long wa_min(long a, long b) { return a < b ? a : b; }
static int wa_dp(int dh) { return dh <= 32 ? 32 : dh <= 64 ? 64 : dh <= 96 ? 96 : 128; }

static int wa_prepare(const VpfWindowAttn* args, WaArgs& w)
{
    if (!args) return VPF_ERR_NULL;
    w = {};
    w.a = *args;
    VpfWindowAttn& a = w.a;
    if (a.B < 0 || a.Lq < 0 || a.Lkv < 0 || a.Hk < 1 || a.Hq < a.Hk || a.Hq % a.Hk || a.head_dim < 8 || a.head_dim > VPF_WINDOW_MAX_DIM || a.head_dim % 8 ||
        a.Lkv >= WA_FAR || a.Lq >= WA_FAR - a.Lkv || a.sinks < 0 || !(a.scale > 0.f) || !(a.scale < INFINITY)) return VPF_ERR_BADSHAPE;
    if (a.dtype != VPF_T_F16 && a.dtype != VPF_T_BF16) return VPF_ERR_UNSUPPORTED;
    a.left = a.left < 0 || a.left > WA_FAR ? WA_FAR : a.left;
    a.right = a.right < 0 || a.right > WA_FAR ? WA_FAR : a.right;
    a.sinks = a.sinks < a.Lkv ? a.sinks : a.Lkv;
    if (a.left >= a.Lkv) a.sinks = 0;                            // everything behind a query is in its window
    w.g = a.Hq / a.Hk;
    if ((long)a.Lq * w.g * w.g >= 1L << 31 || (long)a.B * a.Hk >= 1L << 24) return VPF_ERR_BADSHAPE;
    w.rows = a.Lq * w.g;
    w.magic = w.g > 1 ? (uint32_t)((1ULL << 32) / w.g + 1) : 0;
    w.c = a.scale * WA_LOG2E;
    return VPF_OK;
}
// 16-byte rows; the offsets inside a stage are 32-bit byte offsets: 127 keys' strides below 2^31, and in the dK / dV kernel a row's query
// (at most 63 of them, 32 where heads share a key head) and head: 2 (2^28 + 2^29) bytes with the heads of a key head below 2^29 elements.  Where a
// head or a sample begins is found in 64 bits.
static bool wa_aligned(const void* p, long sb, long sl, long sh)
{
    return vpf_aligned(p, 16) && sb % 8 == 0 && sl % 8 == 0 && sh % 8 == 0 && sl >= 0 && sl < VPF_WINDOW_MAX_STRIDE && sh >= 0;
}

// Row blocks of 32 per workgroup (4, 2 or 1; the waves that are left split a stage's keys): as many as leave a workgroup for each of the 256 CUs.
static int wa_row_blocks(const WaArgs& w)
{
    const long pairs = (long)w.a.B * w.a.Hk;
    return pairs * vpf_cdiv(w.rows, 128) >= 256 ? 4 : pairs * vpf_cdiv(w.rows, 64) >= 256 ? 2 : 1;
}
// Walks of one length: the window leaves most of the keys out, so few tiles are cut short by the ends of the sequence.
static int wa_runs(const WaArgs& w) { return (long)w.a.B * w.a.Hk < 8 && ((long)w.a.left + w.a.right) * 2 < w.a.Lkv; }
// Can a row see nothing?  Not where every query stands at a key that is in use and no padding.
static bool wa_blind(const WaArgs& w) { return w.a.pad || w.a.lens || w.a.Lq > w.a.Lkv; }
// Where even single row blocks are too few, the keys are divided as well: one workgroup per CU (a stage of 128 keys is up to 64 KB of loads in flight),
// each with at least two stages, and at most 64 parts (a wave of the join).
static void wa_plan_fwd(WaArgs& w, int& rb)
{
    rb = wa_row_blocks(w);
    // Two row blocks a wave (256 rows a workgroup) from head dimension 72 on, where the walk over the keys is long beside the queries of a tile
    // (bf16, left window + causal; one / two blocks, us: dim 128, 4 heads a key, window 256 181 / 182, 512 245 / 241, 1024 383 / 368, 4096 1220 / 1137;
    // dim 96, 1 head, 4096 278 / 246; dim 64, 1 head, 4096 173 / 186, which the exponentials bound, not the LDS).
    const long seen = wa_min((long)w.a.left + w.a.right + 1, (long)w.a.Lkv);
    if (rb == 4 && w.a.head_dim > 64 && seen * w.g >= 16 * 256 && (long)w.a.B * w.a.Hk * vpf_cdiv(w.rows, 256) >= 256) rb = 8;
    w.tiles = vpf_cdiv(w.rows, 32 * rb);
    w.splits = 1;
    const long wgs = (long)w.a.B * w.a.Hk * w.tiles;
    if (rb == 1 && wgs <= 128) {
        const long span = (long)w.a.left + w.a.right + 1 + 31 / w.g + w.a.sinks, keys = span < w.a.Lkv ? span : w.a.Lkv;
        const long stages = (keys + 127) / 128, want = 256 / wgs, most = stages / 2 < 64 ? stages / 2 : 64;
        w.splits = (int)(want < most ? want : most);
        if (w.splits < 1) w.splits = 1;
    }
    w.runs = w.splits == 1 && wa_runs(w);
}
static long wa_fwd_ws(const WaArgs& w) { return w.splits > 1 ? (long)w.splits * w.a.B * w.a.Hk * w.rows * (wa_dp(w.a.head_dim) + 2) : 0; }

// Key tiles of 128 at head dimension 128 where that leaves a workgroup for each CU (the stages of Q and dO then serve twice the keys), else of 64.
// The rows behind a sink tile's own window are cut into pieces about as long as the row range of an ordinary tile, where that leaves more than
// one of them: about 32 pieces, at most 33 (they are fp32 scratch), none where the first tokens fill more than 8 tiles (enough workgroups by themselves).
static void wa_plan_bwd(WaArgs& w)
{
    const VpfWindowAttn& a = w.a;
    w.key_tile = wa_dp(a.head_dim) == 128 && (long)a.B * a.Hk * vpf_cdiv(a.Lkv, 128) >= 256 ? 128 : 64;
    w.ktiles = vpf_cdiv(a.Lkv, w.key_tile);
    w.sink_tiles = vpf_cdiv(a.sinks, w.key_tile);
    w.chunks = 0;
    const long range = ((long)a.left + a.right + w.key_tile) * w.g, all = vpf_cdiv(w.rows, WA_ROWS), cycle = range / WA_ROWS + 2;
    w.cycle = (int)(cycle < all ? cycle : all > 0 ? all : 1);
    if (w.sink_tiles > 0 && w.sink_tiles <= 8 && w.rows > 2 * range) {
        long rows = range > 512 ? range : 512;
        rows = rows > w.rows / 32 ? rows : w.rows / 32;
        w.chunk_rows = (int)((rows + 63) / 64 * 64);
        w.chunks = vpf_cdiv(w.rows, w.chunk_rows);
    }
}
static long wa_bwd_ws(const WaArgs& w)
{
    return (long)wa_row_floats(w) + (w.chunks ? (long)w.a.B * w.a.Hk * (w.chunks + 1) * w.a.sinks * 2 * wa_dp(w.a.head_dim) : 0);
}

// more than 64 KB of LDS has to be asked for, once per kernel and device
template <typename K> static int wa_lds(K kernel, size_t bytes, VpfPerDevice& done)
{
    bool& d = done();
    if (!d && bytes > 65536 && hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes) != hipSuccess) return VPF_ERR_HIP;
    d = true;
    return VPF_OK;
}

template <typename T, int DP, int RB, int RW, int KS, int SUBK> static int wa_launch_fwd(const WaArgs& w, hipStream_t st)
{
    constexpr size_t lds = 4 * SUBK * KS * WaTile<DP>::PITCH + SUBK * KS / 4;
    static VpfPerDevice done;
    if (const int rc = wa_lds(wa_fwd_kernel<T, DP, RB, RW, KS, SUBK>, lds, done)) return rc;
    const long grid = (long)w.a.B * w.a.Hk * w.tiles * w.splits;
    if (grid >= WA_MAX_GRID) return VPF_ERR_BADSHAPE;
    hipLaunchKernelGGL((wa_fwd_kernel<T, DP, RB, RW, KS, SUBK>), dim3((unsigned)grid), dim3(WA_THREADS), lds, st, w);
    if (w.splits > 1) hipLaunchKernelGGL((wa_join_kernel<T, DP>), dim3(vpf_cdiv((long)w.a.B * w.a.Hk * w.rows, 4)), dim3(WA_THREADS), 0, st, w);
    VPF_CHECK_LAUNCH();
    return VPF_OK;
}
template <typename T, int DP> static int wa_fwd(const WaArgs& w, int rb, hipStream_t st)
{
    if constexpr (DP > 64) { if (rb == 8) return wa_launch_fwd<T, DP, 4, 2, 1, 64>(w, st); }
    if (rb == 4) return wa_launch_fwd<T, DP, 4, 1, 1, 64>(w, st);
    if (rb == 2) return wa_launch_fwd<T, DP, 2, 1, 2, 32>(w, st);
    return wa_launch_fwd<T, DP, 1, 1, 4, 32>(w, st);
}

template <typename T, int DP, int RB, int KS> static int wa_launch_dq(const WaArgs& w, hipStream_t st)
{
    constexpr int STAGE = (KS == 1 ? 64 : 32) * KS;
    constexpr size_t lds = 4 * STAGE * WaTile<DP>::PITCH + STAGE / 4 + KS * RB * 32 * 4;
    static VpfPerDevice done;
    if (const int rc = wa_lds(wa_dq_kernel<T, DP, RB, KS>, lds, done)) return rc;
    hipLaunchKernelGGL((wa_dq_kernel<T, DP, RB, KS>), dim3((unsigned)((long)w.a.B * w.a.Hk * w.tiles)), dim3(WA_THREADS), lds, st, w);
    VPF_CHECK_LAUNCH();
    return VPF_OK;
}
template <typename T, int DP> static int wa_bwd(WaArgs& w, hipStream_t st)
{
    const long bh = (long)w.a.B * w.a.Hk;
    const int rb = wa_row_blocks(w);
    w.tiles = vpf_cdiv(w.rows, 32 * rb);
    w.splits = 1;
    w.runs = wa_runs(w);
    const long grid = bh * (w.ktiles + (long)w.sink_tiles * w.chunks);
    if (grid >= WA_MAX_GRID || bh * w.tiles >= WA_MAX_GRID || bh * w.a.sinks >= WA_MAX_GRID) return VPF_ERR_BADSHAPE;      // in front of every launch
    if (w.rows > 0) {
        const int rc = rb == 4 ? wa_launch_dq<T, DP, 4, 1>(w, st) : rb == 2 ? wa_launch_dq<T, DP, 2, 2>(w, st) : wa_launch_dq<T, DP, 1, 4>(w, st);
        if (rc) return rc;
    }
    if (w.a.Lkv == 0) return VPF_OK;
    auto launch = [&](auto kernel, int kb, VpfPerDevice& done) -> int {
        const size_t lds = 4 * WA_ROWS * WaTile<DP>::PITCH + (DP <= 96 ? 0 : 32 * kb * WaTile<DP>::PITCH) + 6 * WA_ROWS * 4;
        if (const int rc = wa_lds(kernel, lds, done)) return rc;
        hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(128 * kb), lds, st, w);
        return VPF_OK;
    };
    static VpfPerDevice done2, done4, done2b, done4b;
    const bool blind = wa_blind(w);
    if constexpr (DP == 128) {
        if (w.key_tile == 128)
            if (const int rc = blind ? launch(wa_dkv_kernel<T, DP, 4, true>, 4, done4b) : launch(wa_dkv_kernel<T, DP, 4, false>, 4, done4)) return rc;
    }
    if (w.key_tile == 64)
        if (const int rc = blind ? launch(wa_dkv_kernel<T, DP, 2, true>, 2, done2b) : launch(wa_dkv_kernel<T, DP, 2, false>, 2, done2)) return rc;
    if (w.chunks) {
        hipLaunchKernelGGL((wa_sink_join_kernel<T, DP>), dim3((unsigned)(bh * w.a.sinks)), dim3(2 * DP), 0, st, w);
    }
    VPF_CHECK_LAUNCH();
    return VPF_OK;
}

#define WA_PICK(FN, ...) \
    switch (wa_dp(w.a.head_dim)) { \
        case 32: return w.a.dtype == VPF_T_F16 ? FN<vpf_f16, 32>(__VA_ARGS__) : FN<vpf_bf16, 32>(__VA_ARGS__); \
        case 64: return w.a.dtype == VPF_T_F16 ? FN<vpf_f16, 64>(__VA_ARGS__) : FN<vpf_bf16, 64>(__VA_ARGS__); \
        case 96: return w.a.dtype == VPF_T_F16 ? FN<vpf_f16, 96>(__VA_ARGS__) : FN<vpf_bf16, 96>(__VA_ARGS__); \
        default: return w.a.dtype == VPF_T_F16 ? FN<vpf_f16, 128>(__VA_ARGS__) : FN<vpf_bf16, 128>(__VA_ARGS__); \
    }

extern "C" long vpf_window_attn_ws(const VpfWindowAttn* args, int backward)
{
    WaArgs w;
    if (const int rc = wa_prepare(args, w)) return rc;
    if ((long)w.a.B * w.rows == 0 && !backward) return 0;
    int rb;
    if (backward) { wa_plan_bwd(w); return wa_bwd_ws(w); }
    wa_plan_fwd(w, rb);
    return wa_fwd_ws(w);
}

extern "C" int vpf_window_attn_fwd(const VpfWindowAttn* args, void* stream)
{
    (void)hipGetLastError();
    WaArgs w;
    if (const int rc = wa_prepare(args, w)) return rc;
    const VpfWindowAttn& a = w.a;
    if ((long)a.B * w.rows == 0) return VPF_OK;
    if (!a.q || !a.out || (a.Lkv > 0 && (!a.k || !a.v))) return VPF_ERR_NULL;
    if (!wa_aligned(a.q, a.q_sb, a.q_sl, a.q_sh) || !wa_aligned(a.k, a.k_sb, a.k_sl, a.k_sh) || !wa_aligned(a.v, a.v_sb, a.v_sl, a.v_sh) ||
        !wa_aligned(a.out, a.o_sb, a.o_sl, a.o_sh) || !vpf_aligned(a.ws, 16)) return VPF_ERR_BADALIGN;
    int rb;
    wa_plan_fwd(w, rb);
    if (w.splits > 1 && (!a.ws || a.ws_floats < wa_fwd_ws(w))) return a.ws ? VPF_ERR_BADSHAPE : VPF_ERR_NULL;
    WA_PICK(wa_fwd, w, rb, (hipStream_t)stream)
}

extern "C" int vpf_window_attn_bwd(const VpfWindowAttn* args, void* stream)
{
    (void)hipGetLastError();
    WaArgs w;
    if (const int rc = wa_prepare(args, w)) return rc;
    const VpfWindowAttn& a = w.a;
    if (a.B == 0 || (w.rows == 0 && a.Lkv == 0)) return VPF_OK;
    if ((w.rows > 0 && (!a.q || !a.out || !a.out_lo || !a.dout || !a.lse || !a.dq || !a.ws)) || (a.Lkv > 0 && (!a.k || !a.v || !a.dk || !a.dv))) return VPF_ERR_NULL;
    const struct { const void* p; long sb, sl, sh; } t[] = {{a.q, a.q_sb, a.q_sl, a.q_sh}, {a.k, a.k_sb, a.k_sl, a.k_sh}, {a.v, a.v_sb, a.v_sl, a.v_sh},
        {a.out, a.o_sb, a.o_sl, a.o_sh}, {a.dout, a.do_sb, a.do_sl, a.do_sh}, {a.dq, a.dq_sb, a.dq_sl, a.dq_sh}, {a.dk, a.dk_sb, a.dk_sl, a.dk_sh},
        {a.dv, a.dv_sb, a.dv_sl, a.dv_sh}, {a.out_lo, 0, 0, 0}, {a.ws, 0, 0, 0}};
    for (const auto& x : t) if (!wa_aligned(x.p, x.sb, x.sl, x.sh)) return VPF_ERR_BADALIGN;
    if (w.g * a.q_sh >= VPF_WINDOW_MAX_HEADS || w.g * a.do_sh >= VPF_WINDOW_MAX_HEADS) return VPF_ERR_BADALIGN;
    wa_plan_bwd(w);
    if (a.ws_floats < wa_bwd_ws(w)) return VPF_ERR_BADSHAPE;
    WA_PICK(wa_bwd, w, (hipStream_t)stream)
}
