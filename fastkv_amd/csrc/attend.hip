// Attention over a cache with the matrix instructions: a sliding window with sinks (prompts, chunks, single tokens) and a batch over
// one shared prefix.  The dense decode of decode.hip / decode_step.hip reads every row of a slab for one token; here a query row sees
//   window        rows j <= p with j < sinks or j > p - window                    (p = cached rows before the call + its index)
//   shared prefix the whole prefix, and its request's own rows j <= p
// and a call has T >= 1 tokens per request.  out = sum softmax(scaling q.k) v over what a row sees; a row with p < 0 sees nothing: zeros.
//
// Mathematics.  The G query heads of a KV head and the T tokens are one list of rows r = t*G + g: they share every K / V byte that a
// workgroup reads.  One pass over the keys with a running maximum m and sum l per row (both fp32):
//   S^T = K Q^T          32x32x16 matrix instructions; a lane holds ONE query (column lane & 31) and 16 keys of a 32-key block, so the
//                        row maximum is 16 register operations and one exchange between the wave's halves
//   P^T = exp2(c S^T - c m), c = scaling log2 e (fp16: times 2^7), rounded to the inputs' 16 bits (nearest even: half a step of p, averaged over the
//                        keys; the sum l adds the unrounded p)
//   O^T += V^T P^T       the registers of P^T ARE the second operand: lane half h of a 16-key step holds keys 4h .. 4h+3 and
//                        8+4h .. 8+4h+3, and V^T is read with the same order of keys -- no exchange, no shared memory for P.
//                        V^T comes out of the row-major tile by ds_read_b64_tr_b16 (four keys of one dim per lane)
// O is rescaled only when a maximum grows by more than 2^8 (p stays within the 16-bit types' range).
//
// Keys are numbered through: u in [0, N) = n0 rows of segment 0 (the sinks in front of the window, or the prefix), then rows lo .. hi-1
// of the request's cache.  Work is cut along u, so a window that starts far behind its sinks costs no empty tiles.
//
// Two shapes of a workgroup (4 waves):
//   rows      4 x 32 rows, all waves on one 64-key tile (two tiles in shared memory, one barrier per tile); two workgroups per compute unit, whose
//             products and exponentials fall beside each other as they drift apart
//   keys      <= 32 rows (single tokens): each wave has its own 32-key tiles and running state, merged at the end; a wave's tile is
//             private, so the loop has no barrier and eight waves of a compute unit keep ~128 KB of loads in flight
// Tiles go from memory to shared memory without passing registers (a wave has 512 / 2 of them at 128 dims, all in use).
// Work too small to fill the chip is cut along the keys; slices leave {m, l, O} in a workspace and attend_join adds them up.
//
// What bounds it, measured (H 32, Hkv 8, D 128; times in the kernels, medians of 36 calls on one card -- another card was 3 % faster on the prompts):
//   prompts   the matrix pipe, the vector pipe and the clock together: 8k tokens, window 4096: 0.448 ms, 920 TFLOP/s (an 8192^3 library product:
//             1110); 32k: 2.18 ms, 948.  Per tile of a wave 1024 cycles of products beside ~1000 of vector work; the clock falls to
//             1.95 GHz under it.  Leaving out the exponentials / the loads / the second product gives 7 / 14 / 12 %: nothing alone bounds it.
//             Slower: two groups of waves held half a tile apart by barriers (0.53 ms), raised wave priorities (+3 %), exponentials
//             interleaved with products by hand (+3 %), 32-key tiles (registers spill at three waves per SIMD).
//   tokens    the memory: 32 requests, window 4096: 88 us, 5.4 TB/s of K and V (a large copy: 5.1 read + write); one request, window 2048:
//             8.1 + 3.9 us, the latency of the chain kernel arguments - length - K - V - join - second launch
//   prefix    64 requests on 32768 shared rows: 66 + 9 us: 38 of products (twice 128 rows per KV head), 13 of the requests' own rows, the
//             slices' sums.  Alternating the shared and the own items over the grid is slower (84): a lone rows-shaped workgroup on a compute unit
//             has nothing beside its products.
#include <limits.h>
#include <initializer_list>
#include <type_traits>
#include "fk_device.h"
#include "fk_host.h"
#include "prof.h"

namespace fk {

typedef _Float16 att_h8 __attribute__((ext_vector_type(8)));
typedef __bf16 att_b8 __attribute__((ext_vector_type(8)));
typedef _Float16 att_h2 __attribute__((ext_vector_type(2)));
typedef __bf16 att_b2 __attribute__((ext_vector_type(2)));
typedef float att_f2 __attribute__((ext_vector_type(2)));
typedef float att_f16 __attribute__((ext_vector_type(16)));
typedef short att_s4 __attribute__((ext_vector_type(4)));
typedef uint32_t att_u4 __attribute__((ext_vector_type(4)));

constexpr int ATT_THREADS = 256;
constexpr float ATT_GROWTH = 8.0f;           // log2 of how far p may exceed its scale before O is rescaled
constexpr float ATT_LIFT = 7.0f;             // fp16: p is held times 2^7 (at most 2^15 with the growth), which keeps many small p out of the
                                             // subnormals; l and O carry the same factor

struct AttendArgs {
    const uint16_t *q;                       // [B,H,T,D]
    int64_t q_b, q_h, q_t;
    const uint16_t *k0, *v0;                 // segment 0: rows of [Hkv,n,D]; the cache itself for sinks (then + b * k_b)
    int64_t k0_b, k0_h, k0_r, v0_b, v0_h, v0_r;
    const uint16_t *k, *v;                   // [B,Hkv,rows,D]
    int64_t k_b, k_h, k_r, v_b, v_h, v_r;
    const int32_t *len;                      // rows before the call, per request (len_step 0: one for all); nullptr: len_all
    int len_step, len_all;
    int B, H, Hkv, G, T, rows;
    int window, sinks, prefix;               // prefix: rows of a shared prefix (window = none then)
    float c;                                 // scaling * log2(e)
    uint16_t *out;                           // [B,T,H,D]
    float *part_ml, *part_o;                 // [B*H*T][slots]{m, l}, [B*H*T][slots][D]
    int slots;                               // slices per row; 0: the result goes to `out`
    int packed_tiles, packed_split, slot0;   // shared prefix, few rows per request: row tiles over ALL requests in front of the grid
    int tiles, split;                        // row tiles per request, key slices
    int run;                                 // neighbouring items that one die gets
    bool near_rows;
};

template <bool BF> __device__ __forceinline__ att_f16 att_mfma(att_u4 a, att_u4 b, att_f16 c)
{
    if (BF) return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(att_b8, a), __builtin_bit_cast(att_b8, b), c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(att_h8, a), __builtin_bit_cast(att_h8, b), c, 0, 0, 0);
}
template <bool BF> __device__ __forceinline__ uint32_t att_pack(float x, float y)      // round to nearest even
{
    const att_f2 p = {x, y};
    if (BF) return __builtin_bit_cast(uint32_t, __builtin_convertvector(p, att_b2));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(p, att_h2));
}
template <bool BF> __device__ __forceinline__ float att_float(uint32_t h)
{
    return BF ? __builtin_bit_cast(float, h << 16) : h2f((uint16_t)h);
}
// a 16-bit element that is infinite or NaN in either half of a word
template <bool BF> __device__ __forceinline__ bool att_wild(uint32_t w)
{
    const uint32_t e = BF ? 0x7f80u : 0x7c00u;
    return (w & e) == e || (w >> 16 & e) == e;
}
template <bool BF> __device__ __forceinline__ bool att_wild_piece(att_u4 x)
{
    return att_wild<BF>(x[0]) || att_wild<BF>(x[1]) || att_wild<BF>(x[2]) || att_wild<BF>(x[3]);
}
// x of both halves' lanes of a column (the pair's words are copied out first: a bit cast of a vector element reads element 0 here)
struct AttPair { uint32_t lo, hi; };
__device__ __forceinline__ AttPair att_halves(float x)
{
    const uint32_t w = __builtin_bit_cast(uint32_t, x);
    const auto r = __builtin_amdgcn_permlane32_swap(w, w, false, false);
    AttPair p;
    p.lo = r[0];
    p.hi = r[1];
    return p;
}
__device__ __forceinline__ float att_other_half_max(float x)
{
    const AttPair p = att_halves(x);
    return fmaxf(__builtin_bit_cast(float, p.lo), __builtin_bit_cast(float, p.hi));
}
__device__ __forceinline__ float att_other_half_sum(float x)
{
    const AttPair p = att_halves(x);
    return __builtin_bit_cast(float, p.lo) + __builtin_bit_cast(float, p.hi);
}
// 16-byte piece c of row `row` of a tile lies at piece c ^ att_swz: shared memory serves 16 pieces (64 banks) at a time.  K: equal pieces of 16
// consecutive rows fall on different banks; V: four pieces in a row of each of four consecutive rows do (and eight rows on, all is the same).
template <int D, bool V> __device__ __forceinline__ int att_swz(int row)
{
    if (D == 64) return V ? (row >> 1 & 1) << 2 | (row >> 2 & 1) : (row >> 1 & 1) << 2 | (row >> 2 & 3);       // two rows are one turn of the banks
    return V ? (row & 3) << 2 | (row >> 2 & 1) : (row & 3) << 2 | (row >> 2 & 3);
}

// what a partial sum over keys of maximum m counts for beside the maximum M of all of them (no key at all: both are -inf; a NaN among
// the sums survives a weight of zero, as it survives in the formula)
__device__ __forceinline__ float att_weight(float m, float M, float c) { return M == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f((m - M) * c); }

struct AttKeys {                             // the keys of one item, and which of them a row at position p sees
    const uint16_t *k0, *v0, *k, *v;
    int64_t k0_r, v0_r, k_r, v_r;
    int n0, lo, N;                           // segment 0; first row of segment 1; all
    int window, sinks;
    int end0, end1, seen1, seen2;            // see whole(), lean()

    // For tiles of KT keys; a .. z: the positions of all rows; near_rows: 64 rows of any of the four lie within 31 bits of bytes
    __device__ __forceinline__ void look(int KT, bool near_rows, int a, int z)
    {
        end0 = near_rows ? min(n0, N) - KT : INT_MIN;
        end1 = near_rows ? N - KT : INT_MIN;
        seen1 = max(n0, z - window + 1 - lo + n0);
        seen2 = min(N, a + 1 - lo + n0) - KT;
    }
    // the tile at u lies in one segment with all its keys; ... and every row sees all of them: nearly all tiles are such
    __device__ __forceinline__ bool whole(int u) const { return u <= end0 || (u >= n0 && u <= end1); }
    __device__ __forceinline__ bool lean(int u) const { return u <= end0 || (u >= seen1 && u <= min(seen2, end1)); }
};

// Which keys a row at position p >= 0 sees, by their number from u0 on: k < end, and k < first (segment 0 and sinks) or k > before (the window).
// Written without branches: a select per score (a masked store under a branch has cost wrong code here).
struct AttSees {
    int end, first, before;
    __device__ __forceinline__ AttSees(const AttKeys &K, int u0, int p)
    {
        const int o = K.n0 - K.lo;                           // row j is key j + o
        end = min(K.N, p + o + 1) - u0;
        first = max(K.n0, K.sinks + o) - u0;
        before = p - K.window + o - u0;
    }
    __device__ __forceinline__ bool operator()(int k) const { return (k < end) & ((k < first) | (k > before)); }
};

struct AttState { float m, l; };

// 16 bytes per active lane from memory to shared memory: lane l's land at lds + OFF + 16 l.  Written as assembly because the compiler, which
// cannot tell the tile in flight from the one being read, waits for every such load in front of the next transposing read; the waits are
// att_landed's, and nothing of these loads is in a register.  m0 is reserved: the compiler sets it where it needs it and keeps nothing in it.
template <int OFF> __device__ __forceinline__ void att_bring(att_u4 buffer, int offset, int base_offset, uint32_t lds)
{
    asm volatile("s_add_u32 m0, %0, %4\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds"
                 :: "s"(lds), "v"(offset), "s"(buffer), "s"(base_offset), "n"(OFF) : "memory", "scc");
}
template <int OFF> __device__ __forceinline__ void att_bring(const uint16_t *src, uint32_t lds)
{
    asm volatile("s_add_u32 m0, %0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" :: "s"(lds), "v"(src), "n"(OFF) : "memory", "scc");
}
template <int I, int N, class F> __device__ __forceinline__ void att_each(F &&f)      // f(0) .. f(N - 1), the index a constant
{
    if constexpr (I < N) {
        f(std::integral_constant<int, I>());
        att_each<I + 1, N>(f);
    }
}
__device__ __forceinline__ uint32_t att_uniform(uint32_t x) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)x); }

// Rows u0 .. u0 + 32*NB - 1 of K and V on their way to shared memory, brought by NW waves without passing registers (the 16 bytes of lane l
// land at a wave's base + 16 l; the swizzle is in which piece of the row the lane asks for).
template <int D, int NB, int NW> struct AttLoad {
    static constexpr int KT = 32 * NB, C = D / 8, RPI = 64 / C, CH = KT / (RPI * NW);     // rows per instruction, instructions per wave
    static constexpr int NV = RPI * NW >= 16 ? 1 : 16 / (RPI * NW);                       // distinct swizzles over a lane's rows
    static constexpr int STEP = NW * RPI * D * 2;                                         // bytes from one instruction's rows to the next's

    static __device__ __forceinline__ int row_of(int i, int w, int lane) { return (i * NW + w) * RPI + lane / C; }
    static __device__ __forceinline__ uint32_t lds_of(const uint16_t *dst, int w)
    {
        return att_uniform((uint32_t)(uintptr_t)(const __attribute__((address_space(3))) uint16_t *)dst + w * RPI * D * 2);
    }
    // A whole tile of rows row, row + 1, ... of `base`: a 32-bit offset per lane, the tile's base in scalar registers
    template <bool V> static __device__ __forceinline__ void plain(const uint16_t *base, int64_t r, int row, uint32_t lds, int w)
    {
        const int lane = threadIdx.x & 63, step = (int)r * 2;
        const uintptr_t at = (uintptr_t)(base + (row + w * RPI) * r);
        const att_u4 buffer = {att_uniform((uint32_t)at), att_uniform((uint32_t)(at >> 32)) & 0xffffu, 0x7fffffffu, 0x00020000u};
        att_each<0, CH>([&](auto I) {
            constexpr int i = I;
            const int c = (lane % C) ^ att_swz<D, V>(row_of(i % NV, w, lane));
            att_bring<i * STEP>(buffer, lane / C * step + c * 16, (int)att_uniform(i * NW * RPI * step), lds);
        });
    }
    // Any other tile (over the segments' seam, the last one, rows further apart than 32 bits reach): an address per lane, and zeros behind the
    // last key -- their scores are cut off, but a V row there must be finite.
    template <bool V> static __device__ __forceinline__ void any(const AttKeys &K, int u0, uint16_t *dst, int w)
    {
        int lane = threadIdx.x & 63;
        asm volatile("" : "+v"(lane));           // (nothing of this is worth registers across the loop)
        const uint32_t lds = lds_of(dst, w);
        att_each<0, CH>([&](auto I) {
            constexpr int i = I;
            const int row = row_of(i, w, lane), u = u0 + row, c = (lane % C) ^ att_swz<D, V>(row);
            if (u < K.N) {
                const bool f = u < K.n0;
                const int64_t j = f ? u : K.lo + u - K.n0;
                att_bring<i * STEP>((V ? (f ? K.v0 : K.v) + j * (f ? K.v0_r : K.v_r) : (f ? K.k0 : K.k) + j * (f ? K.k0_r : K.k_r)) + c * 8, lds);
            } else {
                *reinterpret_cast<att_u4 *>(dst + (i * NW + w) * RPI * D + lane * 8) = att_u4{0, 0, 0, 0};
            }
            __builtin_amdgcn_sched_barrier(0);   // (one address at a time)
        });
    }
    template <bool V> static __device__ __forceinline__ void issue(const AttKeys &K, int u0, uint16_t *dst, int w)
    {
        if (!K.whole(u0)) any<V>(K, u0, dst, w);
        else if (u0 < K.n0) plain<V>(V ? K.v0 : K.k0, V ? K.v0_r : K.k0_r, u0, lds_of(dst, w), w);
        else plain<V>(V ? K.v : K.k, V ? K.v_r : K.k_r, K.lo + u0 - K.n0, lds_of(dst, w), w);
    }
    // This lane's V pieces, landed, of a tile that some row does not see all of: an infinity or NaN must not touch the rows that do not see it
    // (0 * inf), so a piece that holds one is taken out of the tile, its row is noted, and att_wild_rows adds it for the rows that see it.
    template <bool BF> static __device__ __forceinline__ void scan(uint16_t *vs, int w, unsigned long long *wild)
    {
        const int lane = threadIdx.x & 63;
#pragma unroll 1
        for (int i = 0; i < CH; ++i) {
            att_u4 *at = reinterpret_cast<att_u4 *>(vs + (i * NW + w) * RPI * D + lane * 8);
            if (att_wild_piece<BF>(*at)) {
                *at = att_u4{0, 0, 0, 0};
                atomicOr(wild, 1ull << row_of(i, w, lane));
            }
        }
    }
};

// all of this wave's loads to shared memory but the last LEFT have landed (they come back in order)
template <int LEFT> __device__ __forceinline__ void att_landed()
{
    __builtin_amdgcn_s_waitcnt(0x0f70 | (LEFT & 15) | (LEFT >> 4) << 14);
    asm volatile("" ::: "memory");
}
// this wave's reads of shared memory are done: what they read may be overwritten
__device__ __forceinline__ void att_read_done()
{
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0xc07f);      // lgkmcnt(0)
    asm volatile("" ::: "memory");
}

// S^T = K Q^T of a tile of 32*NB keys
template <int D, bool BF, int NB> __device__ __forceinline__ void att_scores(const uint16_t *ks, const att_u4 (&Q)[D / 16], att_f16 (&S)[NB])
{
    const int lane = threadIdx.x & 63, col = lane & 31, hi = lane >> 5, sw = att_swz<D, false>(col);
    constexpr int NX = D == 64 ? 4 : 8;      // piece (2 s + hi) ^ sw of row col: the swizzle is in the low three or four bits
    const uint16_t *at[NX];
#pragma unroll
    for (int x = 0; x < NX; ++x) at[x] = ks + col * D + ((2 * x + hi) ^ sw) * 8;
#pragma unroll
    for (int kb = 0; kb < NB; ++kb)
#pragma unroll
        for (int r = 0; r < 16; ++r) S[kb][r] = 0.0f;
#pragma unroll
    for (int s = 0; s < D / 16; ++s)
#pragma unroll
        for (int kb = 0; kb < NB; ++kb) S[kb] = att_mfma<BF>(*reinterpret_cast<const att_u4 *>(at[s % NX] + s / NX * NX * 16 + kb * 32 * D), Q[s], S[kb]);
}

// keys u0 .. of a tile that this lane's row (position p) does not see
template <int NB> __device__ __forceinline__ void att_mask(att_f16 (&S)[NB], const AttKeys &K, int u0, int p)
{
    const AttSees sees(K, u0 + 4 * (threadIdx.x >> 5 & 1), p);
#pragma unroll
    for (int kb = 0; kb < NB; ++kb)
#pragma unroll
        for (int r = 0; r < 16; ++r) S[kb][r] = sees(kb * 32 + (r & 3) + 8 * (r >> 2)) ? S[kb][r] : -INFINITY;
}
// a tile's weights 2^(c (s - m)): P^T as the second operand of V^T P^T, and their sum
template <bool BF, int NB> __device__ __forceinline__ float att_weights(const att_f16 (&S)[NB], att_u4 (&P)[NB * 2], float m, float c)
{
    const float mc = (m == -INFINITY ? 0.0f : m * c) - (BF ? 0.0f : ATT_LIFT);
    float l0 = 0.0f, l1 = 0.0f;
#pragma unroll
    for (int kb = 0; kb < NB; ++kb)
#pragma unroll
        for (int r = 0; r < 16; r += 2) {
            const float a = __builtin_amdgcn_exp2f(__builtin_fmaf(S[kb][r], c, -mc)), b = __builtin_amdgcn_exp2f(__builtin_fmaf(S[kb][r + 1], c, -mc));
            l0 += a;
            l1 += b;
            P[kb * 2 + (r >> 3)][(r & 7) >> 1] = att_pack<BF>(a, b);
        }
    return l0 + l1;
}
// the running softmax over a tile's scores, u0 its first key; `edge`: some row may not see some key
template <int D, bool BF, int NB>
__device__ __forceinline__ void att_softmax(att_f16 (&S)[NB], att_u4 (&P)[NB * 2], att_f16 (&O)[D / 32], AttState &st, float c, const AttKeys &K, int u0,
                                            int p, bool edge)
{
    if (edge) att_mask<NB>(S, K, u0, p);
    float tm = -INFINITY;
#pragma unroll
    for (int kb = 0; kb < NB; ++kb)
#pragma unroll
        for (int r = 0; r < 16; ++r) tm = __builtin_elementwise_maximum(tm, S[kb][r]);
    tm = att_other_half_max(tm);
    if (__any((tm - st.m) * c > ATT_GROWTH)) {
        const float mn = fmaxf(st.m, tm);
        const float f = mn == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f((st.m - mn) * c);
        st.m = mn;
        st.l *= f;
#pragma unroll
        for (int db = 0; db < D / 32; ++db)
#pragma unroll
            for (int r = 0; r < 16; ++r) O[db][r] *= f;
    }
    st.l += att_weights<BF, NB>(S, P, st.m, c);
}

// O^T += V^T P^T
template <int D, bool BF, int NB> __device__ __forceinline__ void att_values(const uint16_t *vs, const att_u4 (&P)[NB * 2], att_f16 (&O)[D / 32])
{
    // lane i of a group of 16 addresses row i / 4, elements 4 * (i % 4) of a 4 x 16 block and receives column i
    const int lane = threadIdx.x & 63, hi = lane >> 5, gi = lane & 15, krow = gi >> 2;
    const int piece = (lane >> 4 & 1) * 2 + (gi >> 1 & 1), sw = att_swz<D, true>(4 * hi + krow);
    typedef __attribute__((address_space(3))) att_s4 lds_s4;
    constexpr int NX = D == 64 ? 2 : 4;      // dims 32 db + 8 piece + ..: the swizzle is in the low three or four bits of 4 db + piece
    const uint16_t *at[NX];
#pragma unroll
    for (int x = 0; x < NX; ++x) at[x] = vs + (4 * hi + krow) * D + ((4 * x + piece) ^ sw) * 8 + (gi & 1) * 4;
#pragma unroll
    for (int s = 0; s < NB * 2; ++s) {
#pragma unroll
        for (int db = 0; db < D / 32; ++db) {
            const uint16_t *v = at[db % NX] + db / NX * NX * 32 + s * 16 * D;
            const att_s4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4 *)v);
            const att_s4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4 *)(v + 8 * D));
            const uint2 xa = __builtin_bit_cast(uint2, x), ya = __builtin_bit_cast(uint2, y);
            O[db] = att_mfma<BF>(att_u4{xa.x, xa.y, ya.x, ya.y}, P[s], O[db]);
        }
    }
}

// the pieces that AttLoad::scan took out of a tile, for the rows that see their keys (bits of `wild`)
template <int D, bool BF, int NB>
__device__ __forceinline__ void att_wild_rows(const att_u4 (&P)[NB * 2], att_f16 (&O)[D / 32], const AttKeys &K, int u0, int p, uint64_t wild)
{
    const int lane = threadIdx.x & 63, col = lane & 31, hi = lane >> 5;
#pragma unroll 1
    for (; wild; wild &= wild - 1) {
        const int key = __builtin_ctzll(wild), u = u0 + key;
        uint32_t w = 0;
#pragma unroll
        for (int s = 0; s < NB * 2; ++s)
#pragma unroll
            for (int e = 0; e < 4; ++e)          // the word of P that holds keys (2e & 3) + 8 (e >> 1) + 4 hi (+1) of step s
                w = s * 16 + (e >> 1) * 8 + (e & 1) * 2 == (key & ~5) ? P[s][e] : w;
        w = (uint32_t)__shfl((int)w, col + 32 * (key >> 2 & 1), 64);
        const float pk = att_float<BF>(key & 1 ? w >> 16 : w & 0xffffu);
        const bool seen = AttSees(K, u0, p)(key);
        const uint16_t *row = u < K.n0 ? K.v0 + u * K.v0_r : K.v + (int64_t)(K.lo + u - K.n0) * K.v_r;
#pragma unroll
        for (int db = 0; db < D / 32; ++db)
#pragma unroll
            for (int e = 0; e < 16; e += 4) {    // dims 32 db + 2 e + 4 hi .. + 3: half of a piece
                const att_u4 x = *reinterpret_cast<const att_u4 *>(row + db * 32 + 2 * e);
                const bool add = seen & att_wild_piece<BF>(x);
                const uint32_t a = hi ? x[2] : x[0], b = hi ? x[3] : x[1];
                const float v[4] = {att_float<BF>(a & 0xffffu), att_float<BF>(a >> 16), att_float<BF>(b & 0xffffu), att_float<BF>(b >> 16)};
#pragma unroll
                for (int i = 0; i < 4; ++i) O[db][e + i] = add ? __builtin_fmaf(pk, v[i], O[db][e + i]) : O[db][e + i];
                __builtin_amdgcn_sched_barrier(0);   // (one piece at a time: this is rare, its registers are not)
            }
    }
}

// Those pieces, behind the loop over the tiles and only where one was taken out: the partly seen tiles once more, their weights from the final
// maximum.  In the loop its registers cost every call (8k tokens, window 4096: 256 dims 1.49 ms instead of 1.36, where O moved between the
// register files in every tile; 128 dims 0.444 instead of 0.429).
// NW = 4: the workgroup's tiles, 1: a wave's own.
template <int D, bool BF, int NB, int NW>
__device__ __forceinline__ void att_wild_tiles(const att_u4 (&Q)[D / 16], att_f16 (&O)[D / 32], const AttState &st, float c, const AttKeys &K, int u, int step,
                                               int p, uint16_t *ks, int w, unsigned long long *word)
{
    typedef AttLoad<D, NB, NW> Load;
    uint16_t *vs = ks + 32 * NB * D;
#pragma unroll 1
    for (; u < K.N; u += step) {
        if (K.lean(u)) continue;
        att_read_done();
        if (NW > 1) __syncthreads();
        if ((NW > 1 ? threadIdx.x : threadIdx.x & 63) == 0) *word = 0;
        Load::template issue<false>(K, u, ks, w);
        Load::template issue<true>(K, u, vs, w);
        att_landed<0>();
        if (NW > 1) __syncthreads();
        asm volatile("" ::: "memory");
        Load::template scan<BF>(vs, w, word);
        asm volatile("" ::: "memory");                       // (one wave's accesses to shared memory are in order)
        if (NW > 1) __syncthreads();
        const unsigned long long x = *word;
        const uint64_t wild = (uint64_t)att_uniform((uint32_t)(x >> 32)) << 32 | att_uniform((uint32_t)x);
        if (!wild) continue;
        att_f16 S[NB];
        att_u4 P[NB * 2];
        att_scores<D, BF, NB>(ks, Q, S);
        att_mask<NB>(S, K, u, p);
        att_weights<BF, NB>(S, P, st.m, c);
        att_wild_rows<D, BF, NB>(P, O, K, u, p, wild);
    }
}

__device__ __forceinline__ int att_len(const AttendArgs &A, int b)
{
    const int n = A.len ? A.len[(int64_t)b * A.len_step] : A.len_all;
    return max(min(n, A.rows - A.T), -A.T);                  // a full cache: the call's rows are its last ones; idle is idle
}

// Item of a workgroup: rows [row0, row0 + count) of request b's list (or of all requests' lists, packed) against keys [u_lo, u_hi)
struct AttItem { int b, hk, row0, slice, slot; bool packed; };

// Neighbouring workgroups go round the chip's eight dies: hand each die runs of `run` neighbouring items, so that the row tiles that read the
// same K / V meet in one L2 (a permutation of [0, n))
__device__ __forceinline__ int att_spread(int i, int n, int run)
{
    const int full = n / (8 * run) * (8 * run), j = i >> 3;
    return i < full ? (j / run * 8 + (i & 7)) * run + j % run : i;
}

template <int RWP, int RW> __device__ __forceinline__ AttItem att_item(const AttendArgs &A)
{
    AttItem it;
    int i = blockIdx.x;
    const int np = A.packed_tiles * A.packed_split * A.Hkv;
    it.packed = i < np;
    if (it.packed) {                                         // (tile fastest: the tiles of one slice share its keys)
        i = att_spread(i, np, max(1, np / 8));
        it.row0 = i % A.packed_tiles * (32 * RWP);
        i /= A.packed_tiles;
        it.slice = i % A.packed_split;
        it.hk = i / A.packed_split;
        it.b = 0;
        it.slot = it.slice;
        return it;
    }
    i = att_spread(i - np, gridDim.x - np, A.run);
    const int tile = i % A.tiles;
    i /= A.tiles;
    it.row0 = (A.tiles - 1 - tile) * (32 * RW);              // the tiles that see most first
    it.slice = i % A.split;
    i /= A.split;
    it.hk = i % A.Hkv;
    it.b = i / A.Hkv;
    it.slot = A.slot0 + it.slice;
    return it;
}

// An item, by four waves.  RW = 4: rows, RW = 1: keys (see above).  SAME: all rows see the same keys (one token per request, the prefix of a batch);
// what partly seen tiles need would cost a single token its registers at 256 dims (1.5 TB/s of the caches instead of 4.8).
template <int D, bool BF, int RW, bool SAME> __device__ __forceinline__ void att_item_body(const AttendArgs &A, const AttItem &it, uint16_t *smem)
{
    constexpr int NB = RW == 4 ? 2 : 1, KT = 32 * NB, KW = 4 / RW;
    constexpr int TILE = KT * D;                             // elements of a K (or V) tile
    __shared__ unsigned long long s_wild[4];                // keys whose V rows had a piece taken out: not 0 if any (keys: per wave)
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), col = lane & 31, hi = lane >> 5;
    const int TG = A.T * A.G, R = it.packed ? A.B * TG : TG;
    // ---- this lane's query row
    const int wrow0 = it.row0 + (RW == 4 ? w * 32 : 0);
    const int r = wrow0 + col, rr = r < R ? r : R - 1;
    const int b = it.packed ? rr / TG : it.b, tg = it.packed ? rr - b * TG : rr;
    const int t = tg / A.G, g = tg - t * A.G, h = it.hk * A.G + g;
    const int n = att_len(A, b);
    const int p = r < R ? n + t : -1;
    att_u4 Q[D / 16];
    {
        const uint16_t *qr = A.q + b * A.q_b + h * A.q_h + t * A.q_t + hi * 8;
#pragma unroll
        for (int s = 0; s < D / 16; ++s) Q[s] = *reinterpret_cast<const att_u4 *>(qr + s * 16);
    }
    // ---- the item's keys
    AttKeys K;
    int p_lo = 0, p_hi = 0, e_lo = 0, e_hi = 0;              // positions of this wave's rows, of the workgroup's
    K.k0_r = A.k0_r;
    K.v0_r = A.v0_r;
    K.k_r = A.k_r;
    K.v_r = A.v_r;
    K.window = A.window;
    K.sinks = A.sinks;
    if (it.packed) {
        K.n0 = K.N = A.prefix;
        K.lo = 0;
        K.k = K.v = nullptr;
        K.k0 = A.k0 + it.hk * A.k0_h;
        K.v0 = A.v0 + it.hk * A.v0_h;
    } else {
        const int n_ = att_len(A, it.b);                     // (uniform: this and what follows is scalar)
        e_lo = n_ + it.row0 / A.G;
        e_hi = n_ + (min(it.row0 + 32 * RW, R) - 1) / A.G;
        p_lo = n_ + wrow0 / A.G;
        p_hi = n_ + (min(wrow0 + 32, R) - 1) / A.G;
        K.lo = max(0, e_lo - A.window + 1);
        K.n0 = A.packed_tiles ? 0 : A.prefix ? A.prefix : min(A.sinks, K.lo);
        if (e_hi < 0) K.n0 = K.lo = 0;                       // rows that see nothing
        K.N = K.n0 + max(0, e_hi + 1 - K.lo);
        K.k0 = A.k0 + it.b * A.k0_b + it.hk * A.k0_h;
        K.v0 = A.v0 + it.b * A.v0_b + it.hk * A.v0_h;
        K.k = A.k + it.b * A.k_b + it.hk * A.k_h;
        K.v = A.v + it.b * A.v_b + it.hk * A.v_h;
    }
    int u_lo;                                                // this workgroup's share of the keys: u_lo .. K.N - 1
    {
        const int nsl = it.packed ? A.packed_split : A.split;
        const int all = (K.N + KT * KW - 1) / (KT * KW), per = (all + nsl - 1) / nsl;
        u_lo = min(K.N, it.slice * per * KT * KW);
        K.N = min(K.N, u_lo + per * KT * KW);
    }
    K.look(KT, A.near_rows, e_lo, e_hi);
    AttState st = {-INFINITY, 0.0f};
    att_f16 O[D / 32], S[NB];
    att_u4 P[NB * 2];
#pragma unroll
    for (int db = 0; db < D / 32; ++db)
#pragma unroll
        for (int e = 0; e < 16; ++e) O[db][e] = 0.0f;

    if (RW == 4) {
        typedef AttLoad<D, NB, 4> Load;
        const bool idle = wrow0 >= R;
        if (tid == 0) s_wild[0] = 0;
        if (u_lo < K.N) {
            Load::template issue<false>(K, u_lo, smem, w);
            Load::template issue<true>(K, u_lo, smem + TILE, w);
        }
        __syncthreads();
        att_landed<0>();
        bool lean = K.lean(u_lo);
        if (!SAME && u_lo < K.N && !lean) Load::template scan<BF>(smem + TILE, w, &s_wild[0]);
        __syncthreads();
        int at = 0;                                           // the tile's place in shared memory
        for (int u = u_lo; u < K.N; u += KT) {
            const uint16_t *cur = smem + at;
            uint16_t *nxt = smem + (at ^ 2 * TILE);
            const int un = u + KT;
            const bool more = un < K.N, next_lean = K.lean(un);
            if (more) {                                       // (the other buffer was last read before the barrier)
                Load::template issue<false>(K, un, nxt, w);
                Load::template issue<true>(K, un, nxt + TILE, w);
            }
            bool skip = idle;
            if (!lean && !it.packed && u >= K.n0) {           // a tile that none of this wave's rows sees
                const int j = K.lo + u - K.n0;
                skip = skip || j > p_hi || (j + KT - 1 <= p_lo - K.window && j >= K.sinks);
            }
            if (!skip) {
                att_scores<D, BF, NB>(cur, Q, S);
                att_softmax<D, BF, NB>(S, P, O, st, A.c, K, u, p, !lean);
                att_values<D, BF, NB>(cur + TILE, P, O);
            }
            att_landed<0>();
            if (!SAME && more && !next_lean) Load::template scan<BF>(nxt + TILE, w, &s_wild[0]);      // (a lane looks at what it brought itself)
            __syncthreads();
            at ^= 2 * TILE;
            lean = next_lean;
        }
        if (!SAME && s_wild[0]) att_wild_tiles<D, BF, NB, 4>(Q, O, st, A.c, K, u_lo, KT, p, smem, w, &s_wild[0]);
    } else {
        typedef AttLoad<D, NB, 1> Load;
        uint16_t *ks = smem + w * 2 * TILE, *vs = ks + TILE;
        int u = u_lo + w * KT;
        if (!SAME && lane == 0) s_wild[w] = 0;
        bool whole = K.whole(u);
        if (u < K.N) {
            Load::template issue<false>(K, u, ks, 0);
            Load::template issue<true>(K, u, vs, 0);
        }
        while (u < K.N) {
            const int un = u + KT * KW;
            const bool more = un < K.N, next_whole = more && K.whole(un), lean = K.lean(u);
            if (whole) att_landed<Load::CH>();               // (a whole tile's V is exactly CH loads behind its K)
            else att_landed<0>();
            att_scores<D, BF, NB>(ks, Q, S);
            att_read_done();
            if (more) Load::template issue<false>(K, un, ks, 0);
            att_softmax<D, BF, NB>(S, P, O, st, A.c, K, u, p, !lean);
            if (next_whole) att_landed<Load::CH>();
            else att_landed<0>();
            if (!SAME && !lean) {
                Load::template scan<BF>(vs, 0, &s_wild[w]);  // (one wave's accesses to shared memory are in order)
                asm volatile("" ::: "memory");
            }
            att_values<D, BF, NB>(vs, P, O);
            att_read_done();
            if (more) Load::template issue<true>(K, un, vs, 0);
            u = un;
            whole = next_whole;
        }
        if (!SAME && s_wild[w]) att_wild_tiles<D, BF, NB, 1>(Q, O, st, A.c, K, u_lo + w * KT, KT * KW, p, ks, 0, &s_wild[w]);
    }
    st.l = att_other_half_sum(st.l);

    if (RW == 4) {
        if (r >= R) return;
        if (A.slots) {
            const int64_t row = ((int64_t)b * A.H + h) * A.T + t;
            float *ml = A.part_ml + (row * A.slots + it.slot) * 2, *o = A.part_o + (row * A.slots + it.slot) * D;
            if (hi == 0) { ml[0] = st.m; ml[1] = p < 0 ? -1.0f : st.l; }           // -1: the row sees nothing
#pragma unroll
            for (int db = 0; db < D / 32; ++db)
#pragma unroll
                for (int e = 0; e < 16; e += 4)
                    *reinterpret_cast<float4 *>(o + db * 32 + 2 * e + 4 * hi) = make_float4(O[db][e], O[db][e + 1], O[db][e + 2], O[db][e + 3]);
        } else {
            const float inv = 1.0f / st.l;
            uint16_t *o = A.out + (((int64_t)b * A.T + t) * A.H + h) * D;
#pragma unroll
            for (int db = 0; db < D / 32; ++db)
#pragma unroll
                for (int e = 0; e < 16; e += 4) {
                    uint2 x = make_uint2(0, 0);
                    if (p >= 0) x = make_uint2(att_pack<BF>(O[db][e] * inv, O[db][e + 1] * inv), att_pack<BF>(O[db][e + 2] * inv, O[db][e + 3] * inv));
                    *reinterpret_cast<uint2 *>(o + db * 32 + 2 * e + 4 * hi) = x;
                }
        }
        return;
    }
    // ---- the four waves' states over their keys, joined: rows of O in shared memory (their pitch of D + 4 words spreads the 16-byte writes over
    // the banks), then a thread per four dims of a row
    __shared__ float s_ml[4][32][2];
    __syncthreads();                                         // nobody reads tiles any more
    float *so = reinterpret_cast<float *>(smem);
    if (r < R) {
        if (hi == 0) { s_ml[w][col][0] = st.m; s_ml[w][col][1] = p < 0 ? -1.0f : st.l; }
#pragma unroll
        for (int db = 0; db < D / 32; ++db)
#pragma unroll
            for (int e = 0; e < 16; e += 4)
                *reinterpret_cast<float4 *>(so + (w * 32 + col) * (D + 4) + db * 32 + 2 * e + 4 * hi) = make_float4(O[db][e], O[db][e + 1], O[db][e + 2], O[db][e + 3]);
    }
    __syncthreads();
    const int rows = min(32, R - it.row0);
    for (int i = tid; i < rows * (D / 4); i += ATT_THREADS) {
        const int k = i / (D / 4), d = i % (D / 4) * 4;
        const float M = fmaxf(fmaxf(s_ml[0][k][0], s_ml[1][k][0]), fmaxf(s_ml[2][k][0], s_ml[3][k][0]));
        float L = 0.0f, x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float f = att_weight(s_ml[j][k][0], M, A.c);
            const float4 y = *reinterpret_cast<const float4 *>(so + (j * 32 + k) * (D + 4) + d);
            L = __builtin_fmaf(s_ml[j][k][1], f, L);
            x[0] = __builtin_fmaf(y.x, f, x[0]); x[1] = __builtin_fmaf(y.y, f, x[1]); x[2] = __builtin_fmaf(y.z, f, x[2]); x[3] = __builtin_fmaf(y.w, f, x[3]);
        }
        const bool none = s_ml[0][k][1] < 0.0f;
        const int q = it.row0 + k, qb = it.packed ? q / TG : it.b, qtg = it.packed ? q - qb * TG : q, qt = qtg / A.G, qh = it.hk * A.G + qtg - qt * A.G;
        if (A.slots) {
            const int64_t row = ((int64_t)qb * A.H + qh) * A.T + qt;
            float *ml = A.part_ml + (row * A.slots + it.slot) * 2, *o = A.part_o + (row * A.slots + it.slot) * D;
            if (d == 0) { ml[0] = M; ml[1] = none ? -1.0f : L; }
            *reinterpret_cast<float4 *>(o + d) = make_float4(x[0], x[1], x[2], x[3]);
        } else {
            const float inv = 1.0f / L;
            uint2 y = make_uint2(0, 0);
            if (!none) y = make_uint2(att_pack<BF>(x[0] * inv, x[1] * inv), att_pack<BF>(x[2] * inv, x[3] * inv));
            *reinterpret_cast<uint2 *>(A.out + (((int64_t)qb * A.T + qt) * A.H + qh) * D + d) = y;
        }
    }
}

// RWP: shape of the items over all requests' rows (a shared prefix), RW: of the others
template <int D, bool BF, int RWP, int RW, bool ONE>
__global__ void __launch_bounds__(ATT_THREADS, D <= 128 ? 2 : 1) attend_kernel(const AttendArgs A)
{
    __shared__ __attribute__((aligned(16))) uint16_t smem[256 * D + 1024];         // tiles: 256 rows of D; the joined rows: 4 * 32 * (D + 4) floats
    const AttItem it = att_item<RWP, RW>(A);
    if (RWP == RW) att_item_body<D, BF, RW, ONE>(A, it, smem);
    else if (it.packed) att_item_body<D, BF, RWP, true>(A, it, smem);
    else att_item_body<D, BF, RW, ONE>(A, it, smem);
}

// The slices of a row, joined: out = sum 2^(c (m_i - M)) O_i / sum 2^(c (m_i - M)) l_i.  A thread has four dims of a row; SG threads share the
// slices of a row (8 where there are many: a few loads in flight each, instead of dozens one behind the other) and are added up in their
// order.  Then the lengths move on: the last reader of the old ones was the launch before.
template <int D, bool BF, int SG>
__global__ void __launch_bounds__(256) attend_join_kernel(const AttendArgs A, int64_t nrows, int advance, int32_t *len, uint32_t *host_flag)
{
    constexpr int LPR = D / 4, ROWS = 256 / (LPR * SG) > 0 ? 256 / (LPR * SG) : 1;
    __shared__ float s_o[SG > 1 ? SG : 1][ROWS][SG > 1 ? D + 4 : 1], s_l[SG > 1 ? SG : 1][ROWS];
    const int tid = threadIdx.x, d = tid % LPR * 4, k = tid / LPR % ROWS, sg = tid / (LPR * ROWS);
    const int64_t row = (int64_t)blockIdx.x * ROWS + k;                        // (b * H + h) * T + t
    const bool mine = row < nrows && sg < SG;
    float M = -INFINITY, L = 0.0f, x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    bool none = false;
    if (mine) {
        const float2 *ml = reinterpret_cast<const float2 *>(A.part_ml) + row * A.slots;
        const float *po = A.part_o + row * A.slots * D + d;
#pragma unroll 8
        for (int i = 0; i < A.slots; ++i) {
            const float2 v = ml[i];
            M = fmaxf(M, v.x);
            none = none | (v.y < 0.0f);
        }
#pragma unroll 4
        for (int i = sg; i < A.slots; i += SG) {
            const float2 v = ml[i];
            const float4 y = *reinterpret_cast<const float4 *>(po + (int64_t)i * D);
            const float f = att_weight(v.x, M, A.c);
            L = __builtin_fmaf(v.y, f, L);
            x[0] = __builtin_fmaf(y.x, f, x[0]); x[1] = __builtin_fmaf(y.y, f, x[1]); x[2] = __builtin_fmaf(y.z, f, x[2]); x[3] = __builtin_fmaf(y.w, f, x[3]);
        }
    }
    if (SG > 1) {
        if (sg < SG) {
            *reinterpret_cast<float4 *>(&s_o[sg][k][d]) = make_float4(x[0], x[1], x[2], x[3]);
            if (d == 0) s_l[sg][k] = L;
        }
        __syncthreads();
        if (sg == 0) {
#pragma unroll
            for (int j = 1; j < SG; ++j) {
                const float4 y = *reinterpret_cast<const float4 *>(&s_o[j][k][d]);
                L += s_l[j][k];
                x[0] += y.x; x[1] += y.y; x[2] += y.z; x[3] += y.w;
            }
        }
    }
    if (mine && sg == 0) {
        const int64_t bh = row / A.T, t = row - bh * A.T, b = bh / A.H, h = bh - b * A.H;
        uint2 y = make_uint2(0, 0);
        if (!none) y = make_uint2(att_pack<BF>(x[0] / L, x[1] / L), att_pack<BF>(x[2] / L, x[3] / L));
        *reinterpret_cast<uint2 *>(A.out + ((b * A.T + t) * A.H + h) * D + d) = y;
    }
    if (advance && blockIdx.x == 0) {
        const int nlen = A.len_step ? A.B : 1;
        for (int i = tid; i < nlen; i += 256) {
            const int n = len[i];
            if (n < 0) continue;                                                // an idle request stays where it is
            len[i] = n <= A.rows - advance ? n + advance : A.rows;
            if (n > A.rows - advance && host_flag) __hip_atomic_store(host_flag + 1, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
        }
    }
}

// ---- how a call is cut.  Shared by the entry points and fastkv_attend_workspace_bytes.
struct AttPlan { int rwp, rw, packed_tiles, packed_split, tiles, split, slots; int64_t blocks; };

// Into how many slices the keys of `items` items (n keys each, `per` keys a step of the workgroup) are cut: the least of a plain sum of times in
// us, whose constants are measured -- what a workgroup takes for itself (2.5) and per step (rows: 1.55 for 128 x 64 at 128 dims alone on its
// compute unit, 2.0 each for two; keys: 1.0, and what the memory gives), and the join (3.5, and the slices' fp32 sums written and read).
// `beside`: the time of other items that run meanwhile; `took`, where given, gets that of these.
static int att_cut(int64_t items, int64_t n, int per, double step, double step2, int64_t rows, int D, int extra, double beside = 0.0,
                   double *took = nullptr)
{
    const int64_t steps = (n + per - 1) / per;
    // 256 dims: one workgroup per compute unit, 3.5 us a step (cut as if there were two: 2 x 512 tokens, window 4096 232 us, 207 so; 64 requests
    // behind 32768 rows 188, 167)
    const int at_once = D > 128 ? 256 : 512;
    int best = 1;
    double least = 1e30;
    for (int s : {1, 2, 3, 4, 6, 8, 12, 16, 24, 32, 48, 64}) {
        if (s > steps) break;
        const int64_t wgs = items * s, each = (steps + s - 1) / s;
        const int64_t full = wgs / at_once, rest = wgs % at_once;
        double t = (double)(full * (2.5 + each * (D > 128 ? step : step2))) + (rest ? 2.5 + each * (rest > 256 ? step2 : step) : 0.0);
        const double alone = t;
        if (t < beside) t = beside;
        if (s + extra > 1) t += 3.5 + rows * (s + extra) * (D + 2) * 8.0 / 4e6;
        if (t < least * 0.99) {
            least = t;
            best = s;
            if (took) *took = alone;
        }
    }
    return best;
}

// The keys that a tile of `n` rows can see at most, of a cache of `rows`: what a call is cut by (the lengths are on the device).  `sees`: what one
// query can; its tile's rows lie at n / G positions (counted with all T of them, 4189 tokens of a window of 67, 8 heads, were cut and joined for
// nothing: 37 us, 19 so).
static int64_t att_keys(int n, int G, int T, int rows, int64_t sees)
{
    const int64_t at = (n + G - 2) / G + 1, all = sees + (at < T ? at : T) - 1;
    return all < rows ? all : rows;
}

static AttPlan att_plan(int B, int H, int Hkv, int D, int T, int rows, int64_t sees, int64_t prefix, bool advance)
{
    AttPlan P = {};
    const int64_t TG = (int64_t)T * (H / Hkv), all = (int64_t)B * H * T;
    const double step = D > 128 ? 3.5 : D * 1.55 / 128, step2 = D * 2.0 / 128, kstep = D * 1.0 / 128;
    if (prefix > 0 && TG < 128 && B > 1) {                    // rows of all requests in one tile: the prefix is read once, not once per request
        const int64_t R = B * TG;
        // rows up to which the keys shape is taken.  Several tokens of 256 dims: 8 requests of 2 / 8 tokens behind 6553 rows 36.7 / 53 us without
        // it, 39.9 / 57 with it; not so where there is a window alone (2 requests of 2 / 8 tokens, window 4096: 35 / 38 us without, 26 / 28 with).
        const int few = T == 1 || D < 256 ? 32 : 0;
        P.rwp = R <= few ? 1 : 4;
        P.rw = TG <= few ? 1 : 4;
        P.packed_tiles = (int)((R + 32 * P.rwp - 1) / (32 * P.rwp));
        // The requests' own rows run beside the prefix: they are cut where they are long (4 requests of 8192 rows, 32 heads on 8, behind 512 shared
        // ones: 77 us in one piece each, 31 so; 2 of 16384, 16 heads on 2: 107 and 17), not where they take little longer
        // than the prefix does (8 of 512, 4 tokens each, behind 4096: 22.5 us whole, 24.0 cut).
        double prefix_takes = 0.0;
        P.packed_split = P.rwp == 1 ? att_cut((int64_t)Hkv * P.packed_tiles, prefix, 128, kstep, 2 * kstep, all, D, 1, 0.0, &prefix_takes)
                                    : att_cut((int64_t)Hkv * P.packed_tiles, prefix, 64, step, step2, all, D, 1, 0.0, &prefix_takes);
        P.tiles = (int)((TG + 32 * P.rw - 1) / (32 * P.rw));
        const double beside = prefix_takes * 1.25;
        const int64_t keys = att_keys(32 * P.rw, H / Hkv, T, rows, sees);
        P.split = P.rw == 1 ? att_cut((int64_t)B * Hkv * P.tiles, keys, 128, kstep, 2 * kstep, all, D, P.packed_split, beside)
                            : att_cut((int64_t)B * Hkv * P.tiles, keys, 64, step, step2, all, D, P.packed_split, beside);
        P.slots = P.packed_split + P.split;
        P.blocks = (int64_t)Hkv * P.packed_tiles * P.packed_split + (int64_t)B * Hkv * P.tiles * P.split;
        return P;
    }
    P.rwp = P.rw = TG <= 32 ? 1 : 4;
    const int per = 32 * P.rw;
    P.tiles = (int)((TG + per - 1) / per);
    const int64_t items = (int64_t)B * Hkv * P.tiles, keys = att_keys(per, H / Hkv, T, rows, sees);
    P.split = P.rw == 1 ? att_cut(items, keys + prefix, 128, kstep, 2 * kstep, all, D, advance ? 1 : 0)
                        : att_cut(items, keys + prefix, 64, step, step2, all, D, advance ? 1 : 0);
    P.slots = P.split > 1 || advance ? P.split : 0;
    P.blocks = items * P.split;
    return P;
}

// rows of a workgroup of the join: attend_join_kernel's ROWS
static int att_join_rows(int slots, int D) { return slots >= 8 ? 256 / (D * 2) + (D == 256) : 1024 / D; }

static size_t att_bytes(const AttPlan &P, int B, int H, int T, int D)
{
    return (size_t)B * H * T * P.slots * (D + 2) * sizeof(float);
}

template <int D, bool BF>
static int att_launch(AttendArgs &A, const AttPlan &P, int advance, int32_t *len, hipStream_t st)
{
    {
        ProfScope ps_(K_ATTEND, st);
        const dim3 grid((unsigned)P.blocks), block(ATT_THREADS);
        constexpr bool SEVERAL = D == 256;                    // (several tokens of 256 dims never have the two shapes side by side: att_plan)
        if (P.rwp == 1 && A.T == 1) hipLaunchKernelGGL((attend_kernel<D, BF, 1, 1, true>), grid, block, 0, st, A);
        else if (P.rwp == 1) hipLaunchKernelGGL((attend_kernel<D, BF, 1, 1, false>), grid, block, 0, st, A);
        else if (P.rw == 1 && A.T == 1) hipLaunchKernelGGL((attend_kernel<D, BF, 4, 1, true>), grid, block, 0, st, A);
        else if (P.rw == 1) hipLaunchKernelGGL((attend_kernel<D, BF, 4, 1, SEVERAL>), grid, block, 0, st, A);
        else hipLaunchKernelGGL((attend_kernel<D, BF, 4, 4, false>), grid, block, 0, st, A);
    }
    if (hipGetLastError() != hipSuccess) return FASTKV_ELAUNCH;
    if (!A.slots) return FASTKV_OK;
    const int64_t nrows = (int64_t)A.B * A.H * A.T;
    ProfScope ps_(K_ATTEND, st);
    const bool many = A.slots >= 8;
    const int per = att_join_rows(A.slots, D);
    const dim3 grid((unsigned)((nrows + per - 1) / per)), block(256);
    uint32_t *flag = advance ? abort_flag_device() : nullptr;
    if (many) hipLaunchKernelGGL((attend_join_kernel<D, BF, D == 256 ? 4 : 8>), grid, block, 0, st, A, nrows, advance ? A.T : 0, len, flag);
    else hipLaunchKernelGGL((attend_join_kernel<D, BF, 1>), grid, block, 0, st, A, nrows, advance ? A.T : 0, len, flag);
    return hipGetLastError() == hipSuccess ? FASTKV_OK : FASTKV_ELAUNCH;
}

static int att_run(AttendArgs &A, int dtype, int D, int advance, int32_t *len, void *workspace, size_t workspace_bytes, void *stream)
{
    const AttPlan P = att_plan(A.B, A.H, A.Hkv, D, A.T, A.rows, (int64_t)A.window + A.sinks, A.prefix, advance != 0);
    const int64_t join = P.slots ? ((int64_t)A.B * A.H * A.T + att_join_rows(P.slots, D) - 1) / att_join_rows(P.slots, D) : 0;
    if (P.blocks > 0xffffff || join > 0xffffff) return FASTKV_EUNSUPPORTED;                          // (launches of less than 2^32 threads)
    const size_t need = att_bytes(P, A.B, A.H, A.T, D);
    if (need && (!workspace || ((uintptr_t)workspace & 15))) return FASTKV_EINVAL;
    if (workspace_bytes < need) return FASTKV_EWORKSPACE;
    if (advance && !abort_flag_device()) return FASTKV_ELAUNCH;               // (no word to report a full cache in: nothing is launched that could not)
    A.G = A.H / A.Hkv;
    A.slots = P.slots;
    A.packed_tiles = P.packed_tiles;
    A.packed_split = P.packed_split;
    A.slot0 = P.packed_split;
    A.tiles = P.tiles;
    A.split = P.split;
    // One run per die where the KV heads divide over the dies.  Elsewhere a run would hold the row tiles that see most and another those that see
    // least (8192 tokens without a window, 16 heads on 2: 452 us so, 331 in runs of four; 8 on 1: 255 and 227).
    const int64_t own = P.blocks - (int64_t)A.Hkv * P.packed_tiles * P.packed_split;
    A.run = (int64_t)A.B * A.Hkv % 8 == 0 || own < 64 ? (int)(own / 8 > 1 ? own / 8 : 1) : 4;
    A.near_rows = true;
    for (int64_t r : {A.k_r, A.v_r, A.k0_r, A.v0_r}) A.near_rows = A.near_rows && r >= 0 && r < (int64_t)1 << 23;
    A.part_o = (float *)workspace;
    A.part_ml = A.part_o + (size_t)A.B * A.H * A.T * P.slots * D;
    hipStream_t st = (hipStream_t)stream;
    if (D == 64) return dtype ? att_launch<64, true>(A, P, advance, len, st) : att_launch<64, false>(A, P, advance, len, st);
    if (D == 128) return dtype ? att_launch<128, true>(A, P, advance, len, st) : att_launch<128, false>(A, P, advance, len, st);
    return dtype ? att_launch<256, true>(A, P, advance, len, st) : att_launch<256, false>(A, P, advance, len, st);
}

static bool att_shape_ok(int dtype, int B, int H, int Hkv, int D, int T, int rows)
{
    return (dtype == FASTKV_F16 || dtype == FASTKV_BF16) && B >= 1 && Hkv >= 1 && H >= Hkv && H % Hkv == 0 && T >= 1 && rows >= 1 &&
           (int64_t)B * H * T <= 0x7fffffff && rows <= 0x1fffffff && D >= 1;
}
// (scores are taken times scaling * log2(e), which has to be a number too)
static bool att_scaling_ok(float scaling) { return scaling > 0.0f && scaling * 1.44269504088896340736f < INFINITY; }
// 16-byte rows of [n0,n1,n2] or [n1,n2]; along an extent of one nothing is stepped, whatever stride the caller has for it: it becomes 0 in `to`
static bool att_rows_ok(const void *p, const int64_t *s, std::initializer_list<int> extents, std::initializer_list<int64_t *> to)
{
    if (!p || !s || ((uintptr_t)p & 15)) return false;
    auto t = to.begin();
    for (int n : extents) {
        if (n > 1 && (*s & 7)) return false;
        **t++ = n > 1 ? *s : 0;
        ++s;
    }
    return true;
}

}  // namespace fk

using namespace fk;

extern "C" {

size_t fastkv_attend_workspace_bytes(int32_t B, int32_t H, int32_t Hkv, int32_t D, int32_t T, int32_t rows, int32_t window, int32_t sinks,
                                     int32_t prefix, int32_t advance)
{
    if (!att_shape_ok(FASTKV_F16, B, H, Hkv, D, T, rows) || window < 0 || sinks < 0 || prefix < 0) return 0;
    const int64_t sees = (int64_t)(window && window < rows ? window : rows) + (sinks < rows ? sinks : rows);
    return att_bytes(att_plan(B, H, Hkv, D, T, rows, sees, prefix, advance != 0), B, H, T, D);
}

int fastkv_window_attention(int32_t dtype, int32_t B, int32_t H, int32_t Hkv, int32_t D, int32_t T, const void *q, const int64_t q_strides[3],
                            const void *k, const int64_t k_strides[3], const void *v, const int64_t v_strides[3], int32_t rows,
                            int32_t *len_dev, int32_t len_step, int32_t advance, int32_t window, int32_t sinks, float scaling, void *out,
                            void *workspace, size_t workspace_bytes, void *stream)
{
    if (!att_shape_ok(dtype, B, H, Hkv, D, T, rows)) return FASTKV_EINVAL;
    if (D != 64 && D != 128 && D != 256) return FASTKV_EUNSUPPORTED;
    AttendArgs A = {};
    if (!att_rows_ok(q, q_strides, {B, H, T}, {&A.q_b, &A.q_h, &A.q_t}) || !att_rows_ok(k, k_strides, {B, Hkv, rows}, {&A.k_b, &A.k_h, &A.k_r}) ||
        !att_rows_ok(v, v_strides, {B, Hkv, rows}, {&A.v_b, &A.v_h, &A.v_r}) || !out || ((uintptr_t)out & 15))
        return FASTKV_EINVAL;
    if (window < 0 || sinks < 0 || !att_scaling_ok(scaling) || len_step < 0 || len_step > 1 || (advance && !len_dev)) return FASTKV_EINVAL;
    A.q = (const uint16_t *)q;
    A.k = A.k0 = (const uint16_t *)k;
    A.k0_b = A.k_b; A.k0_h = A.k_h; A.k0_r = A.k_r;
    A.v = A.v0 = (const uint16_t *)v;
    A.v0_b = A.v_b; A.v0_h = A.v_h; A.v0_r = A.v_r;
    A.len = len_dev;
    A.len_step = len_step;
    A.len_all = rows - T;
    A.B = B; A.H = H; A.Hkv = Hkv; A.T = T; A.rows = rows;
    A.window = window && window < rows ? window : rows;       // p < rows: a window of `rows` sees everything in front of p
    A.sinks = sinks < rows ? sinks : rows;
    A.c = scaling * 1.44269504088896340736f;
    A.out = (uint16_t *)out;
    return att_run(A, dtype, D, advance, len_dev, workspace, workspace_bytes, stream);
}

int fastkv_shared_prefix_attention(int32_t dtype, int32_t B, int32_t H, int32_t Hkv, int32_t D, int32_t T, const void *q, const int64_t q_strides[3],
                                   const void *k_prefix, const int64_t kp_strides[2], const void *v_prefix, const int64_t vp_strides[2],
                                   int32_t prefix_rows, const void *k, const int64_t k_strides[3], const void *v, const int64_t v_strides[3],
                                   int32_t rows, int32_t *len_dev, int32_t len_step, int32_t advance, float scaling, void *out, void *workspace,
                                   size_t workspace_bytes, void *stream)
{
    if (!att_shape_ok(dtype, B, H, Hkv, D, T, rows) || prefix_rows < 1 || prefix_rows > 0x1fffffff) return FASTKV_EINVAL;
    if (D != 64 && D != 128 && D != 256) return FASTKV_EUNSUPPORTED;
    AttendArgs A = {};
    if (!att_rows_ok(q, q_strides, {B, H, T}, {&A.q_b, &A.q_h, &A.q_t}) || !att_rows_ok(k, k_strides, {B, Hkv, rows}, {&A.k_b, &A.k_h, &A.k_r}) ||
        !att_rows_ok(v, v_strides, {B, Hkv, rows}, {&A.v_b, &A.v_h, &A.v_r}) ||
        !att_rows_ok(k_prefix, kp_strides, {Hkv, prefix_rows}, {&A.k0_h, &A.k0_r}) ||
        !att_rows_ok(v_prefix, vp_strides, {Hkv, prefix_rows}, {&A.v0_h, &A.v0_r}) || !out || ((uintptr_t)out & 15))
        return FASTKV_EINVAL;
    if (!att_scaling_ok(scaling) || !len_dev || len_step < 0 || len_step > 1) return FASTKV_EINVAL;
    A.q = (const uint16_t *)q;
    A.k0 = (const uint16_t *)k_prefix;
    A.v0 = (const uint16_t *)v_prefix;
    A.k = (const uint16_t *)k;
    A.v = (const uint16_t *)v;
    A.len = len_dev;
    A.len_step = len_step;
    A.B = B; A.H = H; A.Hkv = Hkv; A.T = T; A.rows = rows;
    A.window = rows;
    A.prefix = prefix_rows;
    A.c = scaling * 1.44269504088896340736f;
    A.out = (uint16_t *)out;
    return att_run(A, dtype, D, advance, len_dev, workspace, workspace_bytes, stream);
}

}  // extern "C"
