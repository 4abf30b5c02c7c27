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
//   rows      4 x 32 rows, all waves on one 64-key tile (two tiles in shared memory, one barrier per tile)
//   keys      <= 32 rows (single tokens): each wave has its own 32-key tiles and running state, merged at the end; a wave's tile is
//             private, so the loop has no barrier and eight waves of a compute unit keep ~128 KB of loads in flight
// Work too small to fill the chip is cut along the keys; slices leave {m, l, O} in a workspace and attend_join adds them up.
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
// 16-byte piece c of row `row` lies at piece c ^ att_swz(row): eight consecutive rows' equal pieces (the K reads), and the piece pairs of
// four consecutive rows (the transposing V reads), fall on different banks
__device__ __forceinline__ int att_swz(int row) { return (row & 3) << 1 | (row >> 2 & 1); }

// what a partial sum over keys of maximum m counts for beside the maximum M of all of them (no key at all: both are -inf; a NaN among
// the sums survives a weight of zero, as it survives in the formula)
__device__ __forceinline__ float att_weight(float m, float M, float c) { return M == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f((m - M) * c); }

struct AttKeys {                             // the keys of one item, and which of them a row at position p sees
    const uint16_t *k0, *v0, *k, *v;
    int64_t k0_r, v0_r, k_r, v_r;
    int n0, lo, N;                           // segment 0; first row of segment 1; all
    int window, sinks;
    __device__ __forceinline__ bool sees(int u, int p) const
    {
        const int j = lo + u - n0;
        return u < N && (u < n0 || (j <= p && (j > p - window || j < sinks)));
    }
};

struct AttState { float m, l; };

// One tile of 32*NB keys, u0 .. : `ks`, `vs` the tile in shared memory; Q the wave's 32 query rows; `edge`: some row may not see some
// key of the tile; `wild`: keys of the tile (bits) whose V row holds an infinity or NaN, given for edge tiles only -- a row that does not see
// such a key must not be touched by it (0 * inf), so these keys are taken out of the product and added for the rows that see them.
template <int D, bool BF, int NB>
__device__ __forceinline__ void att_tile(const uint16_t *ks, const uint16_t *vs, const att_u4 (&Q)[D / 16], att_f16 (&O)[D / 32], AttState &st,
                                         float c, const AttKeys &K, int u0, int p, bool edge, uint64_t wild)
{
    const int lane = threadIdx.x & 63, col = lane & 31, hi = lane >> 5;
    att_f16 S[NB];
#pragma unroll
    for (int kb = 0; kb < NB; ++kb) {
#pragma unroll
        for (int r = 0; r < 16; ++r) S[kb][r] = 0.0f;
    }
    const int swk = att_swz(col);
#pragma unroll
    for (int s = 0; s < D / 16; ++s) {
#pragma unroll
        for (int kb = 0; kb < NB; ++kb) {
            const att_u4 a = *reinterpret_cast<const att_u4 *>(ks + (kb * 32 + col) * D + ((2 * s + hi) ^ swk) * 8);
            S[kb] = att_mfma<BF>(a, Q[s], S[kb]);
        }
    }
    if (edge) {
#pragma unroll
        for (int kb = 0; kb < NB; ++kb)
#pragma unroll
            for (int r = 0; r < 16; ++r)
                if (!K.sees(u0 + kb * 32 + (r & 3) + 8 * (r >> 2) + 4 * hi, p)) S[kb][r] = -INFINITY;
    }
    float tm = -INFINITY;
#pragma unroll
    for (int kb = 0; kb < NB; ++kb)
#pragma unroll
        for (int r = 0; r < 16; ++r) tm = fmaxf(tm, S[kb][r]);
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
    const float mc = (st.m == -INFINITY ? 0.0f : st.m * c) - (BF ? 0.0f : ATT_LIFT);
    att_u4 P[NB * 2];
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
    st.l += l0 + l1;
    // lane i of a group of 16 addresses row i / 4, elements 4 * (i % 4) of a 4 x 16 block and receives column i
    const int gi = lane & 15, dsub = (lane >> 4 & 1) * 16 + (gi & 3) * 4, krow = gi >> 2;
#pragma unroll
    for (int s = 0; s < NB * 2; ++s) {
        const int r0 = s * 16 + 4 * hi + krow, r1 = r0 + 8;
        const uint16_t *v0 = vs + r0 * D, *v1 = vs + r1 * D;
        const int w0 = att_swz(r0), w1 = att_swz(r1);
        const uint32_t cut = edge ? (uint32_t)(wild >> (s * 16 + 4 * hi)) : 0u;
#pragma unroll
        for (int db = 0; db < D / 32; ++db) {
            const int d = db * 32 + dsub;
            typedef __attribute__((address_space(3))) att_s4 lds_s4;
            const att_s4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4 *)(v0 + ((d >> 3) ^ w0) * 8 + (d & 7)));
            const att_s4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4 *)(v1 + ((d >> 3) ^ w1) * 8 + (d & 7)));
            const uint2 xa = __builtin_bit_cast(uint2, x), ya = __builtin_bit_cast(uint2, y);
            att_u4 a = {xa.x, xa.y, ya.x, ya.y};
            if (edge && wild) {
                const uint32_t b = (cut & 0xfu) | (cut >> 4 & 0xf0u);
#pragma unroll
                for (int e = 0; e < 4; ++e) a[e] &= (b >> (2 * e) & 1 ? 0u : 0xffffu) | (b >> (2 * e + 1) & 1 ? 0u : 0xffff0000u);
            }
            O[db] = att_mfma<BF>(a, P[s], O[db]);
        }
    }
    if (edge && wild) {
        for (uint64_t left = wild; left; left &= left - 1) {
            const int key = __builtin_ctzll(left);
            uint32_t w = 0;
#pragma unroll
            for (int s = 0; s < NB * 2; ++s)
#pragma unroll
                for (int e = 0; e < 4; ++e)      // the word of P that holds keys (2e & 3) + 8 (e >> 1) + 4 hi (+1) of step s
                    w = s * 16 + (e >> 1) * 8 + (e & 1) * 2 == (key & ~5) ? P[s][e] : w;
            w = (uint32_t)__shfl((int)w, col + 32 * (key >> 2 & 1), 64);
            const float pk = att_float<BF>(key & 1 ? w >> 16 : w & 0xffffu);
            const bool seen = K.sees(u0 + key, p);
#pragma unroll
            for (int db = 0; db < D / 32; ++db)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int d = db * 32 + (r & 3) + 8 * (r >> 2) + 4 * hi;
                    const float x = att_float<BF>(vs[key * D + ((d >> 3) ^ att_swz(key)) * 8 + (d & 7)]);
                    if (seen) O[db][r] = __builtin_fmaf(pk, x, O[db][r]);
                }
        }
    }
}

// Registers of a tile on its way to shared memory: NT threads, 32*NB rows of K and V, CH pieces each per thread
template <int D, int NB, int NT> struct AttStage {
    static constexpr int C = D / 8, CH = 32 * NB * C / NT;
    att_u4 k[CH], v[CH];
    __device__ __forceinline__ void fetch(const AttKeys &K, int u0, int tid)
    {
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            const int id = i * NT + tid, u = u0 + id / C, e = id % C * 8;
            const att_u4 z = {0, 0, 0, 0};
            k[i] = v[i] = z;                 // behind the last key: zeros (their scores are cut off, their V rows must be finite)
            if (u < K.N) {
                const bool first = u < K.n0;
                const int64_t j = first ? u : K.lo + u - K.n0;
                k[i] = *reinterpret_cast<const att_u4 *>((first ? K.k0 : K.k) + j * (first ? K.k0_r : K.k_r) + e);
                v[i] = *reinterpret_cast<const att_u4 *>((first ? K.v0 : K.v) + j * (first ? K.v0_r : K.v_r) + e);
            }
        }
    }
    template <bool BF> __device__ __forceinline__ void commit(uint16_t *ks, uint16_t *vs, int tid, bool edge, unsigned long long *wild)
    {
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            const int id = i * NT + tid, row = id / C, c = (id % C) ^ att_swz(row);
            *reinterpret_cast<att_u4 *>(ks + row * D + c * 8) = k[i];
            *reinterpret_cast<att_u4 *>(vs + row * D + c * 8) = v[i];
            if (edge && (att_wild<BF>(v[i][0]) || att_wild<BF>(v[i][1]) || att_wild<BF>(v[i][2]) || att_wild<BF>(v[i][3])))
                atomicOr(wild, 1ull << row);
        }
    }
};

__device__ __forceinline__ int att_len(const AttendArgs &A, int b)
{
    const int n = A.len ? A.len[(int64_t)b * A.len_step] : A.len_all;
    return n < A.rows - A.T ? n : A.rows - A.T;              // a full cache: the call's rows are its last ones
}

// Item of a workgroup: rows [row0, row0 + count) of request b's list (or of all requests' lists, packed) against keys [u_lo, u_hi)
struct AttItem { int b, hk, row0, slice, slot; bool packed; };

// Neighbouring workgroups go round the chip's eight dies: hand each die a run of neighbouring items, so that the row tiles that read the
// same K / V meet in one L2 (a permutation of [0, n))
__device__ __forceinline__ int att_spread(int i, int n)
{
    const int per = n / 8, full = per * 8;
    return i < full ? (i & 7) * per + (i >> 3) : i;
}

template <int RW> __device__ __forceinline__ AttItem att_item(const AttendArgs &A)
{
    AttItem it;
    int i = blockIdx.x;
    const int np = A.packed_tiles * A.packed_split * A.Hkv;
    it.packed = i < np;
    if (it.packed) {                                         // (tile fastest: the tiles of one slice share its keys)
        i = att_spread(i, np);
        it.row0 = i % A.packed_tiles * (32 * RW);
        i /= A.packed_tiles;
        it.slice = i % A.packed_split;
        it.hk = i / A.packed_split;
        it.b = 0;
        it.slot = it.slice;
        return it;
    }
    i = att_spread(i - np, gridDim.x - np);
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

// RW = 4: rows, RW = 1: keys (see above)
template <int D, bool BF, int RW>
__global__ void __launch_bounds__(ATT_THREADS) attend_kernel(const AttendArgs A)
{
    constexpr int NB = RW == 4 ? 2 : 1, KT = 32 * NB, KW = 4 / RW;
    constexpr int TILE = KT * D;                             // elements of a K (or V) tile
    constexpr int NBUF = RW == 4 ? 2 : 4;                    // two tiles of the workgroup | one tile of each wave
    __shared__ __attribute__((aligned(16))) uint16_t smem[NBUF * 2 * TILE];
    __shared__ unsigned long long s_wild[RW == 4 ? 3 : 4];
    __shared__ float s_ml[KW][32][2];
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, col = lane & 31, hi = lane >> 5;
    const AttItem it = att_item<RW>(A);
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
    int p_lo = 0, p_hi = 0;                                  // positions of this wave's rows
    int u_lo, u_hi;                                          // this workgroup's share of them
    if (it.packed) {
        K.n0 = K.N = A.prefix;
        K.lo = 0;
        K.window = K.sinks = 0;
        K.k = K.v = nullptr;
        K.k_r = K.v_r = 0;
        K.k0 = A.k0 + it.hk * A.k0_h;
        K.v0 = A.v0 + it.hk * A.v0_h;
    } else {
        const int last = min(it.row0 + 32 * RW, R) - 1;
        const int pa = n + it.row0 / A.G, pb = n + last / A.G;                 // positions of the workgroup's rows
        K.window = A.window;
        K.sinks = A.sinks;
        K.lo = max(0, pa - A.window + 1);
        K.n0 = A.packed_tiles ? 0 : A.prefix ? A.prefix : min(A.sinks, K.lo);
        if (pb < 0) K.n0 = K.lo = 0;                         // rows that see nothing
        K.N = K.n0 + max(0, pb + 1 - K.lo);
        K.k0 = A.k0 + it.b * A.k0_b + it.hk * A.k0_h;
        K.v0 = A.v0 + it.b * A.v0_b + it.hk * A.v0_h;
        K.k = A.k + it.b * A.k_b + it.hk * A.k_h;
        K.v = A.v + it.b * A.v_b + it.hk * A.v_h;
        K.k_r = A.k_r;
        K.v_r = A.v_r;
        p_lo = n + wrow0 / A.G;
        p_hi = n + (min(wrow0 + 32, R) - 1) / A.G;
    }
    K.k0_r = A.k0_r;
    K.v0_r = A.v0_r;
    const int nsl = it.packed ? A.packed_split : A.split;
    {
        const int all = (K.N + KT * KW - 1) / (KT * KW), per = (all + nsl - 1) / nsl;
        u_lo = min(K.N, it.slice * per * KT * KW);
        u_hi = min(K.N, u_lo + per * KT * KW);
        K.N = u_hi;                                          // keys behind the share are no keys
    }
    // what a tile at u needs of this wave (positions of its rows: p_lo .. p_hi)
    auto edge_at = [&](int u, int a, int z) {                // rows at positions a .. z: not every row sees every key
        if (u + KT > K.N) return true;
        if (u + KT <= K.n0) return false;
        if (u < K.n0) return true;
        const int j = K.lo + u - K.n0;
        return j + KT - 1 > a || j <= z - K.window;
    };
    const bool idle_wave = wrow0 >= R;
    const int e_lo = RW == 4 && !it.packed ? n + it.row0 / A.G : p_lo, e_hi = RW == 4 && !it.packed ? n + (min(it.row0 + 32 * RW, R) - 1) / A.G : p_hi;
    AttState st = {-INFINITY, 0.0f};
    att_f16 O[D / 32];
#pragma unroll
    for (int db = 0; db < D / 32; ++db)
#pragma unroll
        for (int e = 0; e < 16; ++e) O[db][e] = 0.0f;

    if (RW == 4) {
        AttStage<D, NB, ATT_THREADS> sg;
        if (tid < 3) s_wild[tid] = 0;
        __syncthreads();
        const int nt = (u_hi - u_lo + KT - 1) / KT;
        if (nt > 0) {
            sg.fetch(K, u_lo, tid);
            sg.template commit<BF>(smem, smem + TILE, tid, edge_at(u_lo, e_lo, e_hi), &s_wild[0]);
        }
        __syncthreads();
        for (int i = 0; i < nt; ++i) {
            const int u = u_lo + i * KT, cur = i & 1;
            if (i + 1 < nt) sg.fetch(K, u + KT, tid);
            bool skip = idle_wave;
            if (!it.packed && u >= K.n0) {                    // a tile that none of this wave's rows sees
                const int j = K.lo + u - K.n0;
                skip = skip || j > p_hi || (j + KT - 1 <= p_lo - K.window && j >= K.sinks);
            }
            if (!skip)
                att_tile<D, BF, NB>(smem + cur * 2 * TILE, smem + cur * 2 * TILE + TILE, Q, O, st, A.c, K, u, p, edge_at(u, p_lo, p_hi),
                                    s_wild[i % 3]);
            if (i + 1 < nt)
                sg.template commit<BF>(smem + (cur ^ 1) * 2 * TILE, smem + (cur ^ 1) * 2 * TILE + TILE, tid, edge_at(u + KT, e_lo, e_hi),
                                       &s_wild[(i + 1) % 3]);
            if (tid == 0) s_wild[(i + 2) % 3] = 0;           // last read a tile ago, written a tile from now
            __syncthreads();
        }
    } else {
        AttStage<D, NB, 64> sg;
        uint16_t *ks = smem + w * 2 * TILE, *vs = ks + TILE;
        int u = u_lo + w * KT;
        if (u < u_hi) sg.fetch(K, u, lane);
        for (; u < u_hi; u += KT * KW) {
            const bool edge = edge_at(u, p_lo, p_hi);
            if (lane == 0) s_wild[w] = 0;
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
            sg.template commit<BF>(ks, vs, lane, edge, &s_wild[w]);
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
            if (u + KT * KW < u_hi) sg.fetch(K, u + KT * KW, lane);
            att_tile<D, BF, NB>(ks, vs, Q, O, st, A.c, K, u, p, edge, s_wild[w]);
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
        }
    }
    st.l = att_other_half_sum(st.l);

    // ---- the waves' states over their keys, joined
    if (KW > 1) {
        if (hi == 0) { s_ml[w][col][0] = st.m; s_ml[w][col][1] = st.l; }
        __syncthreads();                                     // (also: nobody reads tiles any more)
        float M = -INFINITY;
#pragma unroll
        for (int i = 0; i < KW; ++i) M = fmaxf(M, s_ml[i][col][0]);
        float L = 0.0f;
#pragma unroll
        for (int i = 0; i < KW; ++i) L += s_ml[i][col][1] * att_weight(s_ml[i][col][0], M, A.c);
        const float f = att_weight(st.m, M, A.c);
        st.m = M;
        st.l = L;
        // wave w adds up dims [w*D/4, +D/4): every wave leaves its O in shared memory, 32 dims at a time
        float *so = reinterpret_cast<float *>(smem);         // [4 waves][32 rows][32 dims + 1]
        constexpr int DQ = D / 32;
#pragma unroll
        for (int db = 0; db < DQ; ++db) {
#pragma unroll
            for (int e = 0; e < 16; ++e) so[(w * 32 + col) * 33 + (e & 3) + 8 * (e >> 2) + 4 * hi] = O[db][e] * f;
            __syncthreads();
            if (w == 0) {
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const int at = col * 33 + (e & 3) + 8 * (e >> 2) + 4 * hi;
                    O[db][e] = (so[at] + so[at + 32 * 33]) + (so[at + 64 * 33] + so[at + 96 * 33]);
                }
            }
            __syncthreads();
        }
        if (w != 0) return;
    }

    // ---- out
    if (r >= R) return;
    if (A.slots) {
        const int64_t row = ((int64_t)b * A.H + h) * A.T + t;
        float *ml = A.part_ml + (row * A.slots + it.slot) * 2, *o = A.part_o + (row * A.slots + it.slot) * D;
        if (hi == 0) { ml[0] = st.m; ml[1] = n + t < 0 ? -1.0f : st.l; }       // -1: the row sees nothing
#pragma unroll
        for (int db = 0; db < D / 32; ++db)
#pragma unroll
            for (int e = 0; e < 16; e += 4)
                *reinterpret_cast<float4 *>(o + db * 32 + 2 * e + 4 * hi) = make_float4(O[db][e], O[db][e + 1], O[db][e + 2], O[db][e + 3]);
    } else {
        const float inv = p < 0 ? 0.0f : 1.0f / st.l;
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
}

// The slices of a row, joined: out = sum 2^(c (m_i - M)) O_i / sum 2^(c (m_i - M)) l_i.  A wave per row, D / 64 dims per lane; then the lengths
// move on (the last reader of the old ones is behind this launch's start).
template <int D, bool BF>
__global__ void __launch_bounds__(256) attend_join_kernel(const AttendArgs A, int64_t nrows, int advance, int32_t *len, uint32_t *host_flag)
{
    constexpr int E = D / 64;
    const int lane = threadIdx.x & 63;
    const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);          // (b * H + h) * T + t
    if (row < nrows) {
        const float *ml = A.part_ml + row * A.slots * 2, *po = A.part_o + row * A.slots * D + lane * E;
        float M = -INFINITY;
        bool none = false;
        for (int i = lane; i < A.slots; i += 64) {
            M = fmaxf(M, ml[2 * i]);
            none = none || ml[2 * i + 1] < 0.0f;
        }
        M = wave_max(M);
        none = __any(none);
        float L = 0.0f, o[E];
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = 0.0f;
        for (int i = 0; i < A.slots; ++i) {
            const float m = ml[2 * i], f = att_weight(m, M, A.c);
            L += f * ml[2 * i + 1];
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const float x = po[(int64_t)i * D + e];
                o[e] = __builtin_fmaf(f, x, o[e]);
            }
        }
        const int64_t bh = row / A.T, t = row - bh * A.T, b = bh / A.H, h = bh - b * A.H;
        uint16_t *out = A.out + ((b * A.T + t) * A.H + h) * D + lane * E;
#pragma unroll
        for (int e = 0; e < E; ++e) out[e] = none ? 0 : (uint16_t)(att_pack<BF>(o[e] / L, 0.0f) & 0xffffu);
    }
    if (advance && blockIdx.x == 0) {
        const int nlen = A.len_step ? A.B : 1;
        for (int i = threadIdx.x; i < nlen; i += 256) {
            const int n = len[i];
            if (n < 0) continue;                                                // an idle request stays where it is
            len[i] = n <= A.rows - advance ? n + advance : A.rows;
            if (n > A.rows - advance && host_flag) __hip_atomic_store(host_flag + 1, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
        }
    }
}

// ---- how a call is cut.  Shared by the entry points and fastkv_attend_workspace_bytes.
struct AttPlan { int rw, packed_tiles, packed_split, tiles, split, slots; int64_t blocks; };

static AttPlan att_plan(int B, int H, int Hkv, int T, int64_t keys, int64_t prefix, bool advance)
{
    AttPlan P = {};
    const int64_t TG = (int64_t)T * (H / Hkv);
    const int64_t want = 512;                                 // workgroups: two per compute unit
    auto cut = [&](int64_t items, int64_t n, int64_t least) { // slices of n keys: enough to fill the chip, none shorter than `least`
        int64_t s = (want + items - 1) / items;
        const int64_t most = (n + least - 1) / least;
        s = s < most ? s : most;
        return (int)(s < 1 ? 1 : s > 64 ? 64 : s);
    };
    if (prefix > 0 && TG < 128 && B > 1) {                    // rows of all requests in one tile: the prefix is read once, not once per request
        const int64_t R = B * TG;
        P.rw = R <= 32 ? 1 : 4;
        const int per = 32 * P.rw;
        P.packed_tiles = (int)((R + per - 1) / per);
        P.packed_split = cut((int64_t)Hkv * P.packed_tiles, prefix, P.rw == 1 ? 128 : 64);
        P.tiles = (int)((TG + per - 1) / per);
        P.split = 1;
        P.slots = P.packed_split + 1;
        P.blocks = (int64_t)Hkv * P.packed_tiles * P.packed_split + (int64_t)B * Hkv * P.tiles;
        return P;
    }
    P.rw = TG <= 32 ? 1 : 4;
    const int per = 32 * P.rw;
    P.tiles = (int)((TG + per - 1) / per);
    P.split = cut((int64_t)B * Hkv * P.tiles, keys + prefix, P.rw == 1 ? 128 : 64);
    P.slots = P.split > 1 || advance ? P.split : 0;
    P.blocks = (int64_t)B * Hkv * P.tiles * P.split;
    return P;
}

static size_t att_bytes(const AttPlan &P, int B, int H, int T, int D)
{
    return (size_t)B * H * T * P.slots * (D + 2) * sizeof(float);
}

// rows that one query row can see at most: what a call is cut by (the lengths are on the device)
static int64_t att_keys(int T, int rows, int64_t window, int sinks)
{
    const int64_t w = window + sinks + T - 1;
    return w < rows ? w : rows;
}

template <int D, bool BF>
static int att_launch(AttendArgs &A, const AttPlan &P, int advance, int32_t *len, hipStream_t st)
{
    {
        ProfScope ps_(K_ATTEND, st);
        if (P.rw == 1) hipLaunchKernelGGL((attend_kernel<D, BF, 1>), dim3((unsigned)P.blocks), dim3(ATT_THREADS), 0, st, A);
        else hipLaunchKernelGGL((attend_kernel<D, BF, 4>), dim3((unsigned)P.blocks), dim3(ATT_THREADS), 0, st, A);
    }
    if (hipGetLastError() != hipSuccess) return FASTKV_ELAUNCH;
    if (!A.slots) return FASTKV_OK;
    const int64_t nrows = (int64_t)A.B * A.H * A.T;
    ProfScope ps_(K_ATTEND, st);
    hipLaunchKernelGGL((attend_join_kernel<D, BF>), dim3((unsigned)((nrows + 3) / 4)), dim3(256), 0, st, A, nrows, advance ? A.T : 0, len,
                       advance ? abort_flag_device() : nullptr);
    return hipGetLastError() == hipSuccess ? FASTKV_OK : FASTKV_ELAUNCH;
}

static int att_run(AttendArgs &A, int dtype, int D, int64_t keys, int advance, int32_t *len, void *workspace, size_t workspace_bytes, void *stream)
{
    const AttPlan P = att_plan(A.B, A.H, A.Hkv, A.T, keys, A.prefix, advance != 0);
    if (P.blocks > 0x7fffffff) return FASTKV_EUNSUPPORTED;
    const size_t need = att_bytes(P, A.B, A.H, A.T, D);
    if (need && (!workspace || ((uintptr_t)workspace & 15))) return FASTKV_EINVAL;
    if (workspace_bytes < need) return FASTKV_EWORKSPACE;
    A.G = A.H / A.Hkv;
    A.slots = P.slots;
    A.packed_tiles = P.packed_tiles;
    A.packed_split = P.packed_split;
    A.slot0 = P.packed_split;
    A.tiles = P.tiles;
    A.split = P.split;
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
           (int64_t)B * H * T <= 0x7fffffff && rows <= 0x3fffffff && D >= 1;
}
static bool att_rows_ok(const void *p, const int64_t *s, int n)                  // 16-byte rows
{
    if (!p || !s || ((uintptr_t)p & 15)) return false;
    for (int i = 0; i < n; ++i) if (s[i] & 7) return false;
    return true;
}

}  // namespace fk

using namespace fk;

extern "C" {

size_t fastkv_attend_workspace_bytes(int32_t B, int32_t H, int32_t Hkv, int32_t D, int32_t T, int32_t rows, int32_t window, int32_t sinks,
                                     int32_t prefix, int32_t advance)
{
    if (!att_shape_ok(FASTKV_F16, B, H, Hkv, D, T, rows) || window < 0 || sinks < 0 || prefix < 0) return 0;
    return att_bytes(att_plan(B, H, Hkv, T, att_keys(T, rows, window ? window : rows, sinks), prefix, advance != 0), B, H, T, D);
}

int fastkv_window_attention(int32_t dtype, int32_t B, int32_t H, int32_t Hkv, int32_t D, int32_t T, const void *q, const int64_t q_strides[3],
                            const void *k, const int64_t k_strides[3], const void *v, const int64_t v_strides[3], int32_t rows,
                            int32_t *len_dev, int32_t len_step, int32_t advance, int32_t window, int32_t sinks, float scaling, void *out,
                            void *workspace, size_t workspace_bytes, void *stream)
{
    if (!att_shape_ok(dtype, B, H, Hkv, D, T, rows)) return FASTKV_EINVAL;
    if (D != 64 && D != 128 && D != 256) return FASTKV_EUNSUPPORTED;
    if (!att_rows_ok(q, q_strides, 3) || !att_rows_ok(k, k_strides, 3) || !att_rows_ok(v, v_strides, 3) || !out || ((uintptr_t)out & 15)) return FASTKV_EINVAL;
    if (window < 0 || sinks < 0 || !(scaling > 0.0f) || scaling > 3.0e38f || len_step < 0 || len_step > 1 || (advance && !len_dev)) return FASTKV_EINVAL;
    AttendArgs A = {};
    A.q = (const uint16_t *)q;
    A.q_b = q_strides[0]; A.q_h = q_strides[1]; A.q_t = q_strides[2];
    A.k = A.k0 = (const uint16_t *)k;
    A.k_b = A.k0_b = k_strides[0]; A.k_h = A.k0_h = k_strides[1]; A.k_r = A.k0_r = k_strides[2];
    A.v = A.v0 = (const uint16_t *)v;
    A.v_b = A.v0_b = v_strides[0]; A.v_h = A.v0_h = v_strides[1]; A.v_r = A.v0_r = v_strides[2];
    A.len = len_dev;
    A.len_step = len_step;
    A.len_all = rows - T;
    A.B = B; A.H = H; A.Hkv = Hkv; A.T = T; A.rows = rows;
    A.window = window && window < rows ? window : rows;       // p < rows: a window of `rows` sees everything in front of p
    A.sinks = sinks < rows ? sinks : rows;
    A.c = scaling * 1.44269504088896340736f;
    A.out = (uint16_t *)out;
    return att_run(A, dtype, D, att_keys(T, rows, A.window, A.sinks), advance, len_dev, workspace, workspace_bytes, stream);
}

int fastkv_shared_prefix_attention(int32_t dtype, int32_t B, int32_t H, int32_t Hkv, int32_t D, int32_t T, const void *q, const int64_t q_strides[3],
                                   const void *k_prefix, const int64_t kp_strides[2], const void *v_prefix, const int64_t vp_strides[2],
                                   int32_t prefix_rows, const void *k, const int64_t k_strides[3], const void *v, const int64_t v_strides[3],
                                   int32_t rows, int32_t *len_dev, int32_t len_step, int32_t advance, float scaling, void *out, void *workspace,
                                   size_t workspace_bytes, void *stream)
{
    if (!att_shape_ok(dtype, B, H, Hkv, D, T, rows) || prefix_rows < 1 || prefix_rows > 0x3fffffff) return FASTKV_EINVAL;
    if (D != 64 && D != 128 && D != 256) return FASTKV_EUNSUPPORTED;
    if (!att_rows_ok(q, q_strides, 3) || !att_rows_ok(k, k_strides, 3) || !att_rows_ok(v, v_strides, 3) || !att_rows_ok(k_prefix, kp_strides, 2) ||
        !att_rows_ok(v_prefix, vp_strides, 2) || !out || ((uintptr_t)out & 15))
        return FASTKV_EINVAL;
    if (!(scaling > 0.0f) || scaling > 3.0e38f || !len_dev || len_step < 0 || len_step > 1) return FASTKV_EINVAL;
    AttendArgs A = {};
    A.q = (const uint16_t *)q;
    A.q_b = q_strides[0]; A.q_h = q_strides[1]; A.q_t = q_strides[2];
    A.k0 = (const uint16_t *)k_prefix;
    A.k0_h = kp_strides[0]; A.k0_r = kp_strides[1];
    A.v0 = (const uint16_t *)v_prefix;
    A.v0_h = vp_strides[0]; A.v0_r = vp_strides[1];
    A.k = (const uint16_t *)k;
    A.k_b = k_strides[0]; A.k_h = k_strides[1]; A.k_r = k_strides[2];
    A.v = (const uint16_t *)v;
    A.v_b = v_strides[0]; A.v_h = v_strides[1]; A.v_r = v_strides[2];
    A.len = len_dev;
    A.len_step = len_step;
    A.B = B; A.H = H; A.Hkv = Hkv; A.T = T; A.rows = rows;
    A.window = rows;
    A.prefix = prefix_rows;
    A.c = scaling * 1.44269504088896340736f;
    A.out = (uint16_t *)out;
    return att_run(A, dtype, D, rows, advance, len_dev, workspace, workspace_bytes, stream);
}

}  // extern "C"
