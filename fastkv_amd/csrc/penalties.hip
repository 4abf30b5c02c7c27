// Penalties, biases and masks on the logits of a step, in front of the sampling (decode.hip decode_greedy_kernel): row b, token v
//   x = logit;  seen: x = x > 0 ? x / repetition : x * repetition;  x -= frequency * count;  count > 0: x -= presence;  x += bias[v];
//   not allowed: x = -inf;  one rounding to the logits' type
// seen: v is among the first n_tokens ids of the row; count: how often from the n_prompt-th on.
//
// Bound by the bytes of the logits (read and written once).  A workgroup owns a run of the vocabulary: it walks the row's whole history,
// counts the ids that fall into its run in shared memory (integer additions: no order to depend on) and then streams its logits through.
// The history is read once per run and row, out of L2; the alternative, a table of counts per row in memory, costs 4 bytes per
// vocabulary entry each step instead.  Measured (medians): 64 rows of 131072 fp32 logits with biases and masks per row 20.8 us (103 MB: 4.9 TB/s; a
// large copy 5.1); one row of 128256 fp16 logits with a history of 2304: 5.0 us, a launch's latency and two passes through shared memory.
#include "fk_device.h"
#include "fk_host.h"
#include "prof.h"

namespace fk {

constexpr int PEN_THREADS = 512;

struct PenaltyArgs {
    const void *logits;
    void *out;
    int64_t row, out_row;                    // elements
    const int64_t *tokens;                   // [B,L]; nullptr: no history
    int64_t tok_row;
    const int32_t *n_tokens, *n_prompt;      // nullptr: L, 0
    const float *repetition, *presence, *frequency, *bias;
    const uint32_t *allowed;
    int64_t bias_row, allowed_row;
    int n_tokens_step, n_prompt_step, repetition_step, presence_step, frequency_step;
    int V, L, chunk;
};

template <int DT> __device__ __forceinline__ float pen_load(const void *p, int64_t i)
{
    if (DT == FASTKV_F32) return reinterpret_cast<const float *>(p)[i];
    const uint32_t h = reinterpret_cast<const uint16_t *>(p)[i];
    return DT == FASTKV_BF16 ? __builtin_bit_cast(float, h << 16) : h2f((uint16_t)h);
}
template <int DT> __device__ __forceinline__ uint16_t pen_round(float x)       // nearest even
{
    if (DT == FASTKV_BF16) return __builtin_bit_cast(uint16_t, (__bf16)x);
    return f2h(x);
}

// grid (runs, B); VEC: rows of logits, out and bias are 16-byte aligned, eight elements per thread and step
template <int DT, bool VEC>
__global__ void __launch_bounds__(PEN_THREADS) penalties_kernel(const PenaltyArgs A)
{
    extern __shared__ uint32_t s_cnt[];      // [chunk]: bit 31 = in the prompt, below: the count behind it
    const int b = blockIdx.y, v0 = blockIdx.x * A.chunk, nv = min(A.chunk, A.V - v0), tid = threadIdx.x;
    float rep = 1.0f, pres = 0.0f, freq = 0.0f;
    if (A.tokens) {
        for (int i = tid; i < nv; i += PEN_THREADS) s_cnt[i] = 0;
        if (A.repetition) rep = A.repetition[(int64_t)b * A.repetition_step];
        if (A.presence) pres = A.presence[(int64_t)b * A.presence_step];
        if (A.frequency) freq = A.frequency[(int64_t)b * A.frequency_step];
        int n = A.n_tokens ? A.n_tokens[(int64_t)b * A.n_tokens_step] : A.L;
        n = n < A.L ? n : A.L;
        const int np = A.n_prompt ? A.n_prompt[(int64_t)b * A.n_prompt_step] : 0;
        __syncthreads();
        const int64_t *row = A.tokens + b * A.tok_row;
        for (int i = tid; i < n; i += PEN_THREADS) {
            const int64_t v = row[i] - v0;
            if (v >= 0 && v < nv) {
                if (i < np) atomicOr(&s_cnt[v], 0x80000000u);
                else atomicAdd(&s_cnt[v], 1u);
            }
        }
        __syncthreads();
    }
    const uint32_t *mask = A.allowed ? A.allowed + b * A.allowed_row : nullptr;
    const float *bias = A.bias ? A.bias + b * A.bias_row : nullptr;
    auto one = [&](float x, int i, float add, bool ok) {
        if (A.tokens) {
            const uint32_t w = s_cnt[i], c = w & 0x7fffffffu;
            if (A.repetition && w) x = x > 0.0f ? x / rep : x * rep;
            if (A.frequency) x = x - freq * (float)c;
            if (A.presence && c) x = x - pres;
        }
        if (bias) x = x + add;
        return ok ? x : -INFINITY;
    };
    const int64_t in0 = b * A.row + v0, out0 = b * A.out_row + v0;
    const int whole = VEC ? nv & ~7 : 0;
    for (int i = tid * 8; i < whole; i += PEN_THREADS * 8) {
        float x[8], add[8];
        uint32_t ok = 0xffu;
        if (mask) ok = mask[(v0 + i) >> 5] >> (i & 24);      // (v0 is a multiple of 32)
        if (DT == FASTKV_F32) {
            const float4 *p = reinterpret_cast<const float4 *>(reinterpret_cast<const float *>(A.logits) + in0 + i);
            const float4 a = p[0], c = p[1];
            x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = c.x; x[5] = c.y; x[6] = c.z; x[7] = c.w;
        } else {
            const uint4 a = *reinterpret_cast<const uint4 *>(reinterpret_cast<const uint16_t *>(A.logits) + in0 + i);
            const uint32_t wd[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const uint32_t h = wd[e >> 1] >> ((e & 1) * 16) & 0xffffu;
                x[e] = DT == FASTKV_BF16 ? __builtin_bit_cast(float, h << 16) : h2f((uint16_t)h);
            }
        }
        if (bias) {
            const float4 *p = reinterpret_cast<const float4 *>(bias + v0 + i);
            const float4 a = p[0], c = p[1];
            add[0] = a.x; add[1] = a.y; add[2] = a.z; add[3] = a.w; add[4] = c.x; add[5] = c.y; add[6] = c.z; add[7] = c.w;
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = one(x[e], i + e, bias ? add[e] : 0.0f, ok >> e & 1);
        if (DT == FASTKV_F32) {
            float4 *p = reinterpret_cast<float4 *>(reinterpret_cast<float *>(A.out) + out0 + i);
            p[0] = make_float4(x[0], x[1], x[2], x[3]);
            p[1] = make_float4(x[4], x[5], x[6], x[7]);
        } else {
            uint32_t o[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = (uint32_t)pen_round<DT>(x[2 * e]) | (uint32_t)pen_round<DT>(x[2 * e + 1]) << 16;
            *reinterpret_cast<uint4 *>(reinterpret_cast<uint16_t *>(A.out) + out0 + i) = make_uint4(o[0], o[1], o[2], o[3]);
        }
    }
    for (int i = whole + tid; i < nv; i += PEN_THREADS) {
        const float x = one(pen_load<DT>(A.logits, in0 + i), i, bias ? bias[v0 + i] : 0.0f, !mask || (mask[(v0 + i) >> 5] >> (i & 31) & 1));
        if (DT == FASTKV_F32) reinterpret_cast<float *>(A.out)[out0 + i] = x;
        else reinterpret_cast<uint16_t *>(A.out)[out0 + i] = pen_round<DT>(x);
    }
}

template <int DT> static void pen_launch(const PenaltyArgs &A, int B, bool vec, hipStream_t st)
{
    const dim3 grid((unsigned)((A.V + A.chunk - 1) / A.chunk), (unsigned)B);
    const size_t lds = A.tokens ? (size_t)A.chunk * 4 : 0;
    if (vec) hipLaunchKernelGGL((penalties_kernel<DT, true>), grid, dim3(PEN_THREADS), lds, st, A);
    else hipLaunchKernelGGL((penalties_kernel<DT, false>), grid, dim3(PEN_THREADS), lds, st, A);
}

// Rows of aw bytes, as apart, na of them from `a` on, and such rows from `b` on: no byte is in both.  (Equal distances: also where the rows lie between
// each other, like two halves of one wide tensor.)
static bool pen_apart(uintptr_t a, int64_t na, int64_t as, int64_t aw, uintptr_t b, int64_t nb, int64_t bs, int64_t bw)
{
    const uintptr_t a1 = a + (na - 1) * as + aw, b1 = b + (nb - 1) * bs + bw;
    if (a1 <= b || b1 <= a) return true;
    if (as != bs || as <= 0) return false;
    const int64_t d = b >= a ? (int64_t)((b - a) % as) : (as - (int64_t)((a - b) % as)) % as;
    return d >= aw && d + bw <= as;
}

}  // namespace fk

using namespace fk;

extern "C" int fastkv_decode_penalties(int32_t dtype, int32_t B, int32_t V, const void *logits, int64_t row_stride, const int64_t *tokens,
                                       int64_t token_stride, int32_t L, const int32_t *n_tokens, int32_t n_tokens_step, const int32_t *n_prompt,
                                       int32_t n_prompt_step, const float *repetition, int32_t repetition_step, const float *presence,
                                       int32_t presence_step, const float *frequency, int32_t frequency_step, const float *bias,
                                       int64_t bias_stride, const int32_t *allowed, int64_t allowed_stride, void *out, int64_t out_stride,
                                       void *stream)
{
    if (dtype < FASTKV_F16 || dtype > FASTKV_F32 || B < 1 || B > 65535 || V < 1 || L < 0 || !logits || !out || row_stride < V || out_stride < V)
        return FASTKV_EINVAL;
    if ((L > 0 && (!tokens || token_stride < 0)) || bias_stride < 0 || allowed_stride < 0) return FASTKV_EINVAL;
    const int word = dtype == FASTKV_F32 ? 4 : 2;
    if (((uintptr_t)logits | (uintptr_t)out) % word || ((uintptr_t)tokens & 7)) return FASTKV_EINVAL;
    const int32_t steps[5] = {n_tokens_step, n_prompt_step, repetition_step, presence_step, frequency_step};
    for (int i = 0; i < 5; ++i) if (steps[i] < 0 || steps[i] > 1) return FASTKV_EINVAL;
    // in place, or apart; and what other workgroups still read is never written
    auto out_apart = [&](const void *p, int64_t n, int64_t stride, int64_t width) {
        return !p || pen_apart((uintptr_t)out, B, out_stride * word, (int64_t)V * word, (uintptr_t)p, n, stride, width);
    };
    if (!(logits == out && (row_stride == out_stride || B == 1)) && !out_apart(logits, B, row_stride * word, (int64_t)V * word)) return FASTKV_EINVAL;
    if ((L > 0 && !out_apart(tokens, B, token_stride * 8, (int64_t)L * 8)) || !out_apart(bias, B, bias_stride * 4, (int64_t)V * 4) ||
        !out_apart(allowed, B, allowed_stride * 4, (V + 31LL) / 32 * 4))
        return FASTKV_EINVAL;
    const void *const values[5] = {n_tokens, n_prompt, repetition, presence, frequency};
    for (int i = 0; i < 5; ++i) if (!out_apart(values[i], B, steps[i] * 4, 4)) return FASTKV_EINVAL;
    PenaltyArgs A = {};
    A.logits = logits;
    A.out = out;
    A.row = row_stride;
    A.out_row = out_stride;
    if (L > 0 && (repetition || presence || frequency)) A.tokens = tokens;
    A.tok_row = token_stride;
    A.n_tokens = n_tokens;
    A.n_prompt = n_prompt;
    A.repetition = repetition;
    A.presence = presence;
    A.frequency = frequency;
    A.bias = bias;
    A.allowed = (const uint32_t *)allowed;
    A.bias_row = bias_stride;
    A.allowed_row = allowed_stride;
    A.n_tokens_step = n_tokens_step;
    A.n_prompt_step = n_prompt_step;
    A.repetition_step = repetition_step;
    A.presence_step = presence_step;
    A.frequency_step = frequency_step;
    A.V = V;
    A.L = L;
    const int64_t runs = (512 + B - 1) / B;                  // two workgroups per compute unit; 4096 .. 16384 entries each
    int64_t chunk = ((V + runs - 1) / runs + 4095) / 4096 * 4096;
    A.chunk = (int)(chunk > 16384 ? 16384 : chunk);
    const bool vec = !(((uintptr_t)logits | (uintptr_t)out | (uintptr_t)bias) & 15) && !((row_stride | out_stride) * word & 15) && !(bias_stride & 3);
    ProfScope ps_(K_DECODE, (hipStream_t)stream);
    if (dtype == FASTKV_F16) pen_launch<FASTKV_F16>(A, B, vec, (hipStream_t)stream);
    else if (dtype == FASTKV_BF16) pen_launch<FASTKV_BF16>(A, B, vec, (hipStream_t)stream);
    else pen_launch<FASTKV_F32>(A, B, vec, (hipStream_t)stream);
    return hipGetLastError() == hipSuccess ? FASTKV_OK : FASTKV_ELAUNCH;
}
