// Quantize-and-append of packed prompts into the int8 arena.
//
// Per (token, head) row of K and of V, as every other writer of the arena:
//   s = max(max|x| / 127, 1e-12)            IEEE f32 division
//   q = clamp(round_half_even(x / s), -127, 127)
// This file is compiled with -fmad=false -prec-div=true, as quant.cu.
//
// A streaming kernel: 2 bytes in and 1 out an element (bf16).  What bounds it is
// the issue of the division's instructions, so x / s is Markstein's division with
// y = RN(1/s) computed once a row, on packed pairs:
//   q0 = x y,  q1 = q0 + (x - q0 s) y,  q2 = q1 + (x - q1 s) y     (FMAs)
// q0 is within 1.5 units of the last place of x/s, q1 within (1/2 + 2^-22), and
// from an estimate nearer than one unit the last step gives RN(x/s) (P. Markstein,
// IBM J. Res. Dev. 34, 1990).  Nothing over- or underflows where it matters: s is
// at least 1e-12, and below |x/s| = 1/4 the code is 0 whatever the last bits say.
// RN(m/127) is taken the same way with RN(1/127), by one step, which is right for
// all 2^23 mantissas (the tests go through them).  Rounding is the addition of
// 1.5 * 2^23, whose low byte is the code; with |x| <= max|x| no clamp is needed.
// 16 prompts of 1493 to 2048 tokens, 16 heads of 128: 73 us, 4.8 TB/s, 61 % of issue
// slots (f32 97 us, 6.0 TB/s); with the division instruction it took 156.  1023 tokens of 24 heads of 64:
// 3 us.  Twice the rows a lane, for more loads in flight, cost more registers than
// they hid.
// A row that is not finite is divided one by one.  (Dividing only near half
// integers does not pay: quotients of bf16 numbers fall on them too often.)
#include "common.cuh"
#include "../host/internal.h"

namespace pp {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxChunk = 64;  // tokens of a CTA
constexpr int kE = 16;         // elements of a lane

struct AppendArgs {
    const void* src[2];  // K, V
    uint64_t ts[2], hs[2];
    uint8_t* codes[2];
    float* scales[2];
    const uint32_t* starts;
    const uint32_t* offsets;
    uint32_t tokens, branches, heads, capacity, chunk;
    uint32_t vec;
    uint32_t* status;
};

// A lane's 16 elements as they lie in memory.
template <bool BF>
struct Raw {
    uint4 w[BF ? 2 : 4];
};

template <bool BF>
__device__ __forceinline__ Raw<BF> load_raw(const void* p, uint64_t i, bool vec) {
    Raw<BF> r;
    if (vec) {
        const uint4* s = reinterpret_cast<const uint4*>(reinterpret_cast<const char*>(p) + i * (BF ? 2 : 4));
#pragma unroll
        for (int h = 0; h < (BF ? 2 : 4); ++h) r.w[h] = __ldg(s + h);
    } else if constexpr (BF) {
        const uint16_t* s = reinterpret_cast<const uint16_t*>(p) + i;
#pragma unroll
        for (int h = 0; h < 2; ++h)
            r.w[h] = make_uint4(s[8 * h] | (uint32_t)s[8 * h + 1] << 16, s[8 * h + 2] | (uint32_t)s[8 * h + 3] << 16,
                                s[8 * h + 4] | (uint32_t)s[8 * h + 5] << 16, s[8 * h + 6] | (uint32_t)s[8 * h + 7] << 16);
    } else {
        const uint32_t* s = reinterpret_cast<const uint32_t*>(p) + i;
#pragma unroll
        for (int h = 0; h < 4; ++h) r.w[h] = make_uint4(s[4 * h], s[4 * h + 1], s[4 * h + 2], s[4 * h + 3]);
    }
    return r;
}

template <bool BF>
__device__ __forceinline__ void unpack(const Raw<BF>& r, float (&v)[kE]) {
#pragma unroll
    for (int h = 0; h < (BF ? 2 : 4); ++h) {
        const uint32_t w[4] = {r.w[h].x, r.w[h].y, r.w[h].z, r.w[h].w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if constexpr (BF) {
                v[8 * h + 2 * k] = bf16_lo_to_f32(w[k]);
                v[8 * h + 2 * k + 1] = bf16_hi_to_f32(w[k]);
            } else {
                v[4 * h + k] = __uint_as_float(w[k]);
            }
        }
    }
}

// max|x| of a lane's elements; NaN if one is.
template <bool BF>
__device__ __forceinline__ float largest(const Raw<BF>& r) {
    if constexpr (BF) {
        uint32_t m = 0u;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint32_t w[4] = {r.w[h].x, r.w[h].y, r.w[h].z, r.w[h].w};
#pragma unroll
            for (int k = 0; k < 4; ++k) asm("max.NaN.bf16x2 %0, %0, %1;" : "+r"(m) : "r"(w[k] & 0x7fff7fffu));
        }
        float lo = bf16_lo_to_f32(m);
        asm("max.NaN.f32 %0, %0, %1;" : "+f"(lo) : "f"(bf16_hi_to_f32(m)));
        return lo;
    } else {
        float m = 0.f;
#pragma unroll
        for (int h = 0; h < 4; ++h) {
            const uint32_t w[4] = {r.w[h].x, r.w[h].y, r.w[h].z, r.w[h].w};
#pragma unroll
            for (int k = 0; k < 4; ++k) asm("max.NaN.f32 %0, %0, %1;" : "+f"(m) : "f"(fabsf(__uint_as_float(w[k]))));
        }
        return m;
    }
}

__device__ __forceinline__ float over_127(float m) {  // RN(m / 127)
    const float y = 0x1.020408p-7f, q = m * y;         // y = RN(1 / 127)
    return __fmaf_rn(__fmaf_rn(-127.f, q, m), y, q);
}

struct Divided {
    uint4 codes;
    float s;
    bool finite;
};

// A lane's part of a row that is not finite, as quant_row.cuh: the scale passes over NaN.
template <int D, bool BF>
__device__ __noinline__ Divided divided(const void* src, uint64_t from, bool vec) {
    constexpr int L = D / kE;
    float v[kE], m = 0.f;
    bool finite = true;
    unpack<BF>(load_raw<BF>(src, from, vec), v);
#pragma unroll
    for (int k = 0; k < kE; ++k) {
        finite = finite && isfinite(v[k]);
        m = fmaxf(m, fabsf(v[k]));
    }
    const uint32_t row_lanes = ((1u << L) - 1u) << (threadIdx.x % 32 / L * L);
#pragma unroll
    for (int o = L / 2; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(row_lanes, m, o));
    const float s = fmaxf(__fdiv_rn(m, 127.f), 1e-12f);
    uint32_t w[kE / 4];
#pragma unroll
    for (int k = 0; k < kE; k += 4) {
        w[k / 4] = 0u;
#pragma unroll
        for (int h = 0; h < 4; ++h)
            w[k / 4] |= (uint32_t)(max(-127, min(127, __float2int_rn(__fdiv_rn(v[k + h], s)))) & 0xff) << (8 * h);
    }
    return Divided{make_uint4(w[0], w[1], w[2], w[3]), s, finite};
}

// CTA (x, y) takes `chunk` tokens of all heads of K (y = 0) or V; D / 16 lanes a row.
template <int D, bool BF>
__global__ void __launch_bounds__(kThreads) prompt_append_kernel(const AppendArgs a) {
    constexpr int L = D / kE;
    constexpr uint32_t R = kThreads / L;  // rows of the block at a time
    __shared__ uint64_t dst[kMaxChunk];   // slot of head 0 of each token, or ~0
    const uint32_t t0 = blockIdx.x * a.chunk, n_tok = min(a.chunk, a.tokens - t0);
    const uint32_t rows = n_tok * a.heads;
    const int lane = threadIdx.x % L;
    const bool is_v = blockIdx.y;
    const void* src = is_v ? a.src[1] : a.src[0];
    const uint64_t ts = is_v ? a.ts[1] : a.ts[0], hs = is_v ? a.hs[1] : a.hs[0];
    uint8_t* arena = is_v ? a.codes[1] : a.codes[0];
    float* scales = is_v ? a.scales[1] : a.scales[0];
    pdl_wait_primary();
    int bad = 0;
    for (uint32_t b = threadIdx.x; b < a.branches; b += kThreads)
        bad |= a.starts[b + 1] < a.starts[b] || a.starts[b + 1] > a.tokens;
    if (__syncthreads_or(bad)) {
        if (blockIdx.x == 0 && threadIdx.x == 0 && a.status) atomicOr(a.status, PP_DEV_LENGTH_RANGE);
        return;
    }
    if (threadIdx.x < n_tok) {
        const uint32_t t = t0 + threadIdx.x;
        uint32_t lo = 0, hi = a.branches;  // the last branch that starts at or before t
        while (hi - lo > 1) {
            const uint32_t mid = lo + (hi - lo) / 2;
            if (a.starts[mid] <= t) lo = mid;
            else hi = mid;
        }
        uint64_t d = ~0ull;
        if (a.starts[lo] <= t && t < a.starts[lo + 1]) {
            const uint64_t slot = (uint64_t)a.offsets[lo] + (t - a.starts[lo]);
            if (slot < a.capacity) d = (uint64_t)lo * a.heads * a.capacity + slot;
            else if (a.status) atomicOr(a.status, PP_DEV_OFFSET_RANGE);
        }
        dst[threadIdx.x] = d;
    }
    __syncthreads();
    // R rows further: so many tokens and heads, the place in the source and the head's in the arena with them
    const uint32_t step_tok = R / a.heads, step_head = R % a.heads;
    const uint64_t step_from = step_tok * ts + step_head * hs, wrap_from = ts - a.heads * hs;
    const uint64_t step_row = (uint64_t)step_head * a.capacity, wrap_row = (uint64_t)a.heads * a.capacity;
    uint32_t tok = threadIdx.x / L / a.heads, head = threadIdx.x / L % a.heads;
    uint64_t next_from = (uint64_t)(t0 + tok) * ts + head * hs + kE * lane, next_row = (uint64_t)head * a.capacity;
    bool finite = true;
    for (uint32_t r0 = 0; r0 < rows; r0 += R) {  // the same number of turns for all of the block
        uint64_t slot = tok < n_tok ? dst[tok] : ~0ull;
        const uint64_t from = next_from;
        Raw<BF> raw{};
        if (slot != ~0ull) {
            slot += next_row;
            raw = load_raw<BF>(src, from, a.vec);
        }
        tok += step_tok;
        head += step_head;
        next_from += step_from;
        next_row += step_row;
        if (head >= a.heads) {
            head -= a.heads;
            ++tok;
            next_from += wrap_from;
            next_row -= wrap_row;
        }
        float v[kE], m = largest<BF>(raw);
        unpack<BF>(raw, v);
#pragma unroll
        for (int o = L / 2; o; o >>= 1) {
            const float y = __shfl_xor_sync(0xffffffffu, m, o);
            asm("max.NaN.f32 %0, %0, %1;" : "+f"(m) : "f"(y));
        }
        float s = fmaxf(over_127(m), 1e-12f);
        const float y = __frcp_rn(s);
        const uint64_t y2 = f2_pack(y, y), s2 = f2_pack(-s, -s), up = f2_pack(12582912.f, 12582912.f);
        uint32_t w[kE / 4];
#pragma unroll
        for (int k = 0; k < kE; k += 4) {
            float c[4];
#pragma unroll
            for (int h = 0; h < 4; h += 2) {
                const uint64_t x = f2_pack(v[k + h], v[k + h + 1]);
                uint64_t q = f2_mul(x, y2);
                q = f2_fma(f2_fma(q, s2, x), y2, q);
                q = f2_fma(f2_fma(q, s2, x), y2, q);
                f2_unpack(f2_add(q, up), c[h], c[h + 1]);
            }
            w[k / 4] = __byte_perm(__byte_perm(__float_as_uint(c[0]), __float_as_uint(c[1]), 0x0040),
                                   __byte_perm(__float_as_uint(c[2]), __float_as_uint(c[3]), 0x0040), 0x5410);
        }
        uint4 codes = make_uint4(w[0], w[1], w[2], w[3]);
        if (!isfinite(m)) {  // all the row's lanes
            const Divided d = divided<D, BF>(src, from, a.vec);
            codes = d.codes;
            s = d.s;
            finite = finite && d.finite;
        }
        if (slot != ~0ull) {
            *reinterpret_cast<uint4*>(arena + slot * D + kE * lane) = codes;
            if (lane == 0) scales[slot] = s;
        }
    }
    if (!finite && a.status) atomicOr(a.status, PP_DEV_NONFINITE_INPUT);
}

}  // namespace

cudaError_t launch_prompt_append(const PromptAppendLaunch& P, cudaStream_t stream) {
    AppendArgs a{};
    a.src[0] = P.k;
    a.src[1] = P.v;
    a.ts[0] = P.k_ts;
    a.ts[1] = P.v_ts;
    a.hs[0] = P.k_hs;
    a.hs[1] = P.v_hs;
    a.codes[0] = P.arena->k;
    a.codes[1] = P.arena->v;
    a.scales[0] = P.arena->k_scale;
    a.scales[1] = P.arena->v_scale;
    a.starts = P.starts;
    a.offsets = P.offsets;
    a.tokens = P.tokens;
    a.branches = P.arena->rows / P.arena->heads;
    a.heads = P.arena->heads;
    a.capacity = P.arena->capacity;
    a.vec = P.vec;
    a.status = P.status;
    // About 24 CTAs an SM where the prompts are long, at least one turn of rows each where they are short.  64 tokens a
    // CTA throughout: 1023 tokens 13 us instead of 3; one turn throughout: the 16 prompts 106 us instead of 75.
    const uint32_t turn = kThreads / (P.arena->head_dim / kE);
    uint32_t chunk = P.tokens / (12 * P.num_sms);
    chunk = chunk > (turn + a.heads - 1) / a.heads ? chunk : (turn + a.heads - 1) / a.heads;
    a.chunk = chunk < kMaxChunk ? chunk : kMaxChunk;
    const dim3 grid(P.tokens ? (P.tokens + a.chunk - 1) / a.chunk : 1, 2);  // without tokens the starts are checked
    if (P.arena->head_dim == 128)
        return P.bf16 ? launch_pdl(prompt_append_kernel<128, true>, grid, dim3(kThreads), stream, a)
                      : launch_pdl(prompt_append_kernel<128, false>, grid, dim3(kThreads), stream, a);
    return P.bf16 ? launch_pdl(prompt_append_kernel<64, true>, grid, dim3(kThreads), stream, a)
                  : launch_pdl(prompt_append_kernel<64, false>, grid, dim3(kThreads), stream, a);
}

}  // namespace pp
