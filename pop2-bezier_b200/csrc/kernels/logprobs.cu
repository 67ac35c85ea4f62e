// Log probabilities of given tokens, entropy, rank and the best alternatives
// of rows of logits, in one pass over them.
//
// With m the largest logit of the window, e_i = exp(x_i - m), s the sum of all
// e_i less one that is the largest itself, and d = sum of e_i (m - x_i):
//   log p_t = (x_t - m) - log1p(s)         entropy = log1p(s) + d / (1 + s)
// Leaving the largest out of s keeps what is left of a nearly certain token's
// log probability, which 1 + s would round away; both terms of the entropy are
// positive, so nothing cancels.  s is kept as the sum over x < m and the count
// of x = m.  When the maximum rises by g, both change by exp(-g), and d by
// (d + g (s + count)) exp(-g).
//
// A lane holds 8 vectors of 16 bytes in registers: they are read once and looked
// at several times (maximum, sums, rank, alternatives).  NW warps take 4 KB each
// of a row; a longer row is taken in steps, or by a cluster of up to 8 CTAs
// that merge through their shared memory, when there are few rows.
//
// Alternatives: the k-th largest of a warp's 32 lane maxima is no larger than
// the k-th largest logit, and neither is the largest such bound of all warps.
// Only logits from that bound on are candidates, on random rows about k of
// them; one warp sorts them 32 at a time and keeps the best 32 as a sorted list,
// one a lane.  Where the bound leaves more than the buffer holds (long ties),
// the block takes the maximum k times instead.
//
// Bound by HBM on long rows; issue slots come next (about 9 a bf16 element).
#include <math_constants.h>

#include "common.cuh"
#include "../host/internal.h"

namespace pp {
namespace {

#ifndef LOGPROBS_WARPS
#define LOGPROBS_WARPS 32  // resident warps of an SM: bounds the registers
#endif
constexpr int kVecs = 8;              // 16-byte vectors a lane holds
constexpr uint32_t kCandidates = 512;
constexpr float kLog2e = 1.4426950408889634f;

struct Args {
    const void* logits;
    uint64_t stride;
    const int32_t* targets;
    const uint32_t* bounds;
    uint32_t rows, choices, top, cluster;
    float* logprob;
    float* entropy;
    uint32_t* rank;
    uint32_t* top_ids;
    float* top_logprobs;
    uint32_t* status;
};

// What a CTA (or a thread, with its own s, c, d and ahead) knows of a row.
struct Part {
    float m, s, c, d;
    uint32_t ahead;
};

__device__ __forceinline__ void raise(Part& p, float m) {
    if (!(m > p.m)) return;
    if (p.m > -CUDART_INF_F) {
        const float g = m - p.m, f = fast_exp2(-g * kLog2e);
        const float all = p.s + p.c;
        if (f > 0.f) {  // g may be inf between the type's ends
            p.d = (p.d + g * all) * f;
            p.s = all * f;
        } else if (all == all) {
            p.d = p.s = 0.f;
        }
    }
    p.c = 0.f;
    p.m = m;
}

__device__ __forceinline__ Part merge(Part a, Part b) {
    const float m = fmaxf(a.m, b.m);
    raise(a, m);
    raise(b, m);
    a.s += b.s;
    a.c += b.c;
    a.d += b.d;
    a.ahead += b.ahead;
    return a;
}

// Order of the alternatives as one number: larger logit, then lower column.
__device__ __forceinline__ unsigned long long order_of(float x, uint32_t column) {
    const uint32_t b = __float_as_uint(x + 0.f);  // -0 and +0 are one value
    return (unsigned long long)(b & 0x80000000u ? ~b : b | 0x80000000u) << 32 | ~column;
}
__device__ __forceinline__ float order_value(unsigned long long o) {
    const uint32_t k = (uint32_t)(o >> 32);
    return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

// Sorts 32 values, one a lane, largest first (bitonic network).
template <typename T>
__device__ __forceinline__ T sort32(T x, uint32_t lane) {
#pragma unroll
    for (uint32_t k = 2; k <= 32; k <<= 1)
#pragma unroll
        for (uint32_t j = k >> 1; j; j >>= 1) {
            const T y = __shfl_xor_sync(0xffffffffu, x, j);
            const bool big = ((lane & k) == 0) == ((lane & j) == 0);
            x = big == (x > y) ? x : y;
        }
    return x;
}

// The best 32 of two sorted lists, sorted.
__device__ __forceinline__ unsigned long long merge32(unsigned long long a, unsigned long long b, uint32_t lane) {
    b = __shfl_sync(0xffffffffu, b, 31 - lane);
    unsigned long long x = a > b ? a : b;
#pragma unroll
    for (uint32_t j = 16; j; j >>= 1) {
        const unsigned long long y = __shfl_xor_sync(0xffffffffu, x, j);
        x = ((lane & j) == 0) == (x > y) ? x : y;
    }
    return x;
}

template <bool BF>
__device__ __forceinline__ float load_logit(const void* p, uint64_t i) {
    if constexpr (BF) return bf16_lo_to_f32(__ldg(reinterpret_cast<const unsigned short*>(p) + i));
    else return __ldg(reinterpret_cast<const float*>(p) + i);
}

// Elements of a vector: 8 bf16 or 4 f32.
template <bool BF>
__device__ __forceinline__ float element(const uint4& v, int i) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    if constexpr (BF) return i & 1 ? bf16_hi_to_f32(w[i / 2]) : bf16_lo_to_f32(w[i / 2]);
    else return __uint_as_float(w[i]);
}

__device__ __forceinline__ uint32_t max_bf16x2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}

template <bool BF>
__device__ __forceinline__ float vector_max(const uint4& v) {  // of what is not NaN; NaN if all are
    if constexpr (BF) {
        const uint32_t w = max_bf16x2(max_bf16x2(v.x, v.y), max_bf16x2(v.z, v.w));
        return fmaxf(bf16_lo_to_f32(w), bf16_hi_to_f32(w));
    } else {
        return fmaxf(fmaxf(element<false>(v, 0), element<false>(v, 1)), fmaxf(element<false>(v, 2), element<false>(v, 3)));
    }
}

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t ld_peer(const void* p, uint32_t rank) {
    uint32_t a, v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_addr(p)), "r"(rank));
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
    return v;
}

template <bool BF, int NW>
__global__ void __launch_bounds__(32 * NW, LOGPROBS_WARPS / NW) logprobs_kernel(const Args a) {
    constexpr int EPV = BF ? 8 : 4;                    // elements of a vector
    constexpr uint32_t STEP = NW * 32 * kVecs;         // vectors a CTA holds
    __shared__ float s_max[NW], s_bound[NW], s_kth;
    __shared__ unsigned long long s_cand[kCandidates], s_list[32], s_best[NW];
    __shared__ uint32_t s_count[2];
    __shared__ Part s_part[NW], s_cta;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t row = blockIdx.x / a.cluster, part = a.cluster > 1 ? cluster_rank() : 0u;
    const uint32_t k = a.top;
    pdl_wait_primary();
    const uint64_t base = (uint64_t)row * a.stride;
    uint32_t lo = 0, n = a.choices;
    if (a.bounds) {
        lo = a.bounds[2 * row];
        n = a.bounds[2 * row + 1];
        if ((uint64_t)lo + n > a.choices) {
            if (threadIdx.x == 0 && part == 0 && a.status) atomicOr(a.status, PP_DEV_WINDOW_RANGE);
            lo = n = 0;
        }
    }
    const uint32_t hi = lo + n;
    const int64_t target = a.targets[row];
    const bool inside = target >= lo && target < (int64_t)hi;
    const uint32_t t = inside ? (uint32_t)target : 0u;
    const float xt = inside ? load_logit<BF>(a.logits, base + t) : -CUDART_INF_F;
    // ahead of the target: x > xt behind it, x >= xt (x > the float below xt) before it.  A NaN or -inf target is
    // counted by itself, below.
    const bool ordinary = inside && xt > -CUDART_INF_F;
    const float below = ordinary ? nextafterf(xt, -CUDART_INF_F) : 0.f;

    // Vectors lie on 16-byte boundaries of memory: vector v holds the columns first + v * EPV ...
    const uint64_t addr = reinterpret_cast<uint64_t>(a.logits) + (base + lo) * (BF ? 2 : 4);
    const int64_t first = (int64_t)lo - (int64_t)(addr % 16 / (BF ? 2 : 4));
    const uint32_t vectors = n ? (uint32_t)((hi - first + EPV - 1) / EPV) : 0u;

    Part p{-CUDART_INF_F, 0.f, 0.f, 0.f, 0u};
    unsigned long long list = 0;  // warp 0: the best so far, sorted over the lanes
    if (threadIdx.x == 0) {
        s_count[0] = 0;
        s_kth = -CUDART_INF_F;
    }
    uint32_t turn = 0;  // the two counts take turns: one is emptied when nobody reads it
    for (uint64_t v0 = (uint64_t)part * STEP; v0 < vectors; v0 += (uint64_t)a.cluster * STEP, turn ^= 1) {
        uint4 x[kVecs];
        float vm[kVecs];
        const uint32_t mine = (uint32_t)v0 + warp * 32 * kVecs + lane;
#pragma unroll
        for (int v = 0; v < kVecs; ++v) {
            const uint32_t at = mine + 32 * v;
            const int64_t col = first + (int64_t)at * EPV;
            const uint32_t none = BF ? 0xff80ff80u : 0xff800000u;  // -inf
            x[v] = make_uint4(none, none, none, none);
            if (at < vectors) {
                if (col >= lo && col + EPV <= hi) {
                    if constexpr (BF)
                        x[v] = __ldg(reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(a.logits) + base + col));
                    else x[v] = __ldg(reinterpret_cast<const uint4*>(reinterpret_cast<const float*>(a.logits) + base + col));
                } else {  // an end of the window
                    uint32_t w[4] = {none, none, none, none};
#pragma unroll
                    for (int i = 0; i < EPV; ++i)
                        if (col + i >= lo && col + i < hi) {
                            const uint32_t bits = __float_as_uint(load_logit<BF>(a.logits, base + col + i));
                            if constexpr (BF) w[i / 2] = i & 1 ? (w[i / 2] & 0xffffu) | bits : (w[i / 2] & 0xffff0000u) | bits >> 16;
                            else w[i] = bits;
                        }
                    x[v] = make_uint4(w[0], w[1], w[2], w[3]);
                }
            }
        }
        float top = -CUDART_INF_F;
#pragma unroll
        for (int v = 0; v < kVecs; ++v) {
            vm[v] = vector_max<BF>(x[v]);
            top = fmaxf(top, vm[v]);
        }
        float bound = -CUDART_INF_F;
        if (k) {
            top = sort32(top, lane);
            bound = __shfl_sync(0xffffffffu, top, k - 1);
        } else {
#pragma unroll
            for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        }
        if (lane == 0) {
            s_max[warp] = top;
            s_bound[warp] = bound;
        }
        __syncthreads();
        float m = p.m;
        bound = s_kth;
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            m = fmaxf(m, s_max[w]);
            bound = fmaxf(bound, s_bound[w]);
        }
        raise(p, m);
        const float ref = m > -CUDART_INF_F ? m : 0.f;  // nothing but -inf so far (or NaN, which has to show in s)
        const uint64_t neg = f2_pack(-ref, -ref), l2e = f2_pack(kLog2e, kLog2e);
        uint64_t s0 = 0ull, s1 = 0ull, d0 = 0ull, d1 = 0ull;
#pragma unroll
        for (int v = 0; v < kVecs; ++v) {
            const int64_t col = first + (int64_t)(mine + 32 * v) * EPV;
            if (vm[v] == m) {  // holds the maximum: it is counted, not summed
#pragma unroll
                for (int i = 0; i < EPV; ++i) {
                    const float e = element<BF>(x[v], i);
                    const float y = fmaxf((e - ref) * kLog2e, -160.f), f = e == m ? 0.f : fast_exp2(e == e ? y : e);
                    p.c += e == m ? 1.f : 0.f;
                    p.s += f;
                    p.d -= f * y * 0.6931471805599453f;
                }
            } else {
#pragma unroll
                for (int i = 0; i < EPV; i += 2) {
                    float y0, y1;
                    f2_unpack(f2_mul(f2_add(f2_pack(element<BF>(x[v], i), element<BF>(x[v], i + 1)), neg), l2e), y0, y1);
                    // exp2(-160) is 0 and so is its product with y, which -inf would make NaN
                    asm("max.NaN.f32 %0, %0, %1;" : "+f"(y0) : "f"(-160.f));
                    asm("max.NaN.f32 %0, %0, %1;" : "+f"(y1) : "f"(-160.f));
                    const uint64_t e2 = f2_pack(fast_exp2(y0), fast_exp2(y1));
                    uint64_t& s = i & 2 ? s1 : s0;
                    uint64_t& d = i & 2 ? d1 : d0;
                    s = f2_add(s, e2);
                    asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(d) : "l"(e2), "l"(f2_pack(y0, y1)));
                }
            }
            if (ordinary && vm[v] >= xt) {
                const float edge = col < t ? below : xt;
                if (col <= t && t < col + EPV) {
#pragma unroll
                    for (int i = 0; i < EPV; ++i) p.ahead += element<BF>(x[v], i) > (col + i < t ? below : xt);
                } else {
#pragma unroll
                    for (int i = 0; i < EPV; ++i) p.ahead += element<BF>(x[v], i) > edge;
                }
            }
            if (k && vm[v] >= bound) {
#pragma unroll
                for (int i = 0; i < EPV; ++i) {
                    const float e = element<BF>(x[v], i);
                    if (e >= bound && e > -CUDART_INF_F) {
                        const uint32_t at = atomicAdd(&s_count[turn], 1u);
                        if (at < kCandidates) s_cand[at] = order_of(e, (uint32_t)col + i);
                    }
                }
            }
            asm volatile("" ::: "memory");  // one vector at a time: unpacked, they would not fit the registers
        }
        float e0, e1, e2, e3;
        f2_unpack(f2_add(s0, s1), e0, e1);
        f2_unpack(f2_add(d0, d1), e2, e3);
        p.s += e0 + e1;
        p.d -= (e2 + e3) * 0.6931471805599453f;
        if (k) {
            __syncthreads();
            const uint32_t count = s_count[turn];
            if (count <= kCandidates) {
                if (warp == 0) {
                    for (uint32_t c = 0; c < count; c += 32)
                        list = merge32(list, sort32(c + lane < count ? s_cand[c + lane] : 0ull, lane), lane);
                }
            } else {
                const int64_t from = max((int64_t)lo, first + (int64_t)v0 * EPV);
                const int64_t to = min((int64_t)hi, first + (int64_t)(v0 + STEP) * EPV);
                unsigned long long prev = ~0ull, found = 0;
                for (uint32_t j = 0; j < k; ++j) {
                    unsigned long long best = 0;
                    for (int64_t i = from + threadIdx.x; i < to; i += 32 * NW) {
                        const float e = load_logit<BF>(a.logits, base + i);
                        if (!(e >= bound && e > -CUDART_INF_F)) continue;
                        const unsigned long long o = order_of(e, (uint32_t)i);
                        if (o < prev && o > best) best = o;
                    }
#pragma unroll
                    for (int o = 16; o; o >>= 1) {
                        const unsigned long long y = __shfl_xor_sync(0xffffffffu, best, o);
                        best = best > y ? best : y;
                    }
                    if (lane == 0) s_best[warp] = best;
                    __syncthreads();
                    for (int w = 0; w < NW; ++w) best = best > s_best[w] ? best : s_best[w];
                    if (lane == j) found = best;
                    prev = best;
                    __syncthreads();
                }
                if (warp == 0) list = merge32(list, found, lane);
            }
            if (warp == 0) {
                const unsigned long long kth = __shfl_sync(0xffffffffu, list, k - 1);
                __syncwarp();
                if (lane == 0) {
                    s_count[turn ^ 1] = 0;
                    s_kth = kth ? order_value(kth) : -CUDART_INF_F;
                }
            }
        }
        if (!k) __syncthreads();  // s_max has been read before the next step writes it
    }
    // a NaN target comes behind what is not NaN, a -inf one behind what is larger; of its own kind, behind lower columns
    if (inside && !ordinary) {
        for (uint32_t i = lo + part * 32 * NW + threadIdx.x; i < hi; i += a.cluster * 32 * NW) {
            const float e = load_logit<BF>(a.logits, base + i);
            const bool same = xt == xt ? e == xt : e != e;
            p.ahead += same ? i < t : e > xt || (xt != xt && e == e);
        }
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        p.s += __shfl_xor_sync(0xffffffffu, p.s, o);
        p.c += __shfl_xor_sync(0xffffffffu, p.c, o);
        p.d += __shfl_xor_sync(0xffffffffu, p.d, o);
        p.ahead += __shfl_xor_sync(0xffffffffu, p.ahead, o);
    }
    if (lane == 0) s_part[warp] = p;
    __syncthreads();
    if (warp == 0) {
        for (int w = 1; w < NW; ++w) {
            p.s += s_part[w].s;
            p.c += s_part[w].c;
            p.d += s_part[w].d;
            p.ahead += s_part[w].ahead;
        }
    }
    if (a.cluster > 1) {
        if (warp == 0) {
            s_list[lane] = list;
            if (lane == 0) s_cta = p;
        }
        cluster_sync();
        if (part == 0 && warp == 0) {
            for (uint32_t r = 1; r < a.cluster; ++r) {
                Part o;
                o.m = __uint_as_float(ld_peer(&s_cta.m, r));
                o.s = __uint_as_float(ld_peer(&s_cta.s, r));
                o.c = __uint_as_float(ld_peer(&s_cta.c, r));
                o.d = __uint_as_float(ld_peer(&s_cta.d, r));
                o.ahead = ld_peer(&s_cta.ahead, r);
                p = merge(p, o);
                if (k) {
                    const uint32_t* peer = reinterpret_cast<const uint32_t*>(&s_list[lane]);
                    const unsigned long long l = ld_peer(peer, r), h = ld_peer(peer + 1, r);
                    list = merge32(list, h << 32 | l, lane);
                }
            }
        }
        cluster_sync();  // the peers' shared memory has been read
        if (part != 0) return;
    }
    if (warp != 0) return;
    const bool nothing = !(p.m > -CUDART_INF_F && p.m < CUDART_INF_F) || p.s != p.s;
    const double s = (double)p.s + (double)(p.c - 1.f), lse = log1p(s);  // of the sum, less m
    if (lane == 0) {
        a.logprob[row] = nothing ? CUDART_NAN_F : (float)((double)xt - (double)p.m - lse);
        a.entropy[row] = nothing ? CUDART_NAN_F : (float)(lse + (double)p.d / (1.0 + s));
        a.rank[row] = inside ? p.ahead : n;
    }
    if (lane < k) {
        a.top_ids[(uint64_t)row * k + lane] = list ? ~(uint32_t)list : 0xffffffffu;
        float lp = -CUDART_INF_F;
        if (list) lp = nothing ? CUDART_NAN_F : (float)((double)order_value(list) - (double)p.m - lse);
        a.top_logprobs[(uint64_t)row * k + lane] = lp;
    }
}

template <bool BF, int NW>
cudaError_t launch(const Args& a, cudaStream_t stream) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(a.rows * a.cluster);
    cfg.blockDim = dim3(32 * NW);
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = a.cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = a.cluster > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, logprobs_kernel<BF, NW>, a);
}

template <bool BF>
cudaError_t launch_warps(const Args& a, uint32_t warps, cudaStream_t stream) {
    switch (warps) {
        case 1: return launch<BF, 1>(a, stream);
        case 2: return launch<BF, 2>(a, stream);
        case 4: return launch<BF, 4>(a, stream);
        case 8: return launch<BF, 8>(a, stream);
        default: return launch<BF, 16>(a, stream);
    }
}

}  // namespace

cudaError_t launch_token_logprobs(const LogprobsLaunch& L, cudaStream_t stream) {
    Args a{};
    a.logits = L.logits;
    a.stride = L.row_stride;
    a.targets = L.targets;
    a.bounds = L.bounds;
    a.rows = L.rows;
    a.choices = L.choices;
    a.top = L.top;
    a.logprob = L.logprob;
    a.entropy = L.entropy;
    a.rank = L.rank;
    a.top_ids = L.top_ids;
    a.top_logprobs = L.top_logprobs;
    a.status = L.status;
    a.cluster = 1;
    // As many warps as the row has 4 KB, up to 16; with too few rows to give
    // every SM one, 8 warps and a cluster of CTAs for what is longer.
    const uint64_t parts = ((uint64_t)L.choices * (L.bf16 ? 2 : 4) + 16 + 4095) / 4096;
    const uint32_t most = L.rows < L.num_sms ? 8u : 16u;
    uint32_t warps = 1;
    while (warps < most && warps < parts) warps *= 2;
    while (a.cluster < 8 && (uint64_t)L.rows * a.cluster * 2 <= 2ull * L.num_sms && (uint64_t)warps * a.cluster < parts)
        a.cluster *= 2;
    return L.bf16 ? launch_warps<true>(a, warps, stream) : launch_warps<false>(a, warps, stream);
}

}  // namespace pp
