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
// A thread copies 8 vectors of 16 bytes into shared memory (cp.async) and looks at
// them several times (maximum, sums, rank, alternatives) in short loops: nothing
// waits for another thread's copies, and the loops stay in the instruction cache,
// which the same code unrolled over registers did not (4096 rows of 32768, with the
// bound of that time: 154 us against 95).  One buffer a CTA leaves room for five CTAs
// an SM, which hide the copies better than a second buffer with three (117 us).  NW
// warps take 4 KB each of a row; a longer row is taken in steps, with a barrier after
// the first, or by a cluster of up to 8 CTAs that merge through their shared memory,
// when there are few rows.
//
// Alternatives: with q = ceil(k / NW), take every warp's q-th largest lane maximum;
// the ceil(k / q)-th largest of these is reached by at least k logits, so it is no
// larger than the k-th best.  Only logits from the best such bound on are candidates
// (on random rows one or two times k of a step's); they wait in a buffer a warp until
// the row ends; a warp whose buffer is half full keeps its best k.  A candidate's
// place in the list is the number of candidates ahead of it, which one thread each
// counts; the order in which they were found does not matter.
//
// Where a warp finds more candidates in a step than its buffer holds, the block takes
// the maximum of its part of the row k times instead.  That happens
//   - where many logits are equal or come in rising order: 4096 rows of 32768, 5
//     alternatives, 660 us rising and 770 all equal, instead of 76 (searching them with a
//     better bound took 450, but its registers cost random rows 6 to 30 %);
//   - where fewer lanes or warps hold logits than the bound counts, so that it stays -inf:
//     heads and windows of a few times k columns, and the last CTA of a cluster if its
//     part is short.  4096 rows of 128 bf16: 31 us with 20 alternatives and 43 with 32
//     instead of 10 with 5; 8 rows of 50257 with 20: 20 us instead of 9 for 65536; 500
//     columns of 4096 rows of 32768 with 8: 99 us instead of 34 without alternatives.
//
// Bound by issue slots and latency: 4096 rows of 32768 bf16 with 5 alternatives 76 us,
// 3.5 TB/s, 75 % of issue slots (15.5 warp instructions per 32 logits: 9 for maximum
// and sums, 2 the rank, 4.5 alternatives; alone they take 51, 8 and 18 us); in f32 142;
// 2048 of 131072 121 us, 4.4 TB/s; few rows by latency: 8 of 131072 with 20 alternatives
// 10 us; 2304 windows of up to 1024 f32 8 us.  With a barrier a step 81 and 140 us; with
// the least of the first ceil(k / q) warps' values as the bound, twice the candidates, 100.
// In f32 with 8 warps, 8 bytes of spills.
// Candidates pushed lane by lane, with an atomic each, instead of warp by warp: 98.
#include <math_constants.h>

#include "common.cuh"
#include "../host/internal.h"

namespace pp {
namespace {

constexpr int kVecs = 8;              // 16-byte vectors of a thread in a step
constexpr uint32_t kCandidates = 64;  // of a warp
constexpr uint32_t kMostWarps = 8;    // of a CTA
constexpr float kLog2e = 1.4426950408889634f;

struct Args {
    const void* logits;
    uint64_t stride;
    const int32_t* targets;
    const uint32_t* bounds;
    uint32_t choices, top, cluster;
    float* logprob;
    float* entropy;
    uint32_t* rank;
    uint32_t* top_ids;
    float* top_logprobs;
    uint32_t* status;
};

// What a thread or a CTA knows of a row; the threads of a warp have one m.
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

// Element i of a vector in shared memory, i not known beforehand.
template <bool BF>
__device__ __forceinline__ float picked(const uint4* p, int i) {
    if constexpr (BF) return bf16_lo_to_f32(reinterpret_cast<const uint16_t*>(p)[i]);
    else return reinterpret_cast<const float*>(p)[i];
}

// 1 in each half where a > b, as bf16; NaN gives 0.
__device__ __forceinline__ uint32_t above_bf16x2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("set.gt.bf16x2.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
__device__ __forceinline__ uint32_t add_bf16x2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("add.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
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

// Floats of shared memory that only rise, as integers in their order.
__device__ __forceinline__ int rising(float x) {
    const int b = __float_as_int(x);
    return b ^ (b >> 31 & 0x7fffffff);
}
__device__ __forceinline__ float rising_value(int k) { return __int_as_float(k ^ (k >> 31 & 0x7fffffff)); }

// The list of the best 32 candidates, by all of the block; nothing is written beyond them.
__device__ __noinline__ void sort_candidates(const unsigned long long* cand, uint32_t count, unsigned long long* list) {
    for (uint32_t j = threadIdx.x; j < count; j += blockDim.x) {
        const unsigned long long mine = cand[j];
        uint32_t place = 0;
#pragma unroll 4
        for (uint32_t i = 0; i < count; ++i) place += cand[i] > mine;
        if (place < 32) list[place] = mine;
    }
}

// Keeps the best k of a warp's candidates, by the warp; returns how many there are.
__device__ __noinline__ uint32_t keep_best(unsigned long long* cand, uint32_t count, uint32_t k) {
    const uint32_t lane = threadIdx.x & 31;
    __syncwarp();  // other lanes' candidates
    const unsigned long long a = lane < count ? cand[lane] : 0ull, b = lane + 32 < count ? cand[lane + 32] : 0ull;
    uint32_t place_a = 0, place_b = 0;
    for (uint32_t i = 0; i < count; ++i) {
        place_a += cand[i] > a;
        place_b += cand[i] > b;
    }
    __syncwarp();
    if (a && place_a < k) cand[place_a] = a;
    if (b && place_b < k) cand[place_b] = b;
    __syncwarp();
    return min(count, k);
}

template <bool BF, int NW>
__global__ void __launch_bounds__(32 * NW) logprobs_kernel(const Args a) {
    constexpr int EPV = BF ? 8 : 4;                    // elements of a vector
    constexpr uint32_t T = 32 * NW, STEP = T * kVecs;  // vectors a CTA takes at a time
    constexpr int kLow = (int)0x807fffff;              // rising(-inf)
    extern __shared__ uint4 s_row[];                   // a step, vector v of thread t at v T + t
    __shared__ int s_top[NW];
    __shared__ volatile int s_reached[NW];             // only rises: any value read is a bound
    __shared__ unsigned long long s_cand[NW * kCandidates], s_all[NW * kCandidates], s_list[32], s_best[NW];
    __shared__ uint32_t s_found[NW];
    __shared__ Part s_part[NW], s_cta;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t row = a.cluster > 1 ? blockIdx.x / a.cluster : blockIdx.x, part = a.cluster > 1 ? cluster_rank() : 0u;
    const uint32_t k = a.top;
    if (warp == 0) s_list[lane] = 0ull;
    const uint32_t q = (k + NW - 1) / NW;  // lane maxima of a warp that have to reach the bound
    const uint32_t bounding = k ? (k + q - 1) / q : 0u;
    pdl_wait_primary();
    const uint64_t base = (uint64_t)row * a.stride;
    int lo = 0, n = (int)a.choices;  // columns are below 2^31
    if (a.bounds) {
        const uint32_t from = a.bounds[2 * row], count = a.bounds[2 * row + 1];
        const bool fits = (uint64_t)from + count <= a.choices;
        if (!fits && threadIdx.x == 0 && part == 0 && a.status) atomicOr(a.status, PP_DEV_WINDOW_RANGE);
        lo = fits ? (int)from : 0;
        n = fits ? (int)count : 0;
    }
    const int hi = lo + n;
    // Vectors lie on 16-byte boundaries of memory: vector v holds the columns first + v * EPV ...
    const char* row_ptr = reinterpret_cast<const char*>(a.logits) + base * (BF ? 2 : 4);
    const int first = lo - (int)((reinterpret_cast<uint64_t>(row_ptr) + (uint64_t)lo * (BF ? 2 : 4)) % 16 / (BF ? 2 : 4));
    const uint32_t vectors = n ? ((uint32_t)(hi - first) + EPV - 1) / EPV : 0u;

    auto fetch = [&](uint32_t v0) {
        uint4* to = s_row + threadIdx.x;
        const int col0 = first + (int)(v0 + threadIdx.x) * EPV;
        const char* from = row_ptr + (int64_t)col0 * (BF ? 2 : 4);
        if (first + (int)v0 * EPV >= lo && v0 + STEP <= vectors && first + (int)(v0 + STEP) * EPV <= hi) {
#pragma unroll
            for (int v = 0; v < kVecs; ++v) cp_async16(to + v * T, from + v * T * 16);
            return;
        }
#pragma unroll 1
        for (int v = 0; v < kVecs; ++v, to += T, from += T * 16) {
            const uint32_t at = v0 + v * T + threadIdx.x;
            const int col = col0 + v * T * EPV;
            if (at < vectors && col >= lo && col + EPV <= hi) {
                cp_async16(to, from);
                continue;
            }
            const uint32_t none = BF ? 0xff80ff80u : 0xff800000u;  // -inf: an end of the window, or nothing
            *to = make_uint4(none, none, none, none);
            if (at >= vectors) continue;
            for (int i = 0; i < EPV; ++i)
                if (col + i >= lo && col + i < hi) {
                    const uint32_t bits = __float_as_uint(load_logit<BF>(a.logits, base + col + i));
                    if constexpr (BF) reinterpret_cast<uint16_t*>(to)[i] = (uint16_t)(bits >> 16);
                    else reinterpret_cast<uint32_t*>(to)[i] = bits;
                }
        }
    };
    const uint32_t stride = a.cluster * STEP;
    if (part * STEP < vectors) fetch(part * STEP);

    const int t = a.targets[row];
    const bool inside = t >= lo && t < hi;
    const float xt = inside ? load_logit<BF>(a.logits, base + t) : -CUDART_INF_F;
    // ahead of the target: x > xt behind it, x >= xt before it.  A NaN or -inf target is counted by itself, below.
    const bool ordinary = inside && xt > -CUDART_INF_F;

    Part p{-CUDART_INF_F, 0.f, 0.f, 0.f, 0u};
    const uint4* x = s_row + threadIdx.x;
    unsigned long long* cand = s_cand + warp * kCandidates;
    uint32_t found = 0;  // candidates of the warp
    float bound = -CUDART_INF_F;
    bool over = false;  // candidates did not fit: the list is found in the row again
    for (uint32_t v0 = part * STEP; v0 < vectors; v0 += stride) {
        cp_async_wait_all();
        float top = -CUDART_INF_F;
        if constexpr (BF) {
            uint32_t most = 0xff80ff80u;
#pragma unroll
            for (int v = 0; v < kVecs; ++v) {
                const uint4 y = x[v * T];
                most = max_bf16x2(max_bf16x2(most, max_bf16x2(y.x, y.y)), max_bf16x2(y.z, y.w));
            }
            top = fmaxf(bf16_lo_to_f32(most), bf16_hi_to_f32(most));
        } else {
#pragma unroll
            for (int v = 0; v < kVecs; ++v) top = fmaxf(top, vector_max<false>(x[v * T]));
        }
        const int key = rising(top);
        const int warp_key = __reduce_max_sync(0xffffffffu, key);
        const float warp_top = rising_value(warp_key);
        if (k) {
            int reached = warp_key;
            if (q > 8) {
                reached = __shfl_sync(0xffffffffu, sort32(key, lane), q - 1);
            } else {
                uint32_t left = 0xffffffffu;  // lanes not taken yet
                for (uint32_t i = 1; i < q; ++i) {
                    const uint32_t best = __ballot_sync(0xffffffffu, (left >> lane & 1u) && key == reached);
                    left &= ~(best & (0u - best));
                    reached = __reduce_max_sync(0xffffffffu, left >> lane & 1u ? key : kLow);
                }
            }
            if (lane == 0 && (v0 == part * STEP || reached > s_reached[warp])) s_reached[warp] = reached;
        }
        float m = fmaxf(p.m, warp_top);
        if (v0 == part * STEP) {  // the warps start from one maximum and bound, and then go their own ways
            if (lane == 0) s_top[warp] = warp_key;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < NW; ++w) m = fmaxf(m, rising_value(s_top[w]));
        }
        if (k) {
            if (found > kCandidates / 2) {
                over = over || found > kCandidates;
                found = keep_best(cand, min(found, kCandidates), k);
                if (found == k) bound = fmaxf(bound, order_value(cand[k - 1]));
            }
            // the `bounding`-th largest of what the warps have reached
            const int mine = s_reached[lane % NW];
            uint32_t larger = 0;
#pragma unroll
            for (int w = 0; w < NW; ++w) {
                const int other = __shfl_sync(0xffffffffu, mine, w);
                larger += other > mine || (other == mine && w < (int)(lane % NW));
            }
            const uint32_t who = __ballot_sync(0xffffffffu, larger == bounding - 1);
            bound = fmaxf(bound, rising_value(__shfl_sync(0xffffffffu, mine, __ffs(who) - 1)));
        }
        raise(p, m);
        // y = x log2(e) - r with r = m log2(e) rounded: all e come out 2^slip too large, which is taken back below
        const float ref = m > -CUDART_INF_F ? m : 0.f;  // nothing but -inf so far (or NaN, which has to show in s)
        const float r = ref * kLog2e, slip = fmaf(ref, kLog2e, -r);
        const uint64_t neg = f2_pack(-r, -r), l2e = f2_pack(kLog2e, kLog2e);
        // No x is taken below `low`, at least 119 under the maximum also as bf16: exp2 of its y is 0, and so is their
        // product, which that of -inf would not be.  Beyond 2^20 the slip is no small number.
        const float low = ref - 120.f - 0.01f * fabsf(ref);
        const bool plain = fabsf(ref) < 1048576.f;
        const uint32_t low2 = pack_bf16x2(low, low);
        uint64_t s0 = 0ull, s1 = 0ull, d0 = 0ull, d1 = 0ull;
        auto add = [&](const uint4& y4) {
            const uint32_t w[4] = {y4.x, y4.y, y4.z, y4.w};
#pragma unroll
            for (int i = 0; i < EPV; i += 2) {
                float x0, x1, y0, y1;
                if constexpr (BF) {
                    uint32_t u;
                    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(u) : "r"(w[i / 2]), "r"(low2));
                    x0 = bf16_lo_to_f32(u);
                    x1 = bf16_hi_to_f32(u);
                } else {
                    asm("max.NaN.f32 %0, %1, %2;" : "=f"(x0) : "f"(__uint_as_float(w[i])), "f"(low));
                    asm("max.NaN.f32 %0, %1, %2;" : "=f"(x1) : "f"(__uint_as_float(w[i + 1])), "f"(low));
                }
                uint64_t y2;
                asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(y2) : "l"(f2_pack(x0, x1)), "l"(l2e), "l"(neg));
                f2_unpack(y2, y0, y1);
                const uint64_t e2 = f2_pack(fast_exp2(y0), fast_exp2(y1));
                uint64_t& s = i & 2 ? s1 : s0;
                uint64_t& d = i & 2 ? d1 : d0;
                s = f2_add(s, e2);
                asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(d) : "l"(e2), "l"(y2));
            }
        };
        if (warp_top < m && plain) {
#pragma unroll 2
            for (int v = 0; v < kVecs; ++v) add(x[v * T]);
        } else {  // the warp holds the maximum, which is counted, not summed (or -inf and NaN only, or huge numbers)
#pragma unroll 1
            for (int v = 0; v < kVecs; ++v) {
                const uint4 y4 = x[v * T];
                if (vector_max<BF>(y4) < m && plain) {
                    add(y4);
                    continue;
                }
                float es[2] = {0.f, 0.f}, ed[2] = {0.f, 0.f};
#pragma unroll
                for (int i = 0; i < EPV; ++i) {
                    const float e = element<BF>(y4, i);
                    const float y = fmaxf((e - ref) * kLog2e, -160.f), f = e == m ? 0.f : fast_exp2(e == e ? y : e);
                    p.c += e == m ? 1.f : 0.f;
                    es[i & 1] += f;
                    ed[i & 1] += f * y;
                }
                p.s += es[0] + es[1];
                p.d -= (ed[0] + ed[1]) * 0.6931471805599453f;
            }
        }
        if (plain) {
            float e0, e1, e2, e3;
            f2_unpack(f2_add(s0, s1), e0, e1);
            f2_unpack(f2_add(d0, d1), e2, e3);
            const float sum = e0 + e1, back = fast_exp2(-slip);
            p.s += sum * back;
            p.d -= (e2 + e3 - slip * sum) * back * 0.6931471805599453f;
        }
        if (ordinary && warp_top >= xt) {
            if constexpr (BF) {
                // what lies before the target is ahead if it is larger than the number below xt
                const uint32_t bits = __float_as_uint(xt) >> 16;
                const uint32_t below = (bits & 0x7fffu) == 0 ? 0x8001u : bits & 0x8000u ? bits + 1 : bits - 1;
                const uint32_t xt2 = bits * 0x10001u, below2 = below * 0x10001u;
                uint32_t ahead2 = 0;  // two bf16 counts, at most 32 each
                int col = first + (int)(v0 + threadIdx.x) * EPV;
#pragma unroll 4
                for (int v = 0; v < kVecs; ++v, col += T * EPV) {
                    const uint4 y4 = x[v * T];
                    const uint32_t than = col + EPV <= t ? below2 : xt2;
                    ahead2 = add_bf16x2(ahead2, add_bf16x2(above_bf16x2(y4.x, than), above_bf16x2(y4.y, than)));
                    ahead2 = add_bf16x2(ahead2, add_bf16x2(above_bf16x2(y4.z, than), above_bf16x2(y4.w, than)));
                }
                p.ahead += (uint32_t)(bf16_lo_to_f32(ahead2) + bf16_hi_to_f32(ahead2));
            } else {
#pragma unroll 2
                for (int v = 0; v < kVecs; ++v) {
                    const uint4 y4 = x[v * T];
                    const int col = first + (int)(v0 + v * T + threadIdx.x) * EPV;
#pragma unroll
                    for (int i = 0; i < EPV; ++i) {
                        const float e = element<false>(y4, i);
                        p.ahead += col + EPV <= t ? e >= xt : e > xt;
                    }
                }
            }
            // its own vector: what equals it and comes before it
            const uint32_t at = (uint32_t)(t - first) / EPV - v0;  // vector of the step, if it is one
            if (at < STEP && at % T == threadIdx.x) {
#pragma unroll 1
                for (uint32_t i = 0; i < (uint32_t)(t - first) % EPV; ++i) p.ahead += picked<BF>(x + at / T * T, i) == xt;
            }
        }
        if (k && __any_sync(0xffffffffu, top >= bound && top > -CUDART_INF_F)) {
#pragma unroll 1
            for (int v = 0; v < kVecs; ++v) {
                const uint4 y4 = x[v * T];
                const float vm = vector_max<BF>(y4);
                if (!__any_sync(0xffffffffu, vm >= bound && vm > -CUDART_INF_F)) continue;
                const int col = first + (int)(v0 + v * T + threadIdx.x) * EPV;
                uint32_t have = 0;  // candidates of the lane's vector, as bits
#pragma unroll
                for (int i = 0; i < EPV; ++i) {
                    const float e = element<BF>(y4, i);
                    have |= (e >= bound && e > -CUDART_INF_F ? 1u : 0u) << i;
                }
                for (uint32_t who; (who = __ballot_sync(0xffffffffu, have != 0)) != 0; have &= have - 1) {
                    const uint32_t at = found + __popc(who & ((1u << lane) - 1u));
                    found += __popc(who);
                    if (have && at < kCandidates) {
                        const int i = __ffs(have) - 1;
                        cand[at] = order_of(picked<BF>(x + v * T, i), (uint32_t)(col + i));
                    }
                }
            }
        }
        if (v0 + stride < vectors) fetch(v0 + stride);
    }
    if (k) {
        // What has fallen behind the bound goes; the rest of all warps, one after another.
        over = over || found > kCandidates;
        found = min(found, kCandidates);
        __syncwarp();
        const bool has_a = lane < found && order_value(cand[lane]) >= bound;
        const bool has_b = lane + 32 < found && order_value(cand[lane + 32]) >= bound;
        const uint32_t as = __ballot_sync(0xffffffffu, has_a), bs = __ballot_sync(0xffffffffu, has_b);
        const uint32_t below = (1u << lane) - 1u;
        if (lane == 0) s_found[warp] = __popc(as) + __popc(bs);
        over = __syncthreads_or(over);
        if (!over) {
            uint32_t from = 0, all = 0;
#pragma unroll
            for (int w = 0; w < NW; ++w) {
                from += w < (int)warp ? s_found[w] : 0u;
                all += s_found[w];
            }
            if (has_a) s_all[from + __popc(as & below)] = cand[lane];
            if (has_b) s_all[from + __popc(as) + __popc(bs & below)] = cand[lane + 32];
            __syncthreads();
            sort_candidates(s_all, all, s_list);
        } else {
            unsigned long long* list = s_list;
            unsigned long long prev = ~0ull;
            for (uint32_t j = 0; j < k; ++j) {
                unsigned long long best = 0;
                for (uint32_t v0 = part * STEP; v0 < vectors; v0 += stride) {
                    const int64_t from = max((int64_t)lo, first + (int64_t)v0 * EPV);
                    const int64_t to = min((int64_t)hi, first + ((int64_t)v0 + STEP) * EPV);
                    for (int64_t i = from + threadIdx.x; i < to; i += T) {
                        const float e = load_logit<BF>(a.logits, base + i);
                        if (!(e > -CUDART_INF_F)) continue;
                        const unsigned long long o = order_of(e, (uint32_t)i);
                        if (o < prev && o > best) best = o;
                    }
                }
#pragma unroll
                for (int o = 16; o; o >>= 1) {
                    const unsigned long long y = __shfl_xor_sync(0xffffffffu, best, o);
                    best = best > y ? best : y;
                }
                if (lane == 0) s_best[warp] = best;
                __syncthreads();
                for (int w = 0; w < NW; ++w) best = best > s_best[w] ? best : s_best[w];
                if (threadIdx.x == 0) list[j] = best;
                prev = best;
                __syncthreads();
            }
            if (warp == 0 && lane >= k) list[lane] = 0ull;
        }
    }
    // a NaN target comes behind what is not NaN, a -inf one behind what is larger; of its own kind, behind lower columns
    if (inside && !ordinary) {
        for (int64_t i = lo + (int64_t)(part * 32 * NW + threadIdx.x); i < hi; i += a.cluster * 32 * NW) {
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
    if (warp == 0 && NW > 1) {
        p = lane < NW ? s_part[lane] : Part{-CUDART_INF_F, 0.f, 0.f, 0.f, 0u};
        float m = p.m;
#pragma unroll
        for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        raise(p, m);
#pragma unroll
        for (int o = NW / 2; o; o >>= 1) {
            p.s += __shfl_xor_sync(0xffffffffu, p.s, o);
            p.c += __shfl_xor_sync(0xffffffffu, p.c, o);
            p.d += __shfl_xor_sync(0xffffffffu, p.d, o);
            p.ahead += __shfl_xor_sync(0xffffffffu, p.ahead, o);
        }
    }
    if (NW == (int)kMostWarps && a.cluster > 1) {
        if (threadIdx.x == 0) s_cta = p;
        cluster_sync();
        if (part == 0) {
            if (warp == 0) {  // lane r fetches CTA r's part
                if (lane < a.cluster && lane) {
                    const float ms = __uint_as_float(ld_peer(&s_cta.m, lane)), ss = __uint_as_float(ld_peer(&s_cta.s, lane));
                    const float cs = __uint_as_float(ld_peer(&s_cta.c, lane)), ds = __uint_as_float(ld_peer(&s_cta.d, lane));
                    p = Part{ms, ss, cs, ds, ld_peer(&s_cta.ahead, lane)};
                } else if (lane) {
                    p = Part{-CUDART_INF_F, 0.f, 0.f, 0.f, 0u};
                }
                float m = p.m;
#pragma unroll
                for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
                raise(p, m);
#pragma unroll
                for (int o = 4; o; o >>= 1) {
                    p.s += __shfl_xor_sync(0xffffffffu, p.s, o);
                    p.c += __shfl_xor_sync(0xffffffffu, p.c, o);
                    p.d += __shfl_xor_sync(0xffffffffu, p.d, o);
                    p.ahead += __shfl_xor_sync(0xffffffffu, p.ahead, o);
                }
            }
            if (k && warp < a.cluster && lane < k) {  // a warp fetches a CTA's list
                const uint32_t* peer = reinterpret_cast<const uint32_t*>(&s_list[lane]);
                const unsigned long long l = ld_peer(peer, warp), h = ld_peer(peer + 1, warp);
                s_cand[warp * k + lane] = h << 32 | l;
            }
        }
        cluster_sync();  // the peers' shared memory has been read
        if (part != 0) return;
        if (k) {
            if (warp == 0) s_list[lane] = 0ull;
            __syncthreads();
            // missing entries are 0 and land behind the others, where the list is 0
            sort_candidates(s_cand, a.cluster * k, s_list);
            __syncthreads();
        }
    }
    if (warp != 0) return;
    p.s = __shfl_sync(0xffffffffu, p.s, 0);  // lane 0 has the row's; all of them write alternatives
    p.c = __shfl_sync(0xffffffffu, p.c, 0);
    p.m = __shfl_sync(0xffffffffu, p.m, 0);
    const bool nothing = !(p.m > -CUDART_INF_F && p.m < CUDART_INF_F) || p.s != p.s;
    const float s = p.s + (p.c - 1.f), lse = log1pf(s);  // of the sum, less m
    if (lane == 0) {
        a.logprob[row] = nothing ? CUDART_NAN_F : (xt - p.m) - lse;
        a.entropy[row] = nothing ? CUDART_NAN_F : lse + p.d / (1.f + s);
        a.rank[row] = inside ? p.ahead : (uint32_t)n;
    }
    if (lane < k) {
        const unsigned long long o = s_list[lane];
        a.top_ids[(uint64_t)row * k + lane] = o ? ~(uint32_t)o : 0xffffffffu;
        float lp = -CUDART_INF_F;
        if (o) lp = nothing ? CUDART_NAN_F : (order_value(o) - p.m) - lse;
        a.top_logprobs[(uint64_t)row * k + lane] = lp;
    }
}

template <bool BF, int NW>
cudaError_t launch(const Args& a, uint32_t rows, cudaStream_t stream) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(rows * a.cluster);
    cfg.blockDim = dim3(32 * NW);
    cfg.dynamicSmemBytes = NW * 32 * kVecs * 16;
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
cudaError_t launch_warps(const Args& a, uint32_t rows, uint32_t warps, cudaStream_t stream) {
    switch (warps) {
        case 1: return launch<BF, 1>(a, rows, stream);
        case 2: return launch<BF, 2>(a, rows, stream);
        case 4: return launch<BF, 4>(a, rows, stream);
        default: return launch<BF, kMostWarps>(a, rows, stream);
    }
}

}  // namespace

cudaError_t launch_token_logprobs(const LogprobsLaunch& L, cudaStream_t stream) {
    Args a{};
    a.logits = L.logits;
    a.stride = L.row_stride;
    a.targets = L.targets;
    a.bounds = L.bounds;
    a.choices = L.choices;
    a.top = L.top;
    a.logprob = L.logprob;
    a.entropy = L.entropy;
    a.rank = L.rank;
    a.top_ids = L.top_ids;
    a.top_logprobs = L.top_logprobs;
    a.status = L.status;
    a.cluster = 1;
    // As many warps as the row has 4 KB, up to 8; with too few rows to give every SM
    // one, 8 warps and a cluster of CTAs for what is longer.  Always 8 warps: 4096 rows
    // of 1000 take 48 us instead of 12; always 1: 256 rows of 32768 48 instead of 13.
    // Without clusters 8 rows of 131072 take 30 us instead of 10.
    const uint64_t parts = ((uint64_t)L.choices * (L.bf16 ? 2 : 4) + 4095) / 4096;
    uint32_t warps = 1;
    while (warps < kMostWarps && warps < parts) warps *= 2;
    while (a.cluster < 8 && (uint64_t)L.rows * a.cluster <= L.num_sms && (uint64_t)warps * a.cluster < parts)
        a.cluster *= 2;
    return L.bf16 ? launch_warps<true>(a, L.rows, warps, stream) : launch_warps<false>(a, L.rows, warps, stream);
}

}  // namespace pp
