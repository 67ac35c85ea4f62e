// Attention of whole prompts: the plan of a batch of packed sequences, and the
// CUDA-core kernel that takes f32 tensors and rows off the 16-byte grid.
#include <math_constants.h>

#include "prompt.cuh"

namespace pp {
namespace {

// ----------------------------------------------------------------- the plan
//
// One CTA, a thread an entry (up to 1024; a fixed 1024 took 0.7 us longer in small
// batches); it is a chain of a few loads and barriers, 3 to 5 us, in which the
// attention is launched.  Cuts every sequence into entries of 2 * tpt query tokens,
// counts the steps each takes (a step is a key tile of both its query tiles, or two
// key tiles where only one has rows), and writes them longest first (64 classes
// of length), because the attention CTAs take items in this order as they
// become free: the last ones taken are the shortest.  Where the whole batch has
// fewer steps than it takes to keep every CTA busy with whole entries, entries of
// more than one and a half times their share are cut into equal pieces along the
// keys.  Pieces nearer to the share leave less room for the uneven last round (2048
// causal tokens of 16 heads of 128: 41 us at 1.5, 51 at 1; 512 tokens at the end of
// 32768, 16 heads on 2: 134 and 208); longer ones leave SMs without work (172 at 2).
// Uncut it takes 450 us, and one sequence of 8192, one head of 64, 109 against 38.
// Nothing is cut where no entry has kCutSteps, or where the longest would lose less
// than three: partials and their merge take about as long (768 tokens, 8 heads of 64,
// cut from 6 steps on: 20.5 us against 19.8; 1023 tokens, 32 heads on 8 of 128, 6 steps
// instead of 8: 34 against 29; one token over 2000 keys, 2 instead of 8: 20 against 29).
constexpr uint32_t kPlanThreads = 1024;  // at most
constexpr uint32_t kClasses = 64;
constexpr uint32_t kBaseMax = 2048;  // sequences whose first entries are kept in shared memory
constexpr uint32_t kCutSteps = 8;

struct PlanArgs {
    const uint32_t* q_starts;
    const uint32_t* kv_starts;
    unsigned char* ws;
    PromptWsLayout l;
    uint32_t sequences, q_tokens, kv_tokens, causal, tpt, kv_heads;
    uint32_t key[5];
    uint32_t* status;
};

// Exclusive scan over the block; `total` gets the sum.
__device__ __forceinline__ uint32_t block_scan(uint32_t x, uint32_t* warp_tot, uint32_t& total) {
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    uint32_t inc = x;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t y = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += y;
    }
    __syncthreads();  // the totals of the scan before have been read
    if (lane == 31) warp_tot[w] = inc;
    __syncthreads();
    if (w == 0) {
        uint32_t t = lane < (int)(blockDim.x >> 5) ? warp_tot[lane] : 0u;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t y = __shfl_up_sync(0xffffffffu, t, o);
            if (lane >= o) t += y;
        }
        warp_tot[lane] = t;
    }
    __syncthreads();
    total = warp_tot[31];
    return inc - x + (w ? warp_tot[w - 1] : 0u);
}

struct Whole {  // an entry before cutting
    PromptEntry p;
    uint32_t tiles, steps;
};

__device__ __forceinline__ Whole entry_of(const PlanArgs& a, const uint32_t* seq_base, uint32_t e) {
    Whole w;
    uint32_t lo = 0, hi = a.sequences;  // seq_base[lo] <= e < seq_base[hi]
    while (hi - lo > 1) {
        const uint32_t mid = lo + (hi - lo) / 2;
        if (seq_base[mid] <= e) lo = mid;
        else hi = mid;
    }
    PromptEntry& p = w.p;
    p.q0 = a.q_starts[lo];
    p.nq = a.q_starts[lo + 1] - p.q0;
    p.k0 = a.kv_starts[lo];
    p.nk = a.kv_starts[lo + 1] - p.k0;
    p.tok0 = (e - seq_base[lo]) * 2 * a.tpt;
    p.kv_begin = 0;
    p.kv_end = prompt_visible(p, min(p.nq, p.tok0 + 2 * a.tpt) - 1, a.causal);
    w.tiles = max(1u, p.kv_end / kPromptKeyTile + (p.kv_end % kPromptKeyTile != 0));
    w.steps = p.tok0 + a.tpt >= p.nq ? (w.tiles + 1) / 2 : w.tiles;
    return w;
}

__global__ void __launch_bounds__(kPlanThreads) prompt_plan_kernel(const PlanArgs a) {
    __shared__ uint32_t warp_tot[32], hist[kClasses], cursor[kClasses], base_s[kBaseMax + 1];
    __shared__ unsigned long long warp_work[32];
    __shared__ uint32_t longest, slots, cuts;
    const uint32_t t = threadIdx.x, lane = t & 31, threads = blockDim.x;
    PromptHeader* hdr = reinterpret_cast<PromptHeader*>(a.ws);
    uint32_t* seq_base = a.sequences <= kBaseMax ? base_s : reinterpret_cast<uint32_t*>(a.ws + a.l.seq_base);
    PromptEntry* entries = reinterpret_cast<PromptEntry*>(a.ws + a.l.entries);
    PromptEntry* cut_list = reinterpret_cast<PromptEntry*>(a.ws + a.l.cuts);
    if (t == 0) longest = slots = cuts = 0;
    for (uint32_t c = t; c < kClasses; c += threads) hist[c] = 0;
    if (t < 32) warp_work[t] = 0;
    // launched as a programmatic dependent: the kernels before may still read
    // the workspace or write the starts.  A dependent attention launch may
    // start now; it waits for this kernel before it reads the plan.
    pdl_wait_primary();
    pdl_launch_dependents();
    int bad = 0;
    uint32_t n = 0;
    for (uint32_t b0 = 0; b0 < a.sequences; b0 += threads) {
        const uint32_t b = b0 + t;
        uint32_t nq = 0;
        if (b < a.sequences) {
            const uint32_t q0 = a.q_starts[b], q1 = a.q_starts[b + 1], k0 = a.kv_starts[b], k1 = a.kv_starts[b + 1];
            if (q1 < q0 || q1 > a.q_tokens || k1 < k0 || k1 > a.kv_tokens) bad = 1;
            else nq = q1 - q0;
        }
        uint32_t tot;
        const uint32_t at = block_scan(nq / (2 * a.tpt) + (nq % (2 * a.tpt) != 0), warp_tot, tot);
        if (b < a.sequences) seq_base[b] = n + at;
        n += tot;
    }
    if (__syncthreads_or(bad)) {
        n = 0;
        if (t == 0 && a.status) atomicOr(a.status, PP_DEV_LENGTH_RANGE);
    }
    if (t == 0) seq_base[a.sequences] = n;
    __syncthreads();
    Whole first;  // the thread's first entry, often its only one
    if (t < n) first = entry_of(a, seq_base, t);
    {
        unsigned long long mine = 0;
        uint32_t far = 0;
        for (uint32_t e = t; e < n; e += threads) {
            const uint32_t steps = e == t ? first.steps : entry_of(a, seq_base, e).steps;
            mine += steps;
            far = max(far, steps);
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) {
            mine += __shfl_xor_sync(0xffffffffu, mine, o);
            far = max(far, __shfl_xor_sync(0xffffffffu, far, o));
        }
        if (lane == 0) {
            warp_work[t >> 5] = mine;
            if (far) atomicMax(&longest, far);
        }
    }
    __syncthreads();
    unsigned long long all = warp_work[lane];
#pragma unroll
    for (int o = 16; o; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
    const float share = __fdividef((float)all * a.kv_heads, a.l.max_ctas);  // to a few units of 2^-24, which is plenty
    const uint32_t most = longest;
    const uint32_t piece = (uint32_t)fminf(fmaxf(2.f, ceilf(1.5f * share)), 1e9f);
    const uint32_t limit = most < kCutSteps || most < piece + 3 ? most : piece;
    const float per_step = __fdividef((float)kClasses, most);
    // pieces of an entry and the class of their length
    auto cut = [&](const Whole& w, uint32_t& pieces) {
        pieces = 1;
        uint32_t len = w.steps;
        if (len > limit) {
            pieces = (len + limit - 1) / limit;
            len = (len + pieces - 1) / pieces;
        }
        return kClasses - 1 - min(kClasses - 1, (uint32_t)((len - 1) * per_step));
    };
    for (uint32_t e = t; e < n; e += threads) {
        uint32_t pieces;
        const uint32_t c = e == t ? cut(first, pieces) : cut(entry_of(a, seq_base, e), pieces);
        atomicAdd(&hist[c], pieces);
    }
    __syncthreads();
    if (t < 32) {
        uint32_t lo = hist[2 * t], hi = hist[2 * t + 1], inc = lo + hi;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t y = __shfl_up_sync(0xffffffffu, inc, o);
            if (t >= o) inc += y;
        }
        cursor[2 * t] = inc - lo - hi;
        cursor[2 * t + 1] = inc - hi;
        if (t == 31) {
            hdr->n_items = inc * a.kv_heads;
            hdr->next = 0;
#pragma unroll
            for (int i = 0; i < 5; ++i) hdr->key[i] = a.key[i];
        }
    }
    __syncthreads();
    for (uint32_t e = t; e < n; e += threads) {
        Whole w = e == t ? first : entry_of(a, seq_base, e);
        uint32_t pieces;
        const uint32_t at = atomicAdd(&cursor[cut(w, pieces)], pieces);
        PromptEntry p = w.p;
        p.n_splits = pieces;
        p.slot0 = p.pad[0] = p.pad[1] = 0;
        if (pieces > 1) {
            p.slot0 = atomicAdd(&slots, pieces);
            cut_list[atomicAdd(&cuts, 1u)] = p;
        }
        const uint32_t end = p.kv_end;
        for (uint32_t s = 0; s < pieces; ++s) {
            // equal pieces of whole tiles: none is empty, as s * tiles / pieces is strictly increasing
            p.split = s;
            p.kv_begin = (uint32_t)((uint64_t)w.tiles * s / pieces) * kPromptKeyTile;
            p.kv_end = s + 1 == pieces ? end : (uint32_t)((uint64_t)w.tiles * (s + 1) / pieces) * kPromptKeyTile;
            entries[at + s] = p;
        }
    }
    __syncthreads();
    if (t == 0) hdr->n_cuts = cuts;
}

// ------------------------------------------------------ the CUDA-core kernel
//
// A work unit is 64 query rows of an item.  256 threads as 16 x 16: thread
// (ty, tx) holds rows 4 ty .. 4 ty + 3; scores of keys tx + 16 j and channels
// 4 tx + 64 h.  Online softmax in base 2 over key tiles of 64, all of it in
// f32.  Products run two at a time on packed f32 pairs: pairs of channels for
// q k', pairs of output channels for p v.
//
// Bound by the packed multiply-adds (two issue slots each) and, with 16 warps an SM,
// by what hides their operands' latency: 4 sequences of 77 to 1000 tokens, 24 heads of
// 64, not causal: 266 us, 31 TFLOP/s of about 72; 2048 tokens, 8 heads of 128, causal:
// 306.  Copying the next tile meanwhile took them from 296 and 341.
constexpr int kRowsThreads = 256, kBN = 64;

template <bool BF>
__device__ __forceinline__ float4 load4(const void* p, uint64_t i, bool vec) {
    if constexpr (BF) {
        const uint16_t* s = reinterpret_cast<const uint16_t*>(p) + i;
        if (vec) {
            const uint2 u = *reinterpret_cast<const uint2*>(s);
            return make_float4(bf16_lo_to_f32(u.x), bf16_hi_to_f32(u.x), bf16_lo_to_f32(u.y), bf16_hi_to_f32(u.y));
        }
        return make_float4(bf16_lo_to_f32(s[0]), bf16_lo_to_f32(s[1]), bf16_lo_to_f32(s[2]), bf16_lo_to_f32(s[3]));
    } else {
        const float* s = reinterpret_cast<const float*>(p) + i;
        if (vec) return *reinterpret_cast<const float4*>(s);
        return make_float4(s[0], s[1], s[2], s[3]);
    }
}

template <bool BF>
__device__ __forceinline__ void store4(void* p, uint64_t i, float4 x) {
    if constexpr (BF) {
        uint2 u = make_uint2(pack_bf16x2(x.x, x.y), pack_bf16x2(x.z, x.w));
        uint16_t* s = reinterpret_cast<uint16_t*>(p) + i;
        *reinterpret_cast<uint2*>(s) = u;
    } else {
        *reinterpret_cast<float4*>(reinterpret_cast<float*>(p) + i) = x;
    }
}

template <int D>
struct RowsCfg {
    static constexpr int LD = D + 4;  // rows 4 banks apart: 8 lanes' float4 cover all banks
    static constexpr int KV = 64 * LD + 64 * D;  // a tile of keys and its values
    static constexpr int SMEM = (64 * LD + 2 * KV + 64 * (kBN + 4)) * 4;
};

template <int D, bool BF>
__global__ void __launch_bounds__(kRowsThreads, D == 64 ? 2 : 1) prompt_rows_kernel(const PromptArgs a) {
    using C = RowsCfg<D>;
    constexpr int H = D / 64;  // channel groups of 4 a thread holds
    extern __shared__ __align__(16) float sm[];
    float* sq = sm;
    float* skv = sq + 64 * C::LD;
    float* sp = skv + 2 * C::KV;
    __shared__ uint32_t s_next;
    const int t = threadIdx.x, tx = t & 15, ty = t >> 4;
    PromptHeader* hdr = reinterpret_cast<PromptHeader*>(a.ws);
    const PromptEntry* entries = reinterpret_cast<const PromptEntry*>(a.ws + a.l.entries);
    float* acc_ws = reinterpret_cast<float*>(a.ws + a.l.acc);
    float* ml_ws = reinterpret_cast<float*>(a.ws + a.l.ml);
    pdl_wait_primary();
    const uint32_t units = plan_header(a, blockIdx.x == 0 && t == 0).n_items * 4;
    uint32_t unit = blockIdx.x;
    while (unit < units) {
        const uint32_t item = unit >> 2, sub = unit & 3;
        const uint32_t at = item / a.kv_heads, head = item - at * a.kv_heads;
        const PromptEntry e = entries[at];
        const uint32_t tile = sub >> 1, row0 = (sub & 1) * kPromptSubRows;
        const uint32_t rows = min(a.tpt * a.group, row0 + kPromptSubRows);  // of the tile, up to this unit's end
        const uint32_t tile_tok = e.tok0 + tile * a.tpt;
        const bool any = row0 < rows && tile_tok + row0 / a.group < e.nq;
        if (any) {
            auto token_of = [&](uint32_t r) { return tile_tok + (row0 + r) / a.group; };
            auto live = [&](uint32_t r) { return row0 + r < rows && token_of(r) < e.nq; };
            for (int i = t; i < 64 * (D / 4); i += kRowsThreads) {
                const uint32_t r = i / (D / 4), c = i % (D / 4) * 4;
                float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
                if (live(r))
                    x = load4<BF>(a.q, (uint64_t)(e.q0 + token_of(r)) * a.q_ts +
                                           (uint64_t)(head * a.group + (row0 + r) % a.group) * a.q_hs + c, a.vec);
                *reinterpret_cast<float4*>(sq + r * C::LD + c) = x;
            }
            uint32_t lim[4];  // keys that row 4 ty + i sees, within this piece
            uint32_t last = 0, first = 0xffffffffu;
            float m[4], z[4];
            uint64_t acc[4][2 * H];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                lim[i] = live(4 * ty + i) ? min(e.kv_end, prompt_visible(e, token_of(4 * ty + i), a.causal)) : 0u;
                m[i] = -CUDART_INF_F;
                z[i] = 0.f;
#pragma unroll
                for (int j = 0; j < 2 * H; ++j) acc[i][j] = 0ull;
            }
            {  // keys that the unit's last row sees bound the loop; what its first row sees needs no mask
                const uint32_t r_last = min(min(e.nq - tile_tok, a.tpt) * a.group, rows) - 1 - row0;
                last = min(e.kv_end, prompt_visible(e, token_of(r_last), a.causal));
                first = min(e.kv_end, prompt_visible(e, token_of(0), a.causal));
            }
            // The next tile is copied while this one is used (f32 on the 16-byte grid; other rows are converted on the way).
            auto fetch = [&](uint32_t n0, float* sk) {
                float* sv = sk + 64 * C::LD;
                for (int i = t; i < 64 * (D / 4); i += kRowsThreads) {
                    const uint32_t r = i / (D / 4), c = i % (D / 4) * 4;
                    float *to_k = sk + r * C::LD + c, *to_v = sv + r * D + c;
                    if (n0 + r < last) {
                        const uint64_t row = (uint64_t)e.k0 + n0 + r;
                        const uint64_t at_k = row * a.k_ts + (uint64_t)head * a.k_hs + c;
                        const uint64_t at_v = row * a.v_ts + (uint64_t)head * a.v_hs + c;
                        if (!BF && a.vec) {
                            cp_async16(to_k, reinterpret_cast<const float*>(a.k) + at_k);
                            cp_async16(to_v, reinterpret_cast<const float*>(a.v) + at_v);
                            continue;
                        }
                        *reinterpret_cast<float4*>(to_k) = load4<BF>(a.k, at_k, a.vec);
                        *reinterpret_cast<float4*>(to_v) = load4<BF>(a.v, at_v, a.vec);
                    } else {
                        *reinterpret_cast<float4*>(to_k) = *reinterpret_cast<float4*>(to_v) = make_float4(0.f, 0.f, 0.f, 0.f);
                    }
                }
            };
            uint32_t buf = 0;
            if (e.kv_begin < last) fetch(e.kv_begin, skv);
            for (uint32_t n0 = e.kv_begin; n0 < last; n0 += kBN, buf ^= 1) {
                cp_async_wait_all();
                __syncthreads();  // the tile is there, and nobody reads the other one any more
                if (last - n0 > kBN) fetch(n0 + kBN, skv + (buf ^ 1) * C::KV);
                const float *sk = skv + buf * C::KV, *sv = sk + 64 * C::LD;
                uint64_t s2[4][4];
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) s2[i][j] = 0ull;
#pragma unroll 4
                for (int c = 0; c < D; c += 4) {
                    ulonglong2 qv[4], kv[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        qv[i] = *reinterpret_cast<const ulonglong2*>(sq + (4 * ty + i) * C::LD + c);
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        kv[j] = *reinterpret_cast<const ulonglong2*>(sk + (tx + 16 * j) * C::LD + c);
#pragma unroll
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            s2[i][j] = f2_fma(qv[i].y, kv[j].y, f2_fma(qv[i].x, kv[j].x, s2[i][j]));
                }
                const bool masked = n0 + kBN > first;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float s[4], top = -CUDART_INF_F;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        float lo, hi;
                        f2_unpack(s2[i][j], lo, hi);
                        s[j] = (lo + hi) * a.scale_log2;
                        if (n0 + tx + 16 * j >= lim[i]) s[j] = -CUDART_INF_F;
                        top = fmaxf(top, s[j]);
                    }
#pragma unroll
                    for (int o = 8; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
                    const float mn = fmaxf(m[i], top);
                    const float ref = mn == -CUDART_INF_F ? 0.f : mn;  // nothing seen yet: exp2(-inf) = 0
                    const float f = exp2f(m[i] - ref);
                    float sum = 0.f;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float p = exp2f(s[j] - ref);
                        sum += p;
                        sp[(4 * ty + i) * (kBN + 4) + tx + 16 * j] = p;
                    }
#pragma unroll
                    for (int o = 8; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
                    z[i] = z[i] * f + sum;
                    m[i] = mn;
                    const uint64_t f2 = f2_pack(f, f);
#pragma unroll
                    for (int j = 0; j < 2 * H; ++j) acc[i][j] = f2_mul(acc[i][j], f2);
                }
                __syncwarp();  // the rows of a half-warp are its own
                if (!masked) {
#pragma unroll 2
                    for (int n = 0; n < kBN; n += 4) {  // four keys' probabilities of a row in one load
                        float4 p4[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            p4[i] = *reinterpret_cast<const float4*>(sp + (4 * ty + i) * (kBN + 4) + n);
#pragma unroll
                        for (int u = 0; u < 4; ++u) {
                            ulonglong2 vv[H];
#pragma unroll
                            for (int h = 0; h < H; ++h)
                                vv[h] = *reinterpret_cast<const ulonglong2*>(sv + (n + u) * D + 64 * h + 4 * tx);
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                const float p = u == 0 ? p4[i].x : u == 1 ? p4[i].y : u == 2 ? p4[i].z : p4[i].w;
                                const uint64_t p2 = f2_pack(p, p);
#pragma unroll
                                for (int h = 0; h < H; ++h) {
                                    acc[i][2 * h] = f2_fma(p2, vv[h].x, acc[i][2 * h]);
                                    acc[i][2 * h + 1] = f2_fma(p2, vv[h].y, acc[i][2 * h + 1]);
                                }
                            }
                        }
                    }
                } else {
                    // a key that a row does not see leaves it alone whatever its value holds (0 * NaN is NaN)
                    const uint32_t end = min((uint32_t)kBN, last - n0);
                    for (uint32_t n = 0; n < end; ++n) {
                        ulonglong2 vv[H];
#pragma unroll
                        for (int h = 0; h < H; ++h)
                            vv[h] = *reinterpret_cast<const ulonglong2*>(sv + n * D + 64 * h + 4 * tx);
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            if (n0 + n >= lim[i]) continue;
                            const float p = sp[(4 * ty + i) * (kBN + 4) + n];
                            const uint64_t p2 = f2_pack(p, p);
#pragma unroll
                            for (int h = 0; h < H; ++h) {
                                acc[i][2 * h] = f2_fma(p2, vv[h].x, acc[i][2 * h]);
                                acc[i][2 * h + 1] = f2_fma(p2, vv[h].y, acc[i][2 * h + 1]);
                            }
                        }
                    }
                }
            }
            auto write_row = [&](int i, const float (&o)[4 * H], float sum) {
                const uint32_t r = 4 * ty + i;
                const uint64_t at = ((uint64_t)(e.q0 + token_of(r)) * a.heads + head * a.group + (row0 + r) % a.group) * D;
#pragma unroll
                for (int h = 0; h < H; ++h) {  // a row that sees no key: 0 / 0 = NaN
                    store4<BF>(a.out, at + 64 * h + 4 * tx,
                               make_float4(o[4 * h] / sum, o[4 * h + 1] / sum, o[4 * h + 2] / sum, o[4 * h + 3] / sum));
                }
            };
            if (e.n_splits == 1) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (!live(4 * ty + i)) continue;
                    float o[4 * H];
#pragma unroll
                    for (int j = 0; j < 2 * H; ++j) f2_unpack(acc[i][j], o[2 * j], o[2 * j + 1]);
                    write_row(i, o, z[i]);
                }
            } else {
                // partial of this piece, for prompt_merge_kernel
                const uint32_t srow = tile * kPromptTileRows + row0;
                auto slot_row = [&](uint32_t s, uint32_t r) {
                    return (uint64_t)((e.slot0 + s) * a.kv_heads + head) * a.l.slot_rows + srow + r;
                };
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (!live(4 * ty + i)) continue;
                    const uint64_t at = slot_row(e.split, 4 * ty + i);
#pragma unroll
                    for (int h = 0; h < H; ++h)
                        *reinterpret_cast<ulonglong2*>(acc_ws + at * D + 64 * h + 4 * tx) =
                            make_ulonglong2(acc[i][2 * h], acc[i][2 * h + 1]);
                    if (tx == 0) {
                        ml_ws[2 * at] = m[i];
                        ml_ws[2 * at + 1] = z[i];
                    }
                }
            }
        }
        __syncthreads();
        if (t == 0) {
            const uint32_t got = atomicAdd(&hdr->next, 1u);
            if (got == units - 1) hdr->next = 0;  // every CTA has taken its last: ready for the next call
            s_next = got + gridDim.x;
        }
        __syncthreads();
        unit = s_next;
    }
}

// --------------------------------------------------- the pieces of cut rows
//
// A warp merges four rows side by side: out = sum_s 2^(m_s - m) acc_s / sum_s 2^(m_s - m) z_s over
// its pieces, a lane in 8 taking every eighth piece's m and z, in an order that
// does not depend on who finished first.  It is a chain of loads (cut, then maxima
// and partials), so rows run side by side: 8 MB of partials, from L2, take about 4 us,
// one row at a time took 10.  Merging inside the attention
// kernels, by the CTA that brings an entry's last piece, took 17 to 33 thousand
// cycles.
constexpr uint32_t kMergeWarps = 8, kMergeRows = 4;  // rows of a warp at a time

// Here and now: not moved to where it is used.
__device__ __forceinline__ PromptEntry load_entry(const PromptEntry* p) {
    static_assert(sizeof(PromptEntry) == 48, "three vectors");
    union {
        uint32_t w[12];
        PromptEntry e;
    } u;
#pragma unroll
    for (int i = 0; i < 3; ++i)
        asm volatile("ld.global.v4.u32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(u.w[4 * i]), "=r"(u.w[4 * i + 1]), "=r"(u.w[4 * i + 2]), "=r"(u.w[4 * i + 3])
                     : "l"(reinterpret_cast<const uint4*>(p) + i));
    return u.e;
}

template <int D, bool BF>
__global__ void __launch_bounds__(32 * kMergeWarps) prompt_merge_kernel(const __grid_constant__ PromptArgs a) {
    constexpr int C = D / 32;  // channels of a lane
    struct alignas(4 * C) Lane {
        float f[C];
    };
    const uint32_t lane = threadIdx.x & 31;
    const PromptEntry* cuts = reinterpret_cast<const PromptEntry*>(a.ws + a.l.cuts);
    const float* acc = reinterpret_cast<const float*>(a.ws + a.l.acc);
    const float* ml = reinterpret_cast<const float*>(a.ws + a.l.ml);
    const uint32_t rows = a.l.slot_rows, quads = rows / kMergeRows, sub = lane / 8, piece = lane % 8;
    // The plan is complete before the attention lets this kernel start (prompt_tc.cu; prompt_rows_kernel lets it start at
    // its end), so it is read before the wait.
    // plan_header's check, a word a lane: in registers of every lane it cost a CTA of the three that an SM holds (1023
    // tokens, 24 heads of 64: 25.1 us instead of 22.9).
    const uint32_t word = reinterpret_cast<const uint32_t*>(a.ws)[lane % 8];
    uint32_t i = blockIdx.x * kMergeWarps + (threadIdx.x >> 5);
    PromptEntry next = load_entry(cuts + min(i / quads / a.kv_heads, a.l.max_ctas - 1));
    const uint32_t n_cuts = __shfl_sync(0xffffffffu, word, 2);
    if (__any_sync(0xffffffffu, lane - 3 < 5 && word != a.key[min(lane - 3, 4u)])) {
        pdl_wait_primary();  // what comes next on the stream waits for this kernel alone
        return;
    }
    pdl_wait_primary();
    while (i < n_cuts * a.kv_heads * quads) {
        const PromptEntry e = next;
        const uint32_t row0 = i % quads * kMergeRows, head = i / quads % a.kv_heads;
        i += gridDim.x * kMergeWarps;
        next = load_entry(cuts + min(i / quads / a.kv_heads, a.l.max_ctas - 1));
        auto token_of = [&](uint32_t row) {
            return e.tok0 + row / kPromptTileRows * a.tpt + row % kPromptTileRows / a.group;
        };
        auto exists = [&](uint32_t row) { return row % kPromptTileRows < a.tpt * a.group && token_of(row) < e.nq; };
        const uint64_t first = ((uint64_t)e.slot0 * a.kv_heads + head) * rows + row0, step = (uint64_t)a.kv_heads * rows;
        const float2* mz = reinterpret_cast<const float2*>(ml) + first + sub;  // of the lane's row
        const bool mine = exists(row0 + sub);
        const uint32_t live = __ballot_sync(0xffffffffu, mine);
        float m = -CUDART_INF_F, z = 0.f;
        Lane o[kMergeRows] = {};
        for (uint32_t s = piece; s < e.n_splits; s += 8)
            if (mine) m = fmaxf(m, mz[s * step].x);
#pragma unroll
        for (int k = 4; k; k >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, k));
        const float ref = m == -CUDART_INF_F ? 0.f : m;
        for (uint32_t s0 = 0; s0 < e.n_splits; s0 += 8) {
            float w = 0.f;
            if (mine && s0 + piece < e.n_splits) {
                const float2 p = mz[(s0 + piece) * step];
                if (p.y != 0.f) w = exp2f(p.x - ref);  // 0: the row saw nothing of this piece
                z += p.y * w;
            }
            const uint32_t n = min(8u, e.n_splits - s0);
#pragma unroll 2
            for (uint32_t s = 0; s < n; ++s) {
                Lane x[kMergeRows];
#pragma unroll
                for (uint32_t u = 0; u < kMergeRows; ++u)
                    if (live >> 8 * u & 1u)
                        x[u] = *reinterpret_cast<const Lane*>(acc + (first + (s0 + s) * step + u) * D + C * lane);
#pragma unroll
                for (uint32_t u = 0; u < kMergeRows; ++u) {
                    const float ws = __shfl_sync(0xffffffffu, w, 8 * u + s);
                    if (ws == 0.f) continue;
#pragma unroll
                    for (int c = 0; c < C; ++c) o[u].f[c] += x[u].f[c] * ws;
                }
            }
        }
#pragma unroll
        for (int k = 4; k; k >>= 1) z += __shfl_xor_sync(0xffffffffu, z, k);
#pragma unroll
        for (uint32_t u = 0; u < kMergeRows; ++u) {
            if (!(live >> 8 * u & 1u)) continue;
            const uint32_t token = token_of(row0 + u), g = (row0 + u) % kPromptTileRows % a.group;
            const float zu = __shfl_sync(0xffffffffu, z, 8 * u), inv = zu == 0.f ? CUDART_NAN_F : 1.f / zu;  // no key seen
            const uint64_t at = ((uint64_t)(e.q0 + token) * a.heads + head * a.group + g) * D + C * lane;
            float chk = 0.f;
#pragma unroll
            for (int c = 0; c < C; ++c) {
                o[u].f[c] *= inv;
                chk = fmaf(o[u].f[c], 0.f, chk);
            }
            if constexpr (BF) {
#pragma unroll
                for (int c = 0; c < C; c += 2)
                    reinterpret_cast<uint32_t*>(a.out)[(at + c) / 2] = pack_bf16x2(o[u].f[c], o[u].f[c + 1]);
                if (a.vec && zu != 0.f && zu == zu && __any_sync(0xffffffffu, !(chk == 0.f))) redo_row<D>(a, e, head, token, g);
            } else {
                *reinterpret_cast<Lane*>(reinterpret_cast<float*>(a.out) + at) = o[u];
            }
        }
    }
}

template <int D, bool BF>
cudaError_t launch_rows(const PromptArgs& a, uint32_t ctas, cudaStream_t stream) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(ctas);
    cfg.blockDim = dim3(kRowsThreads);
    cfg.dynamicSmemBytes = RowsCfg<D>::SMEM;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, prompt_rows_kernel<D, BF>, a);
}

template <int D, bool BF>
cudaError_t configure_rows() {
    return cudaFuncSetAttribute(prompt_rows_kernel<D, BF>, cudaFuncAttributeMaxDynamicSharedMemorySize, RowsCfg<D>::SMEM);
}

}  // namespace

PromptArgs prompt_args(const PromptLaunch& L) {
    PromptArgs a{};
    a.q = L.g.q;
    a.k = L.g.k;
    a.v = L.g.v;
    a.out = L.out;
    a.ws = L.ws;
    a.l = L.layout;
    a.q_ts = L.g.q_token_stride;
    a.q_hs = L.g.q_head_stride;
    a.k_ts = L.g.k_token_stride;
    a.k_hs = L.g.k_head_stride;
    a.v_ts = L.g.v_token_stride;
    a.v_hs = L.g.v_head_stride;
    a.heads = L.g.heads;
    a.kv_heads = L.g.kv_heads;
    a.group = L.g.heads / L.g.kv_heads;
    a.tpt = kPromptTileRows / a.group;
    a.kv_tokens = L.g.kv_tokens;
    a.causal = L.g.causal;
    a.scale_log2 = L.scale_log2;
    a.vec = L.vec;
    prompt_plan_key(L.g, L.layout.max_ctas, a.key);
    a.status = L.status;
    return a;
}

cudaError_t configure_prompt_kernels() {
    cudaError_t e;
    if ((e = configure_prompt_tc_kernels()) != cudaSuccess) return e;
    if ((e = configure_rows<64, false>()) != cudaSuccess || (e = configure_rows<64, true>()) != cudaSuccess ||
        (e = configure_rows<128, false>()) != cudaSuccess)
        return e;
    return configure_rows<128, true>();
}

cudaError_t launch_prompt_plan(const PromptLaunch& L, cudaStream_t stream) {
    PlanArgs a{};
    a.q_starts = L.q_starts;
    a.kv_starts = L.kv_starts;
    a.ws = L.ws;
    a.l = L.layout;
    a.sequences = L.g.sequences;
    a.q_tokens = L.g.q_tokens;
    a.kv_tokens = L.g.kv_tokens;
    a.causal = L.g.causal;
    a.tpt = kPromptTileRows / (L.g.heads / L.g.kv_heads);
    a.kv_heads = L.g.kv_heads;
    prompt_plan_key(L.g, L.layout.max_ctas, a.key);
    a.status = L.status;
    // A thread an entry, if that many fit.
    uint32_t threads = 32;
    const uint64_t most = (uint64_t)L.g.q_tokens / (2 * a.tpt) + L.g.sequences;
    while (threads < kPlanThreads && threads < most) threads *= 2;
    return launch_pdl(prompt_plan_kernel, dim3(1), dim3(threads), stream, a);
}

cudaError_t launch_prompt_rows(const PromptLaunch& L, cudaStream_t stream) {
    const PromptArgs a = prompt_args(L);
    const bool bf = L.g.dtype == PP_DTYPE_BF16;
    // As many CTAs as are resident at a time, by registers 2 an SM at head_dim 64 and by shared memory 1 at 128:
    // one that waits for its turn would sit on its first unit until another CTA ends.
    if (L.g.head_dim == 64)
        return bf ? launch_rows<64, true>(a, 2 * L.layout.max_ctas, stream)
                  : launch_rows<64, false>(a, 2 * L.layout.max_ctas, stream);
    return bf ? launch_rows<128, true>(a, L.layout.max_ctas, stream) : launch_rows<128, false>(a, L.layout.max_ctas, stream);
}

// An entry takes no more steps than its keys have tiles.
uint32_t prompt_uncut_keys() { return (kCutSteps - 1) * kPromptKeyTile; }

cudaError_t launch_prompt_merge(const PromptLaunch& L, cudaStream_t stream) {
    const PromptArgs a = prompt_args(L);
    const dim3 grid(4 * L.num_sms), block(32 * kMergeWarps);
    const bool bf = L.g.dtype == PP_DTYPE_BF16;
    if (L.g.head_dim == 64)
        return bf ? launch_pdl(prompt_merge_kernel<64, true>, grid, block, stream, a)
                  : launch_pdl(prompt_merge_kernel<64, false>, grid, block, stream, a);
    return bf ? launch_pdl(prompt_merge_kernel<128, true>, grid, block, stream, a)
              : launch_pdl(prompt_merge_kernel<128, false>, grid, block, stream, a);
}

}  // namespace pp
