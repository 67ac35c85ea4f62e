// Attention of whole prompts on the tensor cores (bf16, rows on the 16-byte
// grid): softmax(q k') v of packed sequences, causal or not, grouped heads.
//
// One CTA per SM takes work items (prompt.cuh) as it becomes free.  An item is
// two tiles of 128 query rows against a range of keys in tiles of 128; each
// tile has a warpgroup of its own for the softmax, so that while one
// exponentiates, the tensor cores multiply for the other:
//   warps 0-3, 4-7  softmax of tile 0, 1: a thread owns a row
//   warp 8          issues the matrix products (tcgen05.mma, one thread)
//   warp 9          hands out items and loads tiles (TMA, one thread)
// Tensor memory, 512 columns: the scores S of both tiles (128 each, f32) and
// their outputs O (head_dim each).  S = Q K' from shared memory; the softmax
// writes P in bf16 over S, and O += P V reads P from tensor memory.  P in bf16
// is the tensor cores' operand type; its row sum is taken before the rounding,
// in f32, as are the maximum and O.
//
// The running maximum is a reference point that moves only when a score passes
// it by 2^8: O is then rescaled in tensor memory, in most key tiles nothing is.
// A thread may touch O whenever its scores are ready, because S of tile j was
// issued after P V of tile j - 1 and the tensor cores work in order.
//
// Where only tile 0 has rows (single tokens, short chunks), both warpgroups take
// them, each half of the key tiles with its own maximum, sum and output; at the
// end the first merges the two, both being in its tensor memory lanes.  Such an
// item is bound by the latency of one tile's chain (S, softmax, P V), and two
// chains side by side halve it.
//
// Keys that a row does not see get score -inf, hence P = 0, but 0 * v is not 0
// where v is NaN or infinite (padding, later tokens of the same tile).  Such a
// row ends up not finite, and its warp computes it again from the keys that it
// does see, unless these explain it (prompt.cuh).
//
// What bounds it: the chain S, softmax, P V of a tile, of which two run side by side.
// P lies over S, so that S of the next key tile waits until P V has read P, and the
// softmax waits for both.  Two tiles take 3320 cycles a key tile at head_dim 128, where
// the tensor cores need 2048 (1024 each) and the exponentials 2048 (2 * 16384, 16 a clock
// and SM): 62 % of either.  At 64 it is 2930, the tensor cores need 1024 and are busy
// 35 % of the time, the exponentials 70 %.
// 8192 tokens, 16 heads on 4: 1165 TFLOP/s full and 1157 causal at head_dim 128 (71 %
// of what cuBLAS reaches), 671 and 681 at 64; of the full one's time 14 % is the last
// round, which not all SMs have an item for.  Small batches wait for the plan, the
// first tiles and the code itself: 17 tokens take 10 us, 1023 of 24 heads 23 us.
// The softmax's 128 scores a thread cost 32 bytes of spills at head_dim 128.
// Slower, at the same sizes: P in two halves, so that P V starts earlier (1090: one more
// wait in the issuing thread at every tile costs more than it hides); that thread
// waiting for the next K only before its product (1105); one copy of the waits' slow
// path (1131); both tiles in step, a thread of its own for each tile's products, and
// part of the exponentials as polynomials.
//
// Halves on/off: 16 single tokens over 8192 keys, 32 heads on 8: 93 us against 115;
// 64 over 1000 keys: 91 against 100.
#include <math_constants.h>

#include "prompt.cuh"
#include "tcgen05.cuh"

namespace pp {

PromptArgs prompt_args(const PromptLaunch& L);

namespace {

constexpr int kThreads = 384;
constexpr long long kWaitCycles = 4000000000ll;  // 2 s at 2 GHz: generous, never hit in normal runs

template <int D>
struct TcCfg {
    static constexpr uint32_t PANEL = 128 * 128;          // 128 rows of 64 bf16
    static constexpr uint32_t TILE = PANEL * (D / 64);    // a Q, K or V tile
    static constexpr uint32_t STAGES = D == 128 ? 5 : 8;  // K and V tiles in flight
    static constexpr uint32_t SMEM = 1024 + 2 * TILE + STAGES * TILE;
    static constexpr uint32_t S_COL = 0, O_COL = 256;     // tile t: + 128 t, + D t
    // Registers of a thread of the softmax and of the others (2 x + y = 3 * 168): the
    // products' thread keeps 32 descriptors at head_dim 128, half of them at 64.
    static constexpr int R_SOFTMAX = D == 128 ? 208 : 216, R_OTHER = D == 128 ? 88 : 72;
};

struct Item {
    PromptEntry e;
    uint32_t head, valid;
};

struct Shared {
    uint64_t kv_full[8], kv_empty[8];
    uint64_t q_full[2], q_empty[2];
    uint64_t s_full[2], p_full[2], o_full[2];
    uint64_t item_full[2], item_empty[2];
    uint64_t drain;
    Item item[2];
    uint32_t tmem;
    int abort;
    int redoing;       // warps that compute rows again: the others wait for them without a limit of their own
    uint64_t half_full, half_empty;  // the second half of a shared tile is there, has been merged
    float2 half[128];                // its maximum and sum
};

struct TcMaps {
    CUtensorMap q, k, v;
};

// What the roles derive from an item's tile (0 or 1).
struct Geo {
    uint32_t tok;    // its first token
    uint32_t live;   // rows of it that exist
    uint32_t first;  // its first key
    uint32_t n;      // key tiles it sees from there on
    bool halves;     // tile 1 stands for tile 0's rows and the second half of their key tiles
};

__device__ __forceinline__ Geo geometry_of(const PromptArgs& a, const PromptEntry& e, uint32_t t) {
    Geo g;
    const bool single = e.tok0 + a.tpt >= e.nq;
    g.tok = e.tok0 + (single ? 0u : t * a.tpt);
    const uint32_t tokens = g.tok < e.nq ? min(a.tpt, e.nq - g.tok) : 0u;
    g.live = tokens * a.group;
    g.first = e.kv_begin;
    g.n = 0;
    if (tokens) {
        const uint32_t lim = min(e.kv_end, prompt_visible(e, g.tok + tokens - 1, a.causal));
        if (lim > e.kv_begin) g.n = (lim - e.kv_begin + kPromptKeyTile - 1) / kPromptKeyTile;
    }
    g.halves = single && g.n > 1;
    if (g.halves) {
        const uint32_t low = (g.n + 1) / 2;
        if (t) g.first += low * kPromptKeyTile;
        g.n = t ? g.n - low : low;
    } else if (single && t) {
        g.live = g.n = 0;
    }
    return g;
}

__device__ __forceinline__ void st_global_v8(float* p, const uint32_t* v) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]),
                 "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
                 : "memory");
}

template <int D>
__global__ void __launch_bounds__(kThreads, 1)
    prompt_tc_kernel(const __grid_constant__ PromptArgs a, const __grid_constant__ TcMaps maps) {
    using C = TcCfg<D>;
    extern __shared__ unsigned char raw[];
    __shared__ Shared sh;
    unsigned char* smem = raw + ((1024u - (smem_addr(raw) & 1023u)) & 1023u);
    unsigned char* s_q = smem;
    unsigned char* s_kv = smem + 2 * C::TILE;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    volatile int* abort = &sh.abort;

    if (threadIdx.x == 0) {
        for (uint32_t i = 0; i < C::STAGES; ++i) {
            mbar_init(&sh.kv_full[i], 1);
            mbar_init(&sh.kv_empty[i], 1);
        }
        for (int t = 0; t < 2; ++t) {
            mbar_init(&sh.q_full[t], 1);
            mbar_init(&sh.q_empty[t], 1);
            mbar_init(&sh.s_full[t], 1);
            mbar_init(&sh.p_full[t], 4);
            mbar_init(&sh.o_full[t], 1);
            mbar_init(&sh.item_full[t], 1);
            mbar_init(&sh.item_empty[t], 9);
        }
        mbar_init(&sh.drain, 1);
        mbar_init(&sh.half_full, 4);
        mbar_init(&sh.half_empty, 4);
        fence_mbar_init();
        sh.abort = 0;
        sh.redoing = 0;
        tma_prefetch_desc(&maps.q);
        tma_prefetch_desc(&maps.k);
        tma_prefetch_desc(&maps.v);
    }
    if (warp == 8) tmem_alloc(&sh.tmem, 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sh.tmem;
    pdl_wait_primary();
    pdl_launch_dependents();  // after the wait: what a dependent reads early, kernels before this one have finished writing

    auto give_up = [&] {
        *abort = 1;
        if (a.status) atomicOr(a.status, PP_DEV_WAIT_TIMEOUT);
    };
    // One thread's wait.
    auto wait1 = [&](uint64_t* bar, uint32_t parity) -> bool {
        for (;;) {
            if (mbar_wait_cycles(bar, parity, abort, kWaitCycles)) return true;
            if (*abort == 0 && *reinterpret_cast<volatile int*>(&sh.redoing) > 0) continue;
            give_up();
            return false;
        }
    };
    // A whole warp's: every lane learns the same answer.
    auto wait = [&](uint64_t* bar, uint32_t parity) -> bool {
        for (;;) {
            if (__all_sync(0xffffffffu, mbar_wait_cycles(bar, parity, abort, kWaitCycles))) return true;
            const int busy = *reinterpret_cast<volatile int*>(&sh.redoing);
            if (__any_sync(0xffffffffu, *abort == 0 && busy > 0)) continue;
            if (lane == 0) give_up();
            return false;
        }
    };

    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::R_OTHER));
        if (warp == 9 && lane == 0) {
            // ------------------------------------------------ items and loads
            PromptHeader* hdr = reinterpret_cast<PromptHeader*>(a.ws);
            const PromptEntry* entries = reinterpret_cast<const PromptEntry*>(a.ws + a.l.entries);
            const uint32_t n_items = plan_header(a, blockIdx.x == 0).n_items;
            const uint32_t q_bytes = a.group * a.tpt * 128 * (D / 64);
            uint32_t stage = 0, phase = 0, kv = 0, q_use0 = 0, q_use1 = 0, idx = blockIdx.x;
            bool ok = true;
            auto load_q = [&](uint32_t t, uint32_t use, const PromptEntry& e, uint32_t tok, uint32_t head) {
                if (!ok || !(ok = wait1(&sh.q_empty[t], (use & 1) ^ 1))) return;
                mbar_arrive_expect_tx(&sh.q_full[t], q_bytes);
#pragma unroll
                for (int p = 0; p < D / 64; ++p)
                    tma_load_4d(s_q + t * C::TILE + p * C::PANEL, &maps.q, &sh.q_full[t], p * 64, 0,
                                (int32_t)(e.q0 + tok), (int32_t)head);
            };
            auto load_kv = [&](const CUtensorMap* map, uint32_t row, uint32_t head) {
                if (!ok || !(ok = wait1(&sh.kv_empty[stage], phase ^ 1))) return;
                mbar_arrive_expect_tx(&sh.kv_full[stage], C::TILE);
#pragma unroll
                for (int p = 0; p < D / 64; ++p)
                    tma_load_3d(s_kv + stage * C::TILE + p * C::PANEL, map, &sh.kv_full[stage], p * 64, (int32_t)row,
                                (int32_t)head);
                ++kv;
                if (++stage == C::STAGES) {
                    stage = 0;
                    phase ^= 1;
                }
            };
            for (uint32_t it = 0; ok; ++it) {
                const uint32_t slot = it & 1;
                if (!(ok = wait1(&sh.item_empty[slot], ((it >> 1) & 1) ^ 1))) break;
                Item& item = sh.item[slot];
                const bool valid = idx < n_items;
                item.valid = valid;
                if (!valid) {
                    mbar_arrive(&sh.item_full[slot]);
                    break;
                }
                const uint32_t at = idx / a.kv_heads, head = idx - at * a.kv_heads;
                const PromptEntry e = entries[at];
                item.e = e;
                item.head = head;
                mbar_arrive(&sh.item_full[slot]);
                const uint32_t next = atomicAdd(&hdr->next, 1u);
                if (next == n_items - 1) hdr->next = 0;  // every CTA has taken its last: ready for the next call
                const Geo g0 = geometry_of(a, e, 0), g1 = geometry_of(a, e, 1);
                const uint32_t n_max = max(g0.n, g1.n);
                uint32_t row = e.k0 + g0.first;
                if (g0.halves) {  // in the order of the products below
                    const uint32_t row1 = e.k0 + g1.first;
                    load_q(0, q_use0++, e, g0.tok, head);
                    load_kv(&maps.k, row, head);
                    load_q(1, q_use1++, e, g0.tok, head);
                    load_kv(&maps.k, row1, head);
                    for (uint32_t j = 0; j < g0.n; ++j) {
                        load_kv(&maps.v, row + j * kPromptKeyTile, head);
                        if (j + 1 < g0.n) load_kv(&maps.k, row + (j + 1) * kPromptKeyTile, head);
                        if (j < g1.n) load_kv(&maps.v, row1 + j * kPromptKeyTile, head);
                        if (j + 1 < g1.n) load_kv(&maps.k, row1 + (j + 1) * kPromptKeyTile, head);
                    }
                    idx = next + gridDim.x;
                    continue;
                }
                if (g0.n) load_q(0, q_use0++, e, g0.tok, head);
                if (n_max) load_kv(&maps.k, row, head);
                if (g1.n) load_q(1, q_use1++, e, g1.tok, head);
                if (n_max) load_kv(&maps.v, row, head);
                for (uint32_t j = 1; j < n_max; ++j) {
                    row += kPromptKeyTile;
                    load_kv(&maps.k, row, head);
                    load_kv(&maps.v, row, head);
                }
                idx = next + gridDim.x;
            }
            // Before the CTA leaves, the loads in flight have landed (a bounded wait each, whatever went
            // wrong), and so have the tensor cores' arrivals on the ring.
            int never = 0;
            if (*abort) {
                for (uint32_t i = kv > C::STAGES ? kv - C::STAGES : 0; i < kv; ++i)
                    mbar_wait_cycles(&sh.kv_full[i % C::STAGES], (i / C::STAGES) & 1, &never, kWaitCycles);
                if (q_use0) mbar_wait_cycles(&sh.q_full[0], (q_use0 - 1) & 1, &never, kWaitCycles);
                if (q_use1) mbar_wait_cycles(&sh.q_full[1], (q_use1 - 1) & 1, &never, kWaitCycles);
            } else {
                for (uint32_t i = kv > C::STAGES ? kv - C::STAGES : 0; ok && i < kv; ++i)
                    ok = wait1(&sh.kv_empty[i % C::STAGES], (i / C::STAGES) & 1);
                if (q_use0 && ok) ok = wait1(&sh.q_empty[0], (q_use0 - 1) & 1);
                if (q_use1 && ok) ok = wait1(&sh.q_empty[1], (q_use1 - 1) & 1);
            }
        } else if (warp == 8 && lane == 0) {
            // --------------------------------------------- the matrix products
            constexpr uint32_t QK = tc_bf16_desc(128, 128, false), PV = tc_bf16_desc(128, D, true);
            const uint64_t dq = tc_desc_sw128(smem_addr(s_q), 16, 1024);
            const uint64_t dk = tc_desc_sw128(smem_addr(s_kv), 16, 1024);
            const uint64_t dv = tc_desc_sw128(smem_addr(s_kv), C::PANEL, 1024);
            uint32_t stage = 0, phase = 0, q_use0 = 0, q_use1 = 0, p_use0 = 0, p_use1 = 0;
            bool ok = true;
            auto advance = [&] {
                if (++stage == C::STAGES) {
                    stage = 0;
                    phase ^= 1;
                }
            };
            auto qk = [&](uint32_t t, uint32_t st) {  // S_t = Q_t K'
                const uint64_t da = dq + (t * C::TILE >> 4), db = dk + (st * C::TILE >> 4);
#pragma unroll
                for (int c = 0; c < D / 16; ++c)
                    tc_mma_ss(tmem + C::S_COL + 128 * t, da + (((c / 4) * C::PANEL + (c % 4) * 32) >> 4),
                              db + (((c / 4) * C::PANEL + (c % 4) * 32) >> 4), QK, c > 0);
                tc_commit(&sh.s_full[t]);
            };
            auto pv = [&](uint32_t t, uint32_t st, bool first) {  // O_t += P_t V
                const uint64_t db = dv + (st * C::TILE >> 4);
#pragma unroll
                for (int c = 0; c < 8; ++c)
                    tc_mma_ts(tmem + C::O_COL + D * t, tmem + C::S_COL + 128 * t + 8 * c, db + (c * 2048 >> 4), PV,
                              !first || c > 0);
            };
            for (uint32_t it = 0; ok; ++it) {
                const uint32_t slot = it & 1;
                if (!(ok = wait1(&sh.item_full[slot], (it >> 1) & 1))) break;
                const bool valid = sh.item[slot].valid != 0;
                const PromptEntry& e = sh.item[slot].e;
                uint32_t n0 = 0, n1 = 0;
                bool halves = false;
                if (valid) {
                    const Geo g0 = geometry_of(a, e, 0);
                    n0 = g0.n;
                    halves = g0.halves;
                    n1 = geometry_of(a, e, 1).n;
                }
                const uint32_t n_max = max(n0, n1);
                mbar_arrive(&sh.item_empty[slot]);
                if (!valid) break;
                if (!n_max) continue;
                if (halves) {  // the two chains share nothing but Q's rows; n1 is n0 or n0 - 1
                    auto next_full = [&] { return wait1(&sh.kv_full[stage], phase); };
                    auto release = [&] {
                        tc_commit(&sh.kv_empty[stage]);
                        advance();
                    };
                    if (!(ok = wait1(&sh.q_full[0], q_use0++ & 1) && next_full())) break;
                    tc_fence_after();
                    qk(0, stage);
                    if (n0 == 1) tc_commit(&sh.q_empty[0]);
                    release();
                    if (!(ok = wait1(&sh.q_full[1], q_use1++ & 1) && next_full())) break;
                    tc_fence_after();
                    qk(1, stage);
                    if (n1 == 1) tc_commit(&sh.q_empty[1]);
                    release();
                    for (uint32_t j = 0; ok && j < n0; ++j) {
                        if (!(ok = next_full() && wait1(&sh.p_full[0], p_use0++ & 1))) break;
                        tc_fence_after();
                        pv(0, stage, j == 0);
                        release();
                        if (j + 1 < n0) {
                            if (!(ok = next_full())) break;
                            qk(0, stage);
                            if (j + 2 == n0) tc_commit(&sh.q_empty[0]);
                            release();
                        } else {
                            tc_commit(&sh.o_full[0]);
                        }
                        if (j < n1) {
                            if (!(ok = next_full() && wait1(&sh.p_full[1], p_use1++ & 1))) break;
                            tc_fence_after();
                            pv(1, stage, j == 0);
                            release();
                            if (j + 1 < n1) {
                                if (!(ok = next_full())) break;
                                qk(1, stage);
                                if (j + 2 == n1) tc_commit(&sh.q_empty[1]);
                                release();
                            } else {
                                tc_commit(&sh.o_full[1]);
                            }
                        }
                    }
                    continue;
                }
                // S of the first key tile; after a tile's last S of the item its Q is free
                if (!(ok = wait1(&sh.kv_full[stage], phase))) break;
                if (n0) {
                    if (!(ok = wait1(&sh.q_full[0], q_use0++ & 1))) break;
                    tc_fence_after();
                    qk(0, stage);
                    if (n0 == 1) tc_commit(&sh.q_empty[0]);
                }
                if (n1) {
                    if (!(ok = wait1(&sh.q_full[1], q_use1++ & 1))) break;
                    tc_fence_after();
                    qk(1, stage);
                    if (n1 == 1) tc_commit(&sh.q_empty[1]);
                }
                tc_commit(&sh.kv_empty[stage]);
                advance();
                for (uint32_t j = 0; j < n_max; ++j) {
                    const uint32_t sv = stage, pv_phase = phase;
                    advance();
                    const uint32_t sk = stage, pk_phase = phase;
                    const bool more = j + 1 < n_max;
                    if (!(ok = wait1(&sh.kv_full[sv], pv_phase))) break;
                    if (more && !(ok = wait1(&sh.kv_full[sk], pk_phase))) break;
                    if (j < n0) {
                        if (!(ok = wait1(&sh.p_full[0], p_use0++ & 1))) break;
                        tc_fence_after();
                        pv(0, sv, j == 0);
                        if (j + 1 < n0) {
                            qk(0, sk);
                            if (j + 2 == n0) tc_commit(&sh.q_empty[0]);
                        } else {
                            tc_commit(&sh.o_full[0]);
                        }
                    }
                    if (j < n1) {
                        if (!(ok = wait1(&sh.p_full[1], p_use1++ & 1))) break;
                        tc_fence_after();
                        pv(1, sv, j == 0);
                        if (j + 1 < n1) {
                            qk(1, sk);
                            if (j + 2 == n1) tc_commit(&sh.q_empty[1]);
                        } else {
                            tc_commit(&sh.o_full[1]);
                        }
                    }
                    tc_commit(&sh.kv_empty[sv]);
                    if (more) {
                        tc_commit(&sh.kv_empty[sk]);
                        advance();
                    }
                }
            }
            // no product is running when tensor memory is freed
            tc_commit(&sh.drain);
            int never = 0;
            mbar_wait_cycles(&sh.drain, 0, &never, kWaitCycles);
        }
        __syncwarp();
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::R_SOFTMAX));
        // ------------------------------------------------------- the softmax
        const uint32_t t = warp >> 2, r = threadIdx.x & 127, wl = (warp & 3) * 32;
        const uint32_t s_addr = tmem + (wl << 16) + C::S_COL + 128 * t, o_addr = tmem + (wl << 16) + C::O_COL + D * t;
        const uint64_t scale2 = f2_pack(a.scale_log2, a.scale_log2);
        float* acc_ws = reinterpret_cast<float*>(a.ws + a.l.acc);
        float* ml_ws = reinterpret_cast<float*>(a.ws + a.l.ml);
        uint32_t s_use = 0, o_use = 0, half_use = 0;
        for (uint32_t it = 0;; ++it) {
            const uint32_t slot = it & 1;
            if (!wait(&sh.item_full[slot], (it >> 1) & 1)) break;
            // The item stays in shared memory until this warp is done with it: its fields are read again after the
            // key tiles, whose loop needs the registers.
            const PromptEntry& e = sh.item[slot].e;
            if (!sh.item[slot].valid) break;
            uint32_t n, first, lim;
            {
                const Geo g = geometry_of(a, e, t);
                n = g.n;
                first = g.first;
                // a row that does not exist masks nothing: masks cost time, and nobody looks at it
                lim = r < g.live ? min(e.kv_end, prompt_visible(e, g.tok + r / a.group, a.causal)) : 0xffffffffu;
                if (!g.live) {
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sh.item_empty[slot]);
                    continue;
                }
            }
            float m = -CUDART_INF_F, z = 0.f;
            bool ok = true;
            for (uint32_t j = 0; j < n; ++j) {
                if (!(ok = wait(&sh.s_full[t], s_use++ & 1))) break;
                tc_fence_after();
                uint32_t s[128];
#pragma unroll
                for (int c = 0; c < 4; ++c) tmem_ld32(reinterpret_cast<uint32_t(&)[32]>(s[32 * c]), s_addr + 32 * c);
                tmem_wait_ld();
                const uint32_t n0 = first + j * kPromptKeyTile;
                const uint32_t see = lim > n0 ? lim - n0 : 0u;  // of this tile
                if (__any_sync(0xffffffffu, see < kPromptKeyTile)) {
#pragma unroll
                    for (int c = 0; c < 128; ++c)
                        if (c >= see) s[c] = 0xff800000u;
                }
                float x0 = __uint_as_float(s[0]), x1 = __uint_as_float(s[1]);
#pragma unroll
                for (int c = 2; c < 128; c += 2) {
                    x0 = fmaxf(x0, __uint_as_float(s[c]));
                    x1 = fmaxf(x1, __uint_as_float(s[c + 1]));
                }
                const float top = fmaxf(x0, x1) * a.scale_log2;
                const bool moves = top > m + 8.f || (m == -CUDART_INF_F && top > m);
                if (__any_sync(0xffffffffu, moves)) {
                    const float mn = moves ? top : m;
                    const float f = moves ? exp2f(m - mn) : 1.f;
                    z *= f;
                    m = mn;
                    if (j) {
                        const uint64_t f2 = f2_pack(f, f);
#pragma unroll
                        for (int c = 0; c < D; c += 32) {
                            uint32_t o[32];
                            tmem_ld32(o, o_addr + c);
                            tmem_wait_ld();
#pragma unroll
                            for (int i = 0; i < 32; i += 2) {
                                float lo, hi;
                                f2_unpack(f2_mul(f2_pack(__uint_as_float(o[i]), __uint_as_float(o[i + 1])), f2), lo, hi);
                                o[i] = __float_as_uint(lo);
                                o[i + 1] = __float_as_uint(hi);
                            }
                            tmem_st32(o_addr + c, o);
                        }
                    }
                }
                const float ref = m == -CUDART_INF_F ? 0.f : m;  // nothing seen yet: exp2(-inf) = 0
                const uint64_t neg = f2_pack(-ref, -ref);
                uint64_t sum0 = 0ull, sum1 = 0ull;
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    uint32_t p[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        float lo, hi;
                        f2_unpack(f2_fma(f2_pack(__uint_as_float(s[32 * c + 2 * i]), __uint_as_float(s[32 * c + 2 * i + 1])),
                                       scale2, neg), lo, hi);
                        lo = fast_exp2(lo);
                        hi = fast_exp2(hi);
                        if (i & 1) sum1 = f2_add(sum1, f2_pack(lo, hi));
                        else sum0 = f2_add(sum0, f2_pack(lo, hi));
                        p[i] = pack_bf16x2(lo, hi);
                    }
                    tmem_st16(s_addr + 16 * c, p);
                }
                float lo, hi;
                f2_unpack(f2_add(sum0, sum1), lo, hi);
                z += lo + hi;
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh.p_full[t]);
            }
            if (!ok) break;
            if (n) {
                if (!wait(&sh.o_full[t], o_use++ & 1)) break;
                tc_fence_after();
            }
            const Geo g = geometry_of(a, e, t);
            const uint32_t head = sh.item[slot].head, live_rows = g.live;
            const bool live = r < live_rows;
            auto done_with_item = [&] {
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh.item_empty[slot]);
            };
            float f0 = 1.f, f1 = 0.f;  // of this tile's output and of its other half's
            if (g.halves) {
                if (t) {
                    sh.half[r] = make_float2(m, z);
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sh.half_full);
                    if (!wait(&sh.half_empty, half_use++ & 1)) break;
                    done_with_item();
                    continue;
                }
                if (!wait(&sh.half_full, half_use++ & 1)) break;
                tc_fence_after();
                const float2 other = sh.half[r];
                const float top = fmaxf(m, other.x), ref = top == -CUDART_INF_F ? 0.f : top;
                f0 = z == 0.f ? 0.f : exp2f(m - ref);
                f1 = other.y == 0.f ? 0.f : exp2f(other.x - ref);
                z = z * f0 + other.y * f1;
                m = top;
            }
            auto load_o = [&](uint32_t c, uint32_t (&o)[32]) {  // 32 channels of the row's output
                if (!n) {
#pragma unroll
                    for (int i = 0; i < 32; ++i) o[i] = 0u;
                    return;
                }
                tmem_ld32(o, o_addr + c);
                tmem_wait_ld();
                if (g.halves) {
                    uint32_t x[32];
                    tmem_ld32(x, o_addr + D + c);
                    tmem_wait_ld();
#pragma unroll
                    for (int i = 0; i < 32; ++i)
                        o[i] = __float_as_uint(__uint_as_float(o[i]) * f0 + __uint_as_float(x[i]) * f1);
                }
            };
            uint32_t again = 0;  // rows of this warp that are not finite, though they see keys and their sum of P is a number
            const uint32_t warp_row = (warp & 3) * 32;
            auto out_row = [&](uint32_t row) {
                return reinterpret_cast<__nv_bfloat16*>(a.out) +
                       ((uint64_t)(e.q0 + g.tok + row / a.group) * a.heads + head * a.group + row % a.group) * D;
            };
            if (e.n_splits == 1) {
                const float inv = 1.f / z;  // a row that sees no key: 0 * inf = NaN
                float chk = 0.f;
                __nv_bfloat16* out = out_row(r);
#pragma unroll
                for (int c = 0; c < D; c += 32) {
                    uint32_t o[32];
                    load_o(c, o);
#pragma unroll
                    for (int i = 0; i < 32; i += 16) {
                        uint32_t w[8];
#pragma unroll
                        for (int k = 0; k < 8; ++k) {
                            const float x = __uint_as_float(o[i + 2 * k]) * inv, y = __uint_as_float(o[i + 2 * k + 1]) * inv;
                            chk = fmaf(x, 0.f, chk);
                            chk = fmaf(y, 0.f, chk);
                            w[k] = pack_bf16x2(x, y);
                        }
                        if (live) {
                            reinterpret_cast<uint4*>(out + c + i)[0] = make_uint4(w[0], w[1], w[2], w[3]);
                            reinterpret_cast<uint4*>(out + c + i)[1] = make_uint4(w[4], w[5], w[6], w[7]);
                        }
                    }
                }
                again = __ballot_sync(0xffffffffu, live && lim > 0 && z == z && !(chk == 0.f));
            } else {
                // partial of this piece, for prompt_merge_kernel
                auto slot_row = [&](uint32_t s, uint32_t row) {
                    return (uint64_t)((e.slot0 + s) * a.kv_heads + head) * a.l.slot_rows + t * kPromptTileRows + row;
                };
                const uint64_t at = slot_row(e.split, r);
#pragma unroll
                for (int c = 0; c < D; c += 32) {
                    uint32_t o[32];
                    load_o(c, o);
                    if (live) {
#pragma unroll
                        for (int i = 0; i < 32; i += 8) st_global_v8(acc_ws + at * D + c + i, &o[i]);
                    }
                }
                if (live) *reinterpret_cast<float2*>(ml_ws + 2 * at) = make_float2(m, z);
            }
            if (g.halves && lane == 0) {
                tc_fence_before();
                mbar_arrive(&sh.half_empty);  // O and the other half's have been read
            }
            if (again) {
                if (lane == 0) atomicAdd(&sh.redoing, 1);
                __syncwarp();
                for (; again; again &= again - 1) {
                    const uint32_t row = warp_row + __ffs(again) - 1;
                    redo_row<D>(a, e, head, g.tok + row / a.group, row % a.group);
                }
                __syncwarp();
                if (lane == 0) atomicSub(&sh.redoing, 1);
            }
            done_with_item();
            tc_fence_before();  // O has been read before the next item's first product may start (p_full)
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    // After giving up `next` stays where it is, for the list is not handed out to its end: no plan for later calls.  (Here
    // and not in give_up, whose copies stand at every wait: 17 tokens took 9.9 us there and take 9.8, 1023 23.2 and 23.0.)
    if (threadIdx.x == 0 && *abort) reinterpret_cast<PromptHeader*>(a.ws)->key[4] = 0;
    if (warp == 8) tmem_dealloc(tmem, 512);
}

template <int D>
cudaError_t launch_tc(const PromptArgs& a, const TcMaps& maps, uint32_t ctas, cudaStream_t stream) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(ctas);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = TcCfg<D>::SMEM;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, prompt_tc_kernel<D>, a, maps);
}

}  // namespace

cudaError_t configure_prompt_tc_kernels() {
    cudaError_t e = cudaFuncSetAttribute(prompt_tc_kernel<64>, cudaFuncAttributeMaxDynamicSharedMemorySize, TcCfg<64>::SMEM);
    if (e != cudaSuccess) return e;
    return cudaFuncSetAttribute(prompt_tc_kernel<128>, cudaFuncAttributeMaxDynamicSharedMemorySize, TcCfg<128>::SMEM);
}

cudaError_t launch_prompt_tc(const PromptLaunch& L, const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v,
                             cudaStream_t stream) {
    const PromptArgs a = prompt_args(L);
    TcMaps maps;
    maps.q = q;
    maps.k = k;
    maps.v = v;
    if (L.g.head_dim == 64) return launch_tc<64>(a, maps, L.layout.max_ctas, stream);
    return launch_tc<128>(a, maps, L.layout.max_ctas, stream);
}

}  // namespace pp
