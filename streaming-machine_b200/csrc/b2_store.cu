// b2_store.cu -- the key/value store held in 4 bits: the kernels that write rows into it, read them back and run the
// arrival over it, and the C ABI's b2_store_* (include/base2.h has the formulas).
#include <stdarg.h>
#include <stdio.h>
#include <string.h>

#include <algorithm>
#include <exception>
#include <mutex>
#include <new>
#include <string>
#include <type_traits>
#include <vector>

#include "../../include/base2.h"
#include "b2_ptx.cuh"
#include "b2_store.cuh"

namespace b2 {

// ---------------------------------------------------------------------------------------------------------------------
// write: eight lanes hold a head's key or value (64 int64), lane i of them the pairs of dims i, i + 8, i + 16, i + 24, so
// that a load of the eight is 128 bytes in a row and the first two pairs are the lower half's; U rows, all asked for before
// the first is used. The shift is the bit length of the OR of the magnitudes less 3 (the OR has the largest one's bit
// length). U = 1 where streams give few rows (a decode step, bound by the memory's latency: 1.9 us for 64 rows of 12 heads in
// a graph), 2 for prompts, bound by its bandwidth: 25 us for 10,512 rows of 12 heads (5.4 TB/s, call after call). A row a warp,
// two dims a lane, took three times the instructions and was bound by them (40 us).
// ---------------------------------------------------------------------------------------------------------------------
constexpr int SW_WARPS = 8;

B2_DEV void load_pair(const int64_t* p, bool wide, int64_t& a, int64_t& b) {
    if (wide) {
        const longlong2 t = *reinterpret_cast<const longlong2*>(p);
        a = t.x;
        b = t.y;
    } else {
        a = p[0];
        b = p[1];
    }
}

// the warp's head part and its first row among the stream's (U rows a warp)
template <int U>
B2_DEV bool store_item(int H, int n, int& part, int& i) {
    const int item = blockIdx.x * SW_WARPS + (threadIdx.x >> 5), up = item / (2 * H);
    part = item - up * 2 * H;
    i = up * U;
    return i < n;
}

template <int U>
__global__ void __launch_bounds__(SW_WARPS * 32) k_store_write(Store4 st, StoreRows rw, int layer, StoreVec K, StoreVec V,
                                                               int wide, uint32_t* err, uint64_t* stamp) {
    griddep_wait();
    stamp_begin(stamp);
    griddep_launch();
    const int s = blockIdx.y, sub = threadIdx.x & 7;
    StoreRun run;
    if (!store_run(rw, s, st.lim, run, err)) return;
    // the eight lanes' head part and first row: U = 1 the parts of a row in turn, else four neighbours' rows in turn
    const int item = blockIdx.x * (SW_WARPS * 4) + (threadIdx.x >> 3);
    const int part = U == 1 ? item % (2 * st.H) : (item >> 2) % (2 * st.H);
    const int i = U == 1 ? item / (2 * st.H) : ((item >> 2) / (2 * st.H) * 4 + (item & 3)) * U;
    if (!__any_sync(0xffffffffu, i < run.n)) return;             // past a short stream's rows
    const bool key = part < st.H;
    const int h = key ? part : part - st.H;
    const StoreVec X = key ? K : V;
    const int64_t* x = X.x + (size_t)(run.r0 + i) * X.ld + h * X.hs + 2 * sub;
    int64_t v[U][8];
#pragma unroll
    for (int t = 0; t < U; t++)
#pragma unroll
        for (int k = 0; k < 4; k++) {
            v[t][2 * k] = v[t][2 * k + 1] = 0;
            if (i + t < run.n) load_pair(x + (size_t)t * X.ld + 16 * k, wide, v[t][2 * k], v[t][2 * k + 1]);
        }
    const size_t e = kv_index(rw.slot0 + s, layer, h, run.p0 + i, st.L, st.H, st.ctx);
    uint8_t* const codes = key ? st.k + e * 32 + key_byte(sub) : st.v + e * 32 + sub;
    const int step1 = key ? 16 : 8, step2 = key ? 4 : 16;        // from pair i to i + 8, to i + 16
#pragma unroll
    for (int t = 0; t < U; t++) {
        uint32_t past = 0;                                       // nonzero where 32 bits do not hold a value
#pragma unroll
        for (int k = 0; k < 8; k++) past |= (uint32_t)(v[t][k] >> 32) ^ (uint32_t)((int32_t)v[t][k] >> 31);
        int sh[2], c[8];
        if (__all_sync(0xffffffffu, past == 0)) {                // the usual case
            uint32_t m[2] = {0, 0};
#pragma unroll
            for (int k = 0; k < 8; k++) m[k >> 2] |= mag32((int32_t)v[t][k]);
#pragma unroll
            for (int o = 1; o < 8; o <<= 1) {
                m[0] |= __shfl_xor_sync(0xffffffffu, m[0], o);
                m[1] |= __shfl_xor_sync(0xffffffffu, m[1], o);
            }
            const int big = max(29 - __clz((int)(m[0] | m[1])), 0);
#pragma unroll
            for (int k = 0; k < 2; k++) sh[k] = key ? max(max(29 - __clz((int)m[k]), 0), big - 3) : big;
#pragma unroll
            for (int k = 0; k < 8; k++) {
                const int down = max(sh[k >> 2] - 1, 0), one = sh[k >> 2] > 0;
                c[k] = max(min((((int)v[t][k] >> down) + one) >> one, 7), -8);
            }
        } else {
            uint64_t m[2] = {0, 0};
#pragma unroll
            for (int k = 0; k < 8; k++) m[k >> 2] |= mag(store_clamp(v[t][k]));
#pragma unroll
            for (int o = 1; o < 8; o <<= 1) {
                m[0] |= __shfl_xor_sync(0xffffffffu, m[0], o);
                m[1] |= __shfl_xor_sync(0xffffffffu, m[1], o);
            }
            const int big = min(max(bitlen_u(m[0] | m[1]) - 3, 0), STORE_MAX_SHIFT);
#pragma unroll
            for (int k = 0; k < 2; k++) sh[k] = key ? max(min(max(bitlen_u(m[k]) - 3, 0), STORE_MAX_SHIFT), big - 3) : big;
#pragma unroll
            for (int k = 0; k < 8; k++) c[k] = store_code(store_clamp(v[t][k]), sh[k >> 2]);
        }
        if (i + t < run.n) {
#pragma unroll
            for (int k = 0; k < 4; k++)
                codes[t * 32 + (k & 1) * step1 + (k >> 1) * step2] = (uint8_t)((c[2 * k] & 15) | (c[2 * k + 1] << 4));
            if (key) {
                if (sub < 2) st.ks[(e + t) * 2 + sub] = (int8_t)(sub ? sh[1] : sh[0]);
            } else if (sub == 0) {
                st.vs[e + t] = (int8_t)sh[0];
            }
        }
    }
}

// read: the values that the codes stand for, c 2^s; a warp a head's key or value of U consecutive rows, as above
template <int U>
__global__ void __launch_bounds__(SW_WARPS * 32) k_store_read(Store4 st, StoreRows rw, int layer, int64_t* __restrict__ K,
                                                              int64_t* __restrict__ V, int wide, uint32_t* err) {
    griddep_wait();
    griddep_launch();
    const int s = blockIdx.y, lane = threadIdx.x & 31;
    StoreRun run;
    int part, i;
    if (!store_run(rw, s, st.lim, run, err) || !store_item<U>(st.H, run.n, part, i)) return;
    const bool key = part < st.H;
    const int h = key ? part : part - st.H;
    int64_t* out = key ? K : V;
    if (!out) return;
    const size_t e = kv_index(rw.slot0 + s, layer, h, run.p0 + i, st.L, st.H, st.ctx);
    const uint8_t* const codes = key ? st.k + e * 32 + key_byte(lane) : st.v + e * 32 + lane;
    const int8_t* const shifts = key ? st.ks + e * 2 + (lane >> 4) : st.vs + e;
    int c[U], sh[U];
#pragma unroll
    for (int t = 0; t < U; t++) {
        c[t] = sh[t] = 0;
        if (i + t < run.n) {
            c[t] = (int8_t)codes[t * 32];
            sh[t] = shifts[key ? t * 2 : t];
        }
    }
    int64_t* o = out + ((size_t)(run.r0 + i) * st.H + h) * 64 + 2 * lane;
#pragma unroll
    for (int t = 0; t < U; t++, o += st.H * 64) {
        if (i + t >= run.n) return;
        const int lo = (int)((uint32_t)c[t] << 28) >> 28, hi = c[t] >> 4;
        const int64_t a = (int64_t)((uint64_t)(int64_t)lo << sh[t]), b = (int64_t)((uint64_t)(int64_t)hi << sh[t]);
        if (wide) {
            *reinterpret_cast<longlong2*>(o) = make_longlong2(a, b);
        } else {
            o[0] = a;
            o[1] = b;
        }
    }
}

// ---------------------------------------------------------------------------------------------------------------------
// the arrival of few rows a stream (a decode step), NW warps per (row, head): one where there are many (no barrier, four
// units a CTA), else a CTA of 4, 8 or 16, or a cluster of cs CTAs sharing the keys (attend_few has the rule). The integer
// table softmax needs the largest score before any weight (a = ARR[start - score] does not factor), so the keys are read
// once for the scores, which stay in shared memory, and the values once after it:
//   pass 1  32 keys a warp: their codes as the A rows of m16n8k32 (16 c: the digits stay in a byte's upper half, no sign
//           to extend), the query's two bytes as B columns, so the two products of a key meet in one lane; scores into
//           shared memory, the largest score and value shift by warp maxima
//   pass 2  a = ARR[start - score], Z += a, the weight's three bytes into three planes of shared memory
//   pass 3  num: the planes as the A rows, the values' codes as B (4 keys x 8 dims of nibbles turned by byte permutes)
// PUT (store_step): the warp into whose block the row's own position falls holds its key and value first; early: what earlier
// steps wrote is asked for into L2 before the dependency wait (the engine's steps: 0.586 -> 0.572 ms at 64 x 160). RING: the
// codes come by asynchronous copies into a ring in shared memory, three blocks ahead, in place of loads one block ahead (two at
// 16 warps).
// What shared memory a CTA does not take the table's entries use as L1 (71 KB: with 8 bytes a key and the ring 4 x 32,768 took
// 41 us), so the weights' planes lie where the scores were.
// Bound by the chain of dependent steps where there are few units (3.2 us for 17 keys in a graph, 7.1 for 16 x 1,024). Where
// there are many, by the latency of loads and of dependent steps that too few warps hide (512 x 192: 21 us, 2.8 TB/s; 1,536 CTAs
// are 1.48 rounds of the 7 an SM that 69 registers and 22 KB allow, the second half empty: 34% of the warp places taken, no
// warp ready in 43% of the cycles; about 240 instructions a warp and block of 32 keys). On long contexts by that and by the
// barriers between the passes (4 x 32,768: 30 us, 3.4 TB/s, no warp ready in 51%; 256 x 2,000: 92 us, 4.4 TB/s). Copies of the
// next blocks into L2 ahead of their loads, and two blocks of registers ahead below 16 warps, gave nothing or cost occupancy.
// ---------------------------------------------------------------------------------------------------------------------
constexpr int SF_BYTES = 5;      // shared memory a key: 4 its score, later 3 of them its weight's planes; 1 its value's shift
// a warp's ring of blocks of 32 keys (or values) on their way
struct SfBlock {
    uint8_t codes[32][32];
    int8_t ks[32][2], vs[32];
};
constexpr int SF_RING = 4;
B2_DEV void copy16(void* to, const void* from) {      // 16 bytes, asynchronously, past L1
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(saddr(to)), "l"(from) : "memory");
}
B2_DEV void prefetch_l2(const void* p) { asm volatile("prefetch.global.L2 [%0];" ::"l"(p)); }
B2_DEV void copies_end() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
B2_DEV void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

B2_DEV void mma_s8(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
B2_DEV void mma_u8s8(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
B2_DEV void mma_s8_first(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
        : "=r"(c[0]), "=r"(c[1]), "=r"(c[2]), "=r"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "r"(0));
}
// eight 4-bit codes of a word as signed bytes 16 c: the even dims' and the odd dims'
B2_DEV uint32_t even16(uint32_t w) { return (w << 4) & 0xF0F0F0F0u; }
B2_DEV uint32_t odd16(uint32_t w) { return w & 0xF0F0F0F0u; }

B2_DEV uint32_t shr_u32(uint32_t x, uint32_t s) {     // 0 for s > 31
    uint32_t r;
    asm("shr.u32 %0, %1, %2;" : "=r"(r) : "r"(x), "r"(s));
    return r;
}

// the same score from 16 dot (what the tensor cores give of 16 c): r16 = 32 - u - S
B2_DEV int32_t score16(int32_t dot16, int r16) { return r16 >= 4 ? rnd32(dot16, r16) : store_score(dot16 >> 4, r16 - 4); }

// four words (one of each of four keys, eight dims each) -> byte b of all four in r[b] (dims 2b and 2b + 1)
B2_DEV void turn4(const uint32_t* w, uint32_t (&r)[4]) {
    const uint32_t t0 = __byte_perm(w[0], w[1], 0x5140), t1 = __byte_perm(w[2], w[3], 0x5140);
    const uint32_t t2 = __byte_perm(w[0], w[1], 0x7362), t3 = __byte_perm(w[2], w[3], 0x7362);
    r[0] = __byte_perm(t0, t1, 0x5410);
    r[1] = __byte_perm(t0, t1, 0x7632);
    r[2] = __byte_perm(t2, t3, 0x5410);
    r[3] = __byte_perm(t2, t3, 0x7632);
}

// four weights below 2^24 -> their bytes by place, those of the four weights in a word
B2_DEV void turn3(const uint32_t* w, uint32_t& b0, uint32_t& b1, uint32_t& b2) {
    const uint32_t t0 = __byte_perm(w[0], w[1], 0x5140), t1 = __byte_perm(w[2], w[3], 0x5140);
    b0 = __byte_perm(t0, t1, 0x5410);
    b1 = __byte_perm(t0, t1, 0x7632);
    b2 = __byte_perm(__byte_perm(w[0], w[1], 0x0062), __byte_perm(w[2], w[3], 0x0062), 0x5410);
}

// N rows' 64 query values at 15 bits, as two signed bytes q15 = 256 hi + lo, in a lane's pair (dims 2 lane, 2 lane + 1):
// bytes hi, lo of the first, hi, lo of the second. u: the rows' shifts. Every lane of the warp takes part.
template <int N>
B2_DEV void query_bytes(const int64_t (&x)[N][2], uint32_t (&word)[N], int (&u)[N]) {
    uint32_t past = 0;                                                            // nonzero where 32 bits do not hold a value
#pragma unroll
    for (int k = 0; k < N; k++)
#pragma unroll
        for (int t = 0; t < 2; t++) past |= (uint32_t)(x[k][t] >> 32) ^ (uint32_t)((int32_t)x[k][t] >> 31);
    int a[N], b[N];
    if (__all_sync(0xffffffffu, past == 0)) {                                     // the usual case
#pragma unroll
        for (int k = 0; k < N; k++) {
            const int y0 = (int)x[k][0], y1 = (int)x[k][1];
            // the largest magnitude's bit length is that of the magnitudes' OR
            u[k] = max(18 - __clz((int)__reduce_or_sync(0xffffffffu, mag32(y0) | mag32(y1))), 0);
            const int down = max(u[k] - 1, 0), one = u[k] > 0;
            a[k] = ((y0 >> down) + one) >> one;
            b[k] = ((y1 >> down) + one) >> one;
        }
    } else {
#pragma unroll 1
        for (int k = 0; k < N; k++) {
            int64_t y0 = 0, y1 = 0;
#pragma unroll
            for (int t = 0; t < N; t++)                                           // (a register of the array by constants)
                if (t == k) { y0 = store_clamp(x[t][0]); y1 = store_clamp(x[t][1]); }
            const int r = max((int)__reduce_max_sync(0xffffffffu, (uint32_t)bitlen_u(mag(y0) | mag(y1))) - 14, 0);
            const int c = (int)rnd64(y0, r), d = (int)rnd64(y1, r);
#pragma unroll
            for (int t = 0; t < N; t++)
                if (t == k) { u[t] = r; a[t] = c; b[t] = d; }
        }
    }
    // byte 0: a + 128 >> 8, byte 1: a, byte 2: b + 128 >> 8, byte 3: b
#pragma unroll
    for (int k = 0; k < N; k++)
        word[k] = __byte_perm(__byte_perm(a[k] + 128, a[k], 0x41), __byte_perm(b[k] + 128, b[k], 0x41), 0x5410);
}

// a head row held by a warp (lane l: dims 2l, 2l + 1), put into the store at element e (k_store_write's arithmetic)
B2_DEV void put_row(const Store4& st, size_t e, bool key, int64_t x0, int64_t x1, int lane) {
    x0 = store_clamp(x0);
    x1 = store_clamp(x1);
    const uint32_t t = (uint32_t)bitlen_u(mag(x0) | mag(x1));
    const int lo = (int)__reduce_max_sync(0xffffffffu, lane < 16 ? t : 0u);
    const int hi = (int)__reduce_max_sync(0xffffffffu, lane < 16 ? 0u : t);
    const int big = min(max(max(lo, hi) - 3, 0), STORE_MAX_SHIFT);
    const int sh = key ? max(min(max((lane < 16 ? lo : hi) - 3, 0), STORE_MAX_SHIFT), big - 3) : big;
    const uint8_t c = (uint8_t)((store_code(x0, sh) & 15) | (store_code(x1, sh) << 4));
    if (key) {
        st.k[e * 32 + key_byte(lane)] = c;
        if ((lane & 15) == 0) st.ks[e * 2 + (lane >> 4)] = (int8_t)sh;
    } else {
        st.v[e * 32 + lane] = c;
        if (lane == 0) st.vs[e] = (int8_t)sh;
    }
}

// Pythia's turn of such a row (pythia_base2.py:116-124, the arithmetic of k_turn): dims t and t + 8, t < 8, lie four lanes
// apart
B2_DEV void turn_row(int64_t& x0, int64_t& x1, int lane, int pos, const int32_t* COS, const int32_t* SIN, uint32_t* err) {
    const int64_t o0 = __shfl_xor_sync(0xffffffffu, x0, 4), o1 = __shfl_xor_sync(0xffffffffu, x1, 4);
    if (lane >= 8) return;
    if ((mag(x0) | mag(x1)) >= (1ull << 31)) set_err(err, DERR_RANGE);
    const size_t t = (size_t)pos * 8 + 2 * (lane & 3);
    const int64_t c0 = COS[t], s0 = SIN[t], c1 = COS[t + 1], s1 = SIN[t + 1];
    x0 = rshift(lane < 4 ? wsub(wmul(x0, c0), wmul(o0, s0)) : wadd(wmul(x0, c0), wmul(o0, s0)), 30);
    x1 = rshift(lane < 4 ? wsub(wmul(x1, c1), wmul(o1, s1)) : wadd(wmul(x1, c1), wmul(o1, s1)), 30);
}

template <int NW>
B2_DEV void unit_sync() {
    if (NW == 1) __syncwarp();
    else __syncthreads();
}

template <int NW, bool PUT, bool RING>
__global__ void __launch_bounds__(NW == 1 ? 128 : NW * 32, NW == 1 ? 7 : (NW == 4 ? 6 : (NW == 8 ? 3 : 1)))
    k_store_attend_few(StoreAttend a, int chunk, int cs, int wide) {
    extern __shared__ __align__(16) uint8_t sm[];
    constexpr int UN = NW == 1 ? 4 : 1;                              // (row, head) units a CTA
    constexpr int D = SF_RING, PF = NW == 16 ? 2 : 1;                // blocks of 32 keys that a warp has on their way (PF: in registers)
    __shared__ int32_t s_max[NW], s_shift[NW], s_acc[UN][NW][3][64];
    __shared__ int64_t s_z[NW], s_num[65];
    __shared__ int2 s_own;                                           // cs > 1: this CTA's largest score and shift
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, wid = NW == 1 ? 0 : warp, un = NW == 1 ? warp : 0;
    const int g = lane >> 2, j = lane & 3, ut = NW == 1 ? lane : threadIdx.x;      // ut: the thread of the unit
    SfBlock* const ring = reinterpret_cast<SfBlock*>(sm) + warp * D;
    uint8_t* const mem = sm + (RING ? (NW == 1 ? 4 : NW) * D * sizeof(SfBlock) : 0) + (size_t)un * chunk * SF_BYTES;
    int32_t* const SC = reinterpret_cast<int32_t*>(mem);             // [chunk]; then of four keys each the three planes' words
    int8_t* const VS = reinterpret_cast<int8_t*>(mem + (size_t)chunk * 4);   // [chunk]
    auto begin = [&]() {
        griddep_wait();
        stamp_begin(a.stamp);
        griddep_launch();
    };
    const bool early = PUT && a.early;
    if (!early) begin();
    const int H = a.st.H, s = blockIdx.y, rank = cs > 1 ? (int)cluster_rank() : 0;
    const int unit = NW == 1 ? blockIdx.x * UN + un : blockIdx.x / cs, i = unit / H, h = unit - i * H;
    StoreRun run;
    // (early: a read from L2, since only the wait makes sure of L1; a step has no cu)
    const bool some = early ? store_run(a.rw, s, s + 1, __ldcg(a.rw.pos + s), a.st.lim, run, a.err)
                            : store_run(a.rw, s, a.st.lim, run, a.err);
    if (!some || i >= run.n) {                                       // the same for a whole cluster
        if (early) begin();
        return;
    }
    const int row = run.r0 + i, p = run.p0 + i;
    int lo = a.window > 0 ? max(0, p - a.window + 1) : 0;
    if (a.first) lo = max(lo, a.first[s]);
    int64_t* const out = a.out + ((size_t)row * H + h) * 64;
    // PUT: the row's own key and value, by the warp whose block they fall into
    auto put = [&]() {
        const size_t e = kv_index(a.rw.slot0 + s, a.layer, h, p, a.st.L, H, a.st.ctx);
        int64_t k0, k1, v0, v1;
        load_pair(a.k.x + (size_t)row * a.k.ld + h * a.k.hs + 2 * lane, wide & 4, k0, k1);
        load_pair(a.v.x + (size_t)row * a.v.ld + h * a.v.hs + 2 * lane, wide & 8, v0, v1);
        if (a.COS) turn_row(k0, k1, lane, p, a.COS, a.SIN, a.err);
        put_row(a.st, e, true, k0, k1, lane);
        put_row(a.st, e, false, v0, v1, lane);
        __syncwarp();                                                // the warp's own loads come after it
    };
    if (lo > p) {
        if (early) begin();
        if (PUT && rank == 0 && wid == 0) put();
        if (PUT) unit_sync<NW>();                                    // out may be k or v
        for (int t = ut; t < 64 && rank == 0; t += NW * 32) out[t] = 0;
        return;
    }
    // blocks of 32 positions; this CTA's are b0 .. b0 + nb - 1
    const int first_block = lo >> 5, blocks = (p >> 5) - first_block + 1;
    const int per = cs > 1 ? (blocks + cs - 1) / cs : blocks;
    const int b0 = first_block + rank * per, nb = max(0, min(per, blocks - rank * per));
    const size_t base = kv_index(a.rw.slot0 + s, a.layer, h, 0, a.st.L, H, a.st.ctx) + (size_t)b0 * 32;
    const int from = lo - b0 * 32, to = p - b0 * 32;                 // visible: from <= local key <= to
    if (early) {                                                     // what earlier steps wrote: into L2 while the launch before ends
        const uint8_t* const line = lane < 8 ? a.st.k + base * 32 + lane * 128 : a.st.v + base * 32 + (lane - 8) * 128;
        for (int b = wid; b < nb; b += NW) {
            if (lane < 16) prefetch_l2(line + (size_t)b * 1024);
            else if (lane == 16) prefetch_l2(a.st.ks + (base + (size_t)b * 32) * 2);
            else if (lane == 17) prefetch_l2(a.st.vs + base + (size_t)b * 32);
        }
        begin();
    }
    int64_t x[1][2];
    load_pair(a.q.x + (size_t)row * a.q.ld + h * a.q.hs + 2 * lane, wide & 1, x[0][0], x[0][1]);
    // of a block's keys the one whose score this lane finishes, and its place: a block's scores, shifts and planes are kept in
    // the order of the values' operands, key 4m + x at 8x + m
    const int mine = 16 * (j >> 1) + 8 * (j & 1) + g, place = 8 * (mine & 3) + (mine >> 2);

    // a block on its way: the i-th of this warp's, b0 + wid + i NW; the warp's lanes wait for their own copies, then meet
    auto fetch = [&](int i, bool values) {
        const int b = wid + i * NW;
        if (b < nb) {
            SfBlock& r = ring[i % D];
            const size_t e = base + (size_t)b * 32;
            const uint8_t* const from_ = (values ? a.st.v : a.st.k) + e * 32 + lane * 16;
            copy16(&r.codes[0][0] + lane * 16, from_);
            copy16(&r.codes[0][0] + 512 + lane * 16, from_ + 512);
            if (!values) {
                if (lane < 4) copy16(&r.ks[0][0] + lane * 16, a.st.ks + e * 2 + lane * 16);
                else if (lane < 6) copy16(r.vs + (lane - 4) * 16, a.st.vs + e + (lane - 4) * 16);
            }
        }
        copies_end();
    };
    auto arrived = [&](int i, bool values) {                         // block i is here; the one D - 1 behind it sets out
        copies_wait<D - 2>();
        __syncwarp();
        fetch(i + D - 1, values);
    };
    // a block's keys: rows 8t + g, words j of both halves; this lane's key's shifts and its value's
    struct Keys { uint2 w[4]; int ks, vs; };
    auto keys = [&](const uint8_t* codes, const int8_t* ks, const int8_t* vs, Keys& k) {
#pragma unroll
        for (int t = 0; t < 4; t++) k.w[t] = *reinterpret_cast<const uint2*>(codes + (8 * t + g) * 32 + 8 * j);
        k.ks = *reinterpret_cast<const int16_t*>(ks + 2 * mine);
        k.vs = vs[mine];
    };
    auto keys_at = [&](int b, Keys& k) {
        const size_t e = base + (size_t)b * 32;
        keys(a.st.k + e * 32, a.st.ks + e * 2, a.st.vs + e, k);
    };
    // a block's values: word g (dims 8g .. 8g + 7) of keys j, j + 4, ..
    auto values = [&](const uint8_t* codes, uint32_t (&w)[8]) {
#pragma unroll
        for (int t = 0; t < 8; t++) w[t] = *reinterpret_cast<const uint32_t*>(codes + (4 * t + j) * 32 + 4 * g);
    };
    if (PUT && nb > 0 && b0 + nb - 1 == p >> 5 && (nb - 1) % NW == wid) put();
    Keys k[PF];
    if (RING) {
#pragma unroll
        for (int i = 0; i < D - 1; i++) fetch(i, false);
    } else {
#pragma unroll
        for (int f = 0; f < PF; f++)
            if (wid + f * NW < nb) keys_at(wid + f * NW, k[f]);
    }
    if (PUT && a.COS) turn_row(x[0][0], x[0][1], lane, p, a.COS, a.SIN, a.err);
    uint32_t words[1], q0[2], q1[2];                                 // q0, q1: B operands of the two halves
    int us[1];
    query_bytes(x, words, us);
    const int u = us[0];
    {
        const uint32_t pick = (g & 1) ? 0x51u : 0x40u;               // odd columns the low bytes
#pragma unroll
        for (int x = 0; x < 2; x++) {
            uint32_t w[4];
#pragma unroll
            for (int b = 0; b < 4; b++) w[b] = __shfl_sync(0xffffffffu, words[0], 16 * x + 4 * j + b);
            q0[x] = __byte_perm(__byte_perm(w[0], w[1], pick), __byte_perm(w[2], w[3], pick), 0x5410);
            q1[x] = __byte_perm(__byte_perm(w[0], w[1], pick + 0x22), __byte_perm(w[2], w[3], pick + 0x22), 0x5410);
        }
    }
    int32_t start = -STORE_LIM - 1;
    int M = 0;
    auto score_block = [&](int b, const Keys& c) {
        int d[2][2][4];                                              // [16 keys][half]
#pragma unroll
        for (int m = 0; m < 2; m++) {
            const uint2 wa = c.w[2 * m], wb = c.w[2 * m + 1];
            mma_s8_first(d[m][0], even16(wa.x), even16(wb.x), odd16(wa.x), odd16(wb.x), q0[0], q1[0]);
            mma_s8_first(d[m][1], even16(wa.y), even16(wb.y), odd16(wa.y), odd16(wb.y), q0[1], q1[1]);
        }
        int dot[2];
#pragma unroll
        for (int x = 0; x < 2; x++) {
            const int hi = (j & 2) ? ((j & 1) ? d[1][x][2] : d[1][x][0]) : ((j & 1) ? d[0][x][2] : d[0][x][0]);
            const int lw = (j & 2) ? ((j & 1) ? d[1][x][3] : d[1][x][1]) : ((j & 1) ? d[0][x][3] : d[0][x][1]);
            dot[x] = 256 * hi + lw;
        }
        const int s0 = (int8_t)c.ks, s1 = c.ks >> 8, S = max(s0, s1), key = b * 32 + mine;
        const int32_t sc = score16((dot[0] << (s0 - S + 3)) + (dot[1] << (s1 - S + 3)), 32 - u - S);
        SC[b * 32 + place] = sc;
        VS[b * 32 + place] = (int8_t)c.vs;
        if (key >= from && key <= to) {
            start = max(start, sc);
            M = max(M, c.vs);
        }
    };
    uint32_t v[PF][8];
    if (RING) {
        for (int i = 0, b = wid; b < nb; i++, b += NW) {
            arrived(i, false);
            const SfBlock& r = ring[i % D];
            Keys c;
            keys(&r.codes[0][0], &r.ks[0][0], r.vs, c);
            score_block(b, c);
        }
        __syncwarp();                                                // the ring is free
#pragma unroll
        for (int i = 0; i < D - 1; i++) fetch(i, true);              // on their way over the reductions
    } else {
        for (int b = wid; b < nb; b += NW * PF) {
            Keys c[PF];
#pragma unroll
            for (int f = 0; f < PF; f++) c[f] = k[f];
#pragma unroll
            for (int f = 0; f < PF; f++)                             // the next blocks', while these are worked on
                if (b + (PF + f) * NW < nb) keys_at(b + (PF + f) * NW, k[f]);
#pragma unroll
            for (int f = 0; f < PF; f++)
                if (b + f * NW < nb) score_block(b + f * NW, c[f]);
        }
#pragma unroll
        for (int f = 0; f < PF; f++)
            if (wid + f * NW < nb) values(a.st.v + (base + (size_t)(wid + f * NW) * 32) * 32, v[f]);
    }
    start = __reduce_max_sync(0xffffffffu, start);
    M = __reduce_max_sync(0xffffffffu, M);
    if (NW > 1) {
        if (lane == 0) { s_max[wid] = start; s_shift[wid] = M; }
        __syncthreads();
#pragma unroll
        for (int w = 0; w < NW; w++) {
            start = max(start, s_max[w]);
            M = max(M, s_shift[w]);
        }
        if (cs > 1) {
            if (threadIdx.x == 0) s_own = make_int2(start, M);
            cluster_sync();
            for (int c = 0; c < cs; c++) {
                const int64_t o = ld_dsmem(mapa(saddr(&s_own), (uint32_t)c));
                start = max(start, (int32_t)o);
                M = max(M, (int)(o >> 32));
            }
        }
    } else {
        __syncwarp();
    }
    // ---- weights: four keys a thread
    int64_t z = 0;
    for (int t = ut * 4; t < nb * 32; t += NW * 128) {
        const int4 sc = *reinterpret_cast<const int4*>(SC + t);
        const uint32_t v4 = *reinterpret_cast<const uint32_t*>(VS + t);
        const int scs[4] = {sc.x, sc.y, sc.z, sc.w}, key0 = (t & ~31) + 4 * (t & 7) + ((t >> 3) & 3);
        uint32_t w[4];
        int32_t four = 0;                                            // four entries of at most 2^24
#pragma unroll
        for (int x = 0; x < 4; x++) {
            const int d = start - scs[x];
            const int key = key0 + 4 * x;
            const bool seen = key >= from && key <= to && d < a.alen;
            const int av = seen ? __ldg(a.ARR + d) : 0;
            four += av;
            w[x] = (shr_u32(av, M - (int)(int8_t)(v4 >> (8 * x))) + 1) >> 1;
        }
        z += four;
        uint32_t r[3];
        turn3(w, r[0], r[1], r[2]);
        *reinterpret_cast<uint4*>(SC + t) = make_uint4(r[0], r[1], r[2], 0);
    }
    z = warp_sum64(z);
    if (NW > 1 && lane == 0) s_z[wid] = z;
    unit_sync<NW>();
    // ---- values
    int acc[8][4] = {};
    auto add_block = [&](int b, const uint32_t (&w)[8]) {
        uint32_t p0 = 0, p1 = 0, r0[4], r1[4];
        if (g < 3) {
            p0 = (uint32_t)SC[b * 32 + 8 * j + g];
            p1 = (uint32_t)SC[b * 32 + 8 * j + 4 + g];
        }
        turn4(w, r0);
        turn4(w + 4, r1);
#pragma unroll
        for (int t = 0; t < 4; t++) {
            mma_u8s8(acc[2 * t], p0, 0, p1, 0, even16(r0[t]), even16(r1[t]));
            mma_u8s8(acc[2 * t + 1], p0, 0, p1, 0, odd16(r0[t]), odd16(r1[t]));
        }
    };
    if (RING) {
        for (int i = 0, b = wid; b < nb; i++, b += NW) {
            arrived(i, true);
            uint32_t w[8];
            values(&ring[i % D].codes[0][0], w);
            add_block(b, w);
        }
    } else {
        for (int b = wid; b < nb; b += NW * PF) {
            uint32_t w[PF][8];
#pragma unroll
            for (int f = 0; f < PF; f++)
#pragma unroll
                for (int t = 0; t < 8; t++) w[f][t] = v[f][t];
#pragma unroll
            for (int f = 0; f < PF; f++)
                if (b + (PF + f) * NW < nb) values(a.st.v + (base + (size_t)(b + (PF + f) * NW) * 32) * 32, v[f]);
#pragma unroll
            for (int f = 0; f < PF; f++)
                if (b + f * NW < nb) add_block(b + f * NW, w[f]);
        }
    }
    // row g of the tiles is plane g; columns 2j, 2j + 1 of tile t are dims 16j + t and 16j + 8 + t
    if (g < 3) {
#pragma unroll
        for (int t = 0; t < 8; t++) {
            s_acc[un][wid][g][16 * j + t] = acc[t][0];
            s_acc[un][wid][g][16 * j + 8 + t] = acc[t][1];
        }
    }
    unit_sync<NW>();
    // a thread finishes dim ut (a lone warp's lanes dim ut + 32 as well)
    constexpr int DIMS = NW == 1 ? 2 : 1;
    int64_t num[DIMS];
#pragma unroll
    for (int x = 0; x < DIMS; x++) {
        num[x] = 0;
        if (ut + 32 * x < 64) {
#pragma unroll
            for (int b = 0; b < 3; b++) {
                int t = 0;
#pragma unroll
                for (int w = 0; w < NW; w++) t += s_acc[un][w][b][ut + 32 * x];
                num[x] += (int64_t)t * (1 << 8 * b);
            }
        }
    }
    if (NW > 1) {
        z = 0;
#pragma unroll
        for (int w = 0; w < NW; w++) z += s_z[w];
        if (cs > 1) {
            if (threadIdx.x < 64) {
                s_num[threadIdx.x] = num[0];
                if (threadIdx.x == 0) s_num[64] = z;
            }
            cluster_sync();
            if (rank == 0 && threadIdx.x < 64) {
                num[0] = z = 0;
                for (int c = 0; c < cs; c++) {
                    num[0] += ld_dsmem(mapa(saddr(&s_num[threadIdx.x]), (uint32_t)c));
                    z += ld_dsmem(mapa(saddr(&s_num[64]), (uint32_t)c));
                }
            }
        }
    }
    if (rank == 0 && ut < 64) {
        const int64_t F = 65536ll * (M + STORE_W_SHIFT) - log2fix(z, a.LOG2);
        const uint32_t e = (uint32_t)__ldg(a.EXP2 + (F & 0xFFFF));
        const int down = 19 - (int)(F >> 16);                        // power's shift less one, and 4 digits more: 16 c
        uint64_t any = 0;
#pragma unroll
        for (int x = 0; x < DIMS; x++) {
            const int64_t n = num[x] * (int64_t)e;                   // at most 2^46 2^17
            const int64_t y = down >= 0 ? ((n >> down) + 1) >> 1 : (int64_t)((uint64_t)n << (-1 - down));
            out[ut + 32 * x] = y;
            any |= mag(y);
        }
        if (PUT && a.or_out) {
            any = warp_or64(any);
            if (lane == 0) atomicOr((unsigned long long*)&a.or_out[row], (unsigned long long)any);
        }
    }
    if (NW > 1 && cs > 1) cluster_sync();                            // rank 0 has read the others' sums
}

// ---------------------------------------------------------------------------------------------------------------------
// the arrival of many rows a stream (a prompt pass): a CTA of 8 warps takes 64 consecutive rows of one head, a pair of warps
// 16 of them; where that gives too few CTAs, a cluster of cs shares the rows' keys. Tiles of 64 keys (and values) are copied
// into shared memory two ahead (cp.async), then unpacked once for all the rows as signed bytes in the order of the tensor
// cores' B operands (c 2^(s - S + 3) for keys, 16 c for values); a warp forms the scores of one of a tile's two blocks of 32.
//   pass 1  every score (m16n8k32, the query's two bytes one after the other), the rows' largest and largest value shift
//   pass 2  the scores again (cheaper than keeping 4 bytes a pair), a = ARR[start - score] from a copy of the table in
//           shared memory (a gather from L1 takes a line a lane), the weight's three bytes as A operands (a lane's scores
//           of a tile lie where its A operand wants them when k is taken in the order below). The two warps of a pair
//           swap those through shared memory and each adds w c for half of the 64 dims: 48 registers of sums a lane in
//           place of 96, which lets 16 warps share an SM
// CTAs are persistent so that the table is copied twice an SM, the longest rows first.
// 194 us for 32 prompts of 300 to 512 rows, 183 us for 2 x 256 rows on 8,000 positions. Bound by latency that 16 warps an SM do
// not hide: 1.8 instructions a clock, no warp ready in 55% of the cycles (fixed waits first, then instruction fetches on the
// prompts, shared and global loads, barriers). The 16 warps are what 128 registers a thread allow, 48 of them sums (112 bytes
// are spilled at that). A tile of 64 x 64 pairs takes an SM about 1.4 us, the start and end of each of the 18 items that an SM
// takes of the prompts about 5. Fewer instructions (the table's place in two
// steps less, the weights by a product in place of shifts) gained nothing. The tensor cores are busy 16% of the time on the
// prompts, 23% on the long context; with sums in tensor memory more warps would fit, which was not tried. Slower: 128 rows on 16
// warps a CTA (one CTA an SM: nothing runs while it waits), the sums of all 64 dims in one warp (8 warps an SM), two items a
// CTA side by side that share a table (192 us and 5% more on long contexts), an item's queries and first tiles copied ahead.
// ---------------------------------------------------------------------------------------------------------------------
constexpr int SM_WARPS = 8, SM_THREADS = SM_WARPS * 32, SM_ROWS = 64, SM_KEYS = 64;
constexpr int SM_STREAMS = 1024;         // up to so many streams the items are listed
struct SmRaw {
    uint8_t k[SM_KEYS][32], v[SM_KEYS][32];
    int8_t ks[SM_KEYS][2], vs[SM_KEYS];
};
struct SmTile {
    uint4 k[SM_KEYS / 8][32];            // [8 keys][lane (g, j)]: key g, dims of word j of both halves, even and odd
    uint4 v[SM_KEYS / 32][4][32];        // [32 keys][tiles 2b, 2b + 1][lane (g, j)]: dims 8g + 2b, 8g + 2b + 1 of 8 keys
    int32_t kr[SM_KEYS];                 // 27 - S: a score's shift less one is kr - u
    int32_t vs[SM_KEYS];
};
struct SmShared {
    SmTile tile[2];
    SmRaw raw[2];
    union {
        uint32_t q[SM_ROWS][33];         // the rows' query bytes, until every lane has its operands
        uint4 p[SM_WARPS][3][32];        // a block's weights on the way to the pair's other warp
    };
    int64_t z[SM_WARPS][16];             // a warp's rows: their sums of entries,
    int2 ym[SM_WARPS][16];               // largest score (twice) and value shift
    int32_t u[SM_ROWS], most[SM_WARPS], slow;
    uint16_t rows[SM_STREAMS];           // how many items of rows each stream has (of a head)
};

// bytes c 2^up of the word's even and odd codes; up = 0 .. 3: c + 8 moves up, 8 2^up comes off again (less: 128 - 8 2^up)
B2_DEV uint32_t even_up(uint32_t w, int up, uint32_t less) {
    return ((((w & 0x0F0F0F0Fu) ^ 0x08080808u) << up) + less) ^ 0x80808080u;
}
B2_DEV uint32_t odd_up(uint32_t w, int up, uint32_t less) {
    return ((((w & 0xF0F0F0F0u) ^ 0x80808080u) >> (4 - up)) + less) ^ 0x80808080u;
}
// bits from .. to of a word (none where from > to; either may lie outside)
B2_DEV uint32_t seen(int from, int to) {
    if (from > 31 || to < 0 || from > to) return 0u;
    return (0xFFFFFFFFu << max(from, 0)) & (0xFFFFFFFFu >> (31 - min(to, 31)));
}

__global__ void __launch_bounds__(SM_THREADS, 2) k_store_attend_many(StoreAttend a, int tiles, int cs, int wide) {
    extern __shared__ __align__(16) uint8_t sm[];
    SmShared& S = *reinterpret_cast<SmShared*>(sm);
    int32_t* const TAB = reinterpret_cast<int32_t*>(sm + sizeof(SmShared));   // [alen + 1], 0 at the end
    constexpr int ROWS = SM_ROWS, KEYS = SM_KEYS;
    const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5, g = lane >> 2, j = lane & 3;
    const int pair = wid >> 1, blk = wid & 1, rank = cs > 1 ? (int)cluster_rank() : 0;   // blk: the warp's block of a tile
    const int H = a.st.H, alen = a.alen;
    for (int i = tid; i < alen / 4; i += SM_THREADS) copy16(TAB + 4 * i, a.ARR + 4 * i);
    for (int i = alen / 4 * 4 + tid; i <= alen; i += SM_THREADS) TAB[i] = i < alen ? __ldg(a.ARR + i) : 0;
    griddep_wait();                       // (the table never changes: its copy need not wait)
    stamp_begin(a.stamp);
    griddep_launch();
    // The items: the streams' last tiles of 64 rows before those ahead of them (a stream's first is tile 0), then by heads, then
    // by streams; below 2^31 (the launch sees to it). Cluster me of W takes one of every W, there and back (me, 2 W - 1 - me,
    // 2 W + me, ..), so that the loads come out even: 32 prompts of 300 to 512 rows 195 us, 200 one way, 227 where the
    // streams that lack a tile keep their places; 4 of 512 rows 38, 51, 49. Past SM_STREAMS streams they do
    const int n_str = a.rw.n_streams, me = blockIdx.x / cs, W = gridDim.x / cs;
    const bool listed = n_str <= SM_STREAMS;
    int w_tile = tiles - 1, w_of = n_str;                     // the walk: at items of tile w_tile, w_of streams have one,
    uint32_t w_from = 0, round = 0;                           // the first is item w_from
    if (listed) {
        for (int s = tid; s < n_str; s += SM_THREADS) {
            StoreRun run;
            S.rows[s] = (uint16_t)(store_run(a.rw, s, a.st.lim, run, a.err) ? (run.n + ROWS - 1) / ROWS : 0);
        }
        __syncthreads();
    }
    auto streams_with = [&](int tile) {                       // every warp counts for itself
        int c = 0;
        for (int s = lane; s - lane < n_str; s += 32) c += __popc(__ballot_sync(0xffffffffu, s < n_str && S.rows[s] > tile));
        return c;
    };
    if (listed) {
        int most = 0;
        for (int s = lane; s < n_str; s += 32) most = max(most, (int)S.rows[s]);
        w_tile = __reduce_max_sync(0xffffffffu, most) - 1;
        w_of = streams_with(w_tile);
    }
    // the next item: its tile (-1: there is none), head and stream
    auto next = [&](int& tile, int& h, int& s) {
        const uint32_t k = round * W + ((round & 1) ? W - 1 - me : me);
        round++;
        while (w_tile >= 0 && k >= w_from + (uint32_t)(w_of * H)) {
            w_from += w_of * H;
            w_tile--;
            if (listed && w_tile >= 0) w_of = streams_with(w_tile);
        }
        tile = w_tile;
        if (w_tile < 0) return;
        h = (k - w_from) / w_of;
        s = (k - w_from) - h * w_of;
        if (listed && w_of < n_str) {                         // the s-th of those that have this tile
            int left = s;
            for (int at = 0;; at += 32) {
                const uint32_t has = __ballot_sync(0xffffffffu, at + lane < n_str && S.rows[at + lane] > w_tile);
                if (left < __popc(has)) {
                    const bool it = (has >> lane & 1) && __popc(has & ((1u << lane) - 1)) == left;
                    s = at + __ffs(__ballot_sync(0xffffffffu, it)) - 1;
                    break;
                }
                left -= __popc(has);
            }
        }
    };
    // an item's entries of the row table, read one item ahead
    int n_r0 = 0, n_r1 = 0, n_pos = 0, n_first = 0;
    auto ahead = [&](int s, int tile) {
        if (tile >= 0) {
            n_r0 = a.rw.cu ? a.rw.cu[s] : s;
            n_r1 = a.rw.cu ? a.rw.cu[s + 1] : s + 1;
            n_pos = a.rw.pos[s];
            n_first = a.first ? a.first[s] : 0;
        }
    };
    int tile, h, s, n_tile, n_h, n_s;
    next(tile, h, s);
    ahead(s, tile);
    for (; tile >= 0; tile = n_tile, h = n_h, s = n_s) {
        next(n_tile, n_h, n_s);
        StoreRun run;
        const bool some = store_run(a.rw, n_r0, n_r1, n_pos, a.st.lim, run, a.err);
        const int from = max(0, n_first);
        ahead(n_s, n_tile);
        if (!some || tile * ROWS >= run.n) continue;
        const int i0 = tile * ROWS, nr = min(ROWS, run.n - i0);
        const int win = a.window > 0 ? a.window : 0x40000000;
        const int p_first = run.p0 + i0, p_last = p_first + nr - 1;
        const int k_lo = max(from, p_first - win + 1);       // the first row sees the earliest position
        __syncthreads();                                      // the item before is done with shared memory
        if (k_lo > p_last) {                                  // nothing to see for any row
            for (int t = rank == 0 ? tid : nr * 64; t < nr * 64; t += SM_THREADS)
                a.out[((size_t)(run.r0 + i0 + (t >> 6)) * H + h) * 64 + (t & 63)] = 0;
            continue;
        }
        const int k0 = k_lo & ~31, k1 = (p_last | 31) + 1, all = (k1 - k0 + KEYS - 1) / KEYS;
        // this CTA's tiles: t0 .. t1 - 1
        const int per = cs > 1 ? (all + cs - 1) / cs : all, t0 = rank * per, t1 = min(all, t0 + per);
        const size_t base = kv_index(a.rw.slot0 + s, a.layer, h, k0, a.st.L, H, a.st.ctx);

        // ---- a tile on its way: copied as it is, then unpacked. A warp takes 8 keys, and byte b of the words of 32 values
        // (dims 8g + 2b, 8g + 2b + 1); positions from k1 on are neither copied nor used
        auto fetch = [&](int t, bool values) {
            if (t < t1) {
                const int left = k1 - k0 - t * KEYS;
                const size_t e = base + (size_t)t * KEYS;
                SmRaw& R = S.raw[t & 1];
                if (((tid & 127) >> 1) < left) {
                    if (tid < 128) copy16(&R.k[0][0] + tid * 16, a.st.k + e * 32 + tid * 16);
                    else if (values) copy16(&R.v[0][0] + (tid - 128) * 16, a.st.v + e * 32 + (tid - 128) * 16);
                }
                if (tid < 8) {
                    if (tid * 8 < left) copy16(&R.ks[tid * 8][0], a.st.ks + e * 2 + tid * 16);
                } else if (tid < 12) {
                    if ((tid - 8) * 16 < left) copy16(&R.vs[(tid - 8) * 16], a.st.vs + e + (tid - 8) * 16);
                }
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
        fetch(t0, false);
        fetch(t0 + 1, false);
        if (tid == 0) S.slow = 0;
        {
            int64_t x[SM_ROWS / SM_WARPS][2];
#pragma unroll
            for (int k = 0; k < SM_ROWS / SM_WARPS; k++) {
                const int r = wid + k * SM_WARPS;
                x[k][0] = x[k][1] = 0;
                const int64_t* const from_ = a.q.x + (size_t)(run.r0 + i0 + r) * a.q.ld + h * a.q.hs + 2 * lane;
                if (r < nr) load_pair(from_, wide & 1, x[k][0], x[k][1]);
            }
            uint32_t words[SM_ROWS / SM_WARPS];
            int us[SM_ROWS / SM_WARPS], most = 0;
            query_bytes(x, words, us);
#pragma unroll
            for (int k = 0; k < SM_ROWS / SM_WARPS; k++) {
                S.q[wid + k * SM_WARPS][lane] = words[k];
                if (lane == 0) S.u[wid + k * SM_WARPS] = us[k];
                most = max(most, us[k]);
            }
            if (lane == 0) S.most[wid] = most;
        }
        __syncthreads();
        // this lane's rows and their A operands: [plane][half][even row g, even g + 8, odd g, odd g + 8]
        const int ra = pair * 16 + g, rb = ra + 8;
        uint32_t q[2][2][4];
#pragma unroll
        for (int x = 0; x < 2; x++)
#pragma unroll
            for (int y = 0; y < 2; y++) {
                const uint32_t* w = &S.q[y ? rb : ra][16 * x + 4 * j];
                // hi bytes of two words: even, even, odd, odd; lo bytes the same
                const uint32_t h0 = __byte_perm(w[0], w[1], 0x6240), h1 = __byte_perm(w[2], w[3], 0x6240);
                const uint32_t l0 = __byte_perm(w[0], w[1], 0x7351), l1 = __byte_perm(w[2], w[3], 0x7351);
                q[0][x][y] = __byte_perm(h0, h1, 0x5410);
                q[0][x][2 + y] = __byte_perm(h0, h1, 0x7632);
                q[1][x][y] = __byte_perm(l0, l1, 0x5410);
                q[1][x][2 + y] = __byte_perm(l0, l1, 0x7632);
            }
        const int ua = S.u[ra], ub = S.u[rb];
        int umax = 0;
#pragma unroll
        for (int w = 0; w < SM_WARPS; w++) umax = max(umax, S.most[w]);
        const int pa = min(p_first + ra, p_last), pb = min(p_first + rb, p_last);      // rows past the last repeat it
        const int la = max(from, pa - win + 1), lb = max(from, pb - win + 1);
        const int w_p0 = min(p_first + pair * 16, p_last), w_p1 = min(p_first + pair * 16 + 15, p_last);
        const int w_l0 = max(from, w_p0 - win + 1), w_l1 = max(from, w_p1 - win + 1);
        auto arrived = [&]() { asm volatile("cp.async.wait_group 0;" ::: "memory"); };   // a barrier makes it everybody's
        auto put = [&](int t, bool values) {
            const SmRaw& R = S.raw[t & 1];
            SmTile& T = S.tile[t & 1];
            {
                const int kl = wid * 8 + g;
                const uint2 w = *reinterpret_cast<const uint2*>(&R.k[kl][8 * j]);
                const int both = *reinterpret_cast<const int16_t*>(&R.ks[kl][0]);
                const int s0 = (int8_t)both, s1 = both >> 8, big = max(s0, s1);
                const int up0 = s0 - big + 3, up1 = s1 - big + 3;
                const uint32_t less0 = 0x80808080u - (0x08080808u << up0), less1 = 0x80808080u - (0x08080808u << up1);
                T.k[wid][lane] = make_uint4(even_up(w.x, up0, less0), odd_up(w.x, up0, less0), even_up(w.y, up1, less1),
                                            odd_up(w.y, up1, less1));
                if (j == 0) {
                    T.kr[kl] = 27 - big;
                    if (27 - big < umax && k0 + t * KEYS + kl < k1) S.slow = 1;
                }
            }
            if (tid < KEYS) T.vs[tid] = R.vs[tid];
            if (values) {
                // k of an operand's first register: keys 2j, 2j + 1, 8 + 2j, 9 + 2j; of its second: 16 more
                uint32_t v[2];
#pragma unroll
                for (int c = 0; c < 2; c++) {
                    const uint8_t* r = &R.v[(wid >> 2) * 32 + 16 * c + 2 * j][4 * g + (wid & 3)];
                    v[c] = __byte_perm(__byte_perm(r[0], r[32], 0x40), __byte_perm(r[256], r[288], 0x40), 0x5410);
                }
                T.v[wid >> 2][wid & 3][lane] = make_uint4(even16(v[0]), even16(v[1]), odd16(v[0]), odd16(v[1]));
            }
        };
        // twice the rounded score (fast: its digit below the last one kept; slow: shifts up, and the limits) of tile n of
        // eight keys: rows ra and rb, keys 2j and 2j + 1
        auto scores = [&](const SmTile& T, int n, auto slow, int (&y)[4]) {
            const uint4 b = T.k[n][lane];
            int d[4];
            mma_s8_first(d, q[0][0][0], q[0][0][1], q[0][0][2], q[0][0][3], b.x, b.y);
            mma_s8(d, q[0][1][0], q[0][1][1], q[0][1][2], q[0][1][3], b.z, b.w);
#pragma unroll
            for (int x = 0; x < 4; x++) d[x] = (int)((uint32_t)d[x] << 8);
            mma_s8(d, q[1][0][0], q[1][0][1], q[1][0][2], q[1][0][3], b.x, b.y);
            mma_s8(d, q[1][1][0], q[1][1][1], q[1][1][2], q[1][1][3], b.z, b.w);
            const int2 kr = *reinterpret_cast<const int2*>(&T.kr[n * 8 + 2 * j]);
            const int r[4] = {kr.x - ua, kr.y - ua, kr.x - ub, kr.y - ub};
#pragma unroll
            for (int x = 0; x < 4; x++) y[x] = decltype(slow)::value ? 2 * store_score(d[x], r[x] + 1) : d[x] >> r[x];
        };

        // ---- pass 1
        int ya, yb, ma, mb, mw;
        auto largest = [&](const SmTile& T, int kb, auto slow, auto whole) {
            if (decltype(whole)::value) mw = max(mw, T.vs[blk * 32 + lane]);
            const uint32_t seen_a = seen(la - kb, pa - kb), seen_b = seen(lb - kb, pb - kb);
#pragma unroll
            for (int n = 0; n < 4; n++) {
                int y[4];
                scores(T, blk * 4 + n, slow, y);
                if (decltype(whole)::value) {
                    ya = max(ya, max(y[0], y[1]));
                    yb = max(yb, max(y[2], y[3]));
                } else {
                    const int2 vs = *reinterpret_cast<const int2*>(&T.vs[blk * 32 + n * 8 + 2 * j]);
                    // bits 0 and 1: whether each row sees keys 2j and 2j + 1
                    const uint32_t sa_ = seen_a >> (n * 8 + 2 * j), sb_ = seen_b >> (n * 8 + 2 * j);
                    ya = max(ya, max((sa_ & 1) ? y[0] : INT32_MIN, (sa_ & 2) ? y[1] : INT32_MIN));
                    yb = max(yb, max((sb_ & 1) ? y[2] : INT32_MIN, (sb_ & 2) ? y[3] : INT32_MIN));
                    ma = max(ma, max((sa_ & 1) ? vs.x : 0, (sa_ & 2) ? vs.y : 0));
                    mb = max(mb, max((sb_ & 1) ? vs.x : 0, (sb_ & 2) ? vs.y : 0));
                }
            }
        };
        // a pass over the CTA's tiles: tile t in the works, t + 1 unpacked, t + 2 on its way; its first two are already
        auto pass = [&](bool values, auto work) {
            arrived();
            __syncthreads();
            if (t0 < t1) put(t0, values);
            __syncthreads();
            for (int t = t0; t < t1; t++) {
                if (t + 2 < t1) {
                    fetch(t + 2, values);
                } else if (!values && t + 1 == t1) {   // both buffers are free: the next pass's first tiles
                    fetch(t0, true);
                    fetch(t0 + 1, true);
                }
                work(S.tile[t & 1], k0 + t * KEYS);
                if (t + 1 < t1) put(t + 1, values);
                arrived();
                __syncthreads();
            }
        };
        auto pass1 = [&](auto slow) {
            ya = yb = INT32_MIN;
            ma = mb = mw = 0;             // mw: of blocks that all rows see
            pass(false, [&](const SmTile& T, int kt) {
                const int kb = kt + blk * 32;
                if (kb <= w_p1 && kb + 31 >= w_l0) {
                    if (kb + 31 <= w_p0 && kb >= w_l1) largest(T, kb, slow, std::true_type());
                    else largest(T, kb, slow, std::false_type());
                }
            });
        };
        pass1(std::false_type());
        const bool slow = S.slow;         // some key's score shifts up (or not down): all again with the general form
        if (slow) {
            fetch(t0, false);             // (the second pass's tiles are fetched again after it)
            fetch(t0 + 1, false);
            pass1(std::true_type());
        }
        mw = __reduce_max_sync(0xffffffffu, mw);
        ma = max(ma, mw);
        mb = max(mb, mw);
#pragma unroll
        for (int o = 1; o < 4; o <<= 1) {
            ya = max(ya, __shfl_xor_sync(0xffffffffu, ya, o));
            yb = max(yb, __shfl_xor_sync(0xffffffffu, yb, o));
            ma = max(ma, __shfl_xor_sync(0xffffffffu, ma, o));
            mb = max(mb, __shfl_xor_sync(0xffffffffu, mb, o));
        }
        if (j == 0) {
            S.ym[wid][g] = make_int2(ya, ma);
            S.ym[wid][g + 8] = make_int2(yb, mb);
        }
        if (cs > 1) cluster_sync();
        else __syncthreads();
        for (int k = 0; k < cs; k++)
#pragma unroll
            for (int w = 0; w < 2; w++) {            // the pair's two warps, in every CTA of the cluster
                int2 oa = S.ym[2 * pair + w][g], ob = S.ym[2 * pair + w][g + 8];
                if (cs > 1) {
                    const int64_t a8 = ld_dsmem(mapa(saddr(&S.ym[2 * pair + w][g]), (uint32_t)k));
                    const int64_t b8 = ld_dsmem(mapa(saddr(&S.ym[2 * pair + w][g + 8]), (uint32_t)k));
                    oa = make_int2((int)a8, (int)(a8 >> 32));
                    ob = make_int2((int)b8, (int)(b8 >> 32));
                }
                ya = max(ya, oa.x);
                yb = max(yb, ob.x);
                ma = max(ma, oa.y);
                mb = max(mb, ob.y);
            }
        // the next item's queries into L2 (a row is four lines)
        if (n_tile >= 0 && n_r0 >= 0 && n_r1 <= a.rw.rows) {
            const int row = n_r0 + n_tile * ROWS + (tid >> 2);
            const int64_t* const line = a.q.x + (size_t)row * a.q.ld + n_h * a.q.hs + (tid & 3) * 16;
            if (row < n_r1) asm volatile("prefetch.global.L2 [%0];" ::"l"(line));
        }
        // twice the largest score: a digit below the last rounds up with it
        const uint32_t sa = (uint32_t)(((ya >> 1) + (ya & 1)) * 2), sb = (uint32_t)(((yb >> 1) + (yb & 1)) * 2);

        // ---- pass 2
        int acc[3][4][4];                     // [plane][tile 4 (wid & 1) + t]
#pragma unroll
        for (int x = 0; x < 3; x++)
#pragma unroll
            for (int t = 0; t < 4; t++)
#pragma unroll
                for (int c = 0; c < 4; c++) acc[x][t][c] = 0;
        int64_t za = 0, zb = 0;
        auto weights = [&](const SmTile& T, int kb, auto slow, auto whole) {
            uint32_t p[3][4];                 // the weights' planes as A operands
            int32_t s_a = 0, s_b = 0;         // 8 entries of at most 2^24
            const uint32_t seen_a = seen(la - kb, pa - kb), seen_b = seen(lb - kb, pb - kb);
#pragma unroll
            for (int n = 0; n < 4; n += 2) {
                uint32_t wa[4], wb[4];
#pragma unroll
                for (int x = 0; x < 2; x++) {
                    int y[4];
                    scores(T, blk * 4 + n + x, slow, y);
                    const int2 vs = *reinterpret_cast<const int2*>(&T.vs[blk * 32 + (n + x) * 8 + 2 * j]);
                    // start - score, from twice both: (start2 - y) / 2 rounded down
                    uint32_t d[4] = {(sa - (uint32_t)y[0]) >> 1, (sa - (uint32_t)y[1]) >> 1, (sb - (uint32_t)y[2]) >> 1,
                                     (sb - (uint32_t)y[3]) >> 1};
#pragma unroll
                    for (int c = 0; c < 4; c++) d[c] = min(d[c], (uint32_t)alen);
                    if (!decltype(whole)::value) {
                        const uint32_t sa_ = seen_a >> ((n + x) * 8 + 2 * j), sb_ = seen_b >> ((n + x) * 8 + 2 * j);
                        d[0] = (sa_ & 1) ? d[0] : alen;
                        d[1] = (sa_ & 2) ? d[1] : alen;
                        d[2] = (sb_ & 1) ? d[2] : alen;
                        d[3] = (sb_ & 2) ? d[3] : alen;
                    }
                    const int v[4] = {TAB[d[0]], TAB[d[1]], TAB[d[2]], TAB[d[3]]};
                    s_a += v[0] + v[1];
                    s_b += v[2] + v[3];
                    // rnd(a, 1 + M - vs); a key that a row does not see (whose vs may pass M) has a = 0
                    wa[2 * x] = (shr_u32(v[0], ma - vs.x) + 1) >> 1;
                    wa[2 * x + 1] = (shr_u32(v[1], ma - vs.y) + 1) >> 1;
                    wb[2 * x] = (shr_u32(v[2], mb - vs.x) + 1) >> 1;
                    wb[2 * x + 1] = (shr_u32(v[3], mb - vs.y) + 1) >> 1;
                }
                turn3(wa, p[0][n], p[1][n], p[2][n]);
                turn3(wb, p[0][n + 1], p[1][n + 1], p[2][n + 1]);
            }
            za += s_a;
            zb += s_b;
#pragma unroll
            for (int z = 0; z < 3; z++) S.p[wid][z][lane] = make_uint4(p[z][0], p[z][1], p[z][2], p[z][3]);
        };
        // a block's weights times its values, this warp's half of the dims
        auto add = [&](const SmTile& T, int b) {
            const uint4* const v = &T.v[b][2 * (wid & 1)][lane];
            const uint4 v0 = v[0], v1 = v[32];
#pragma unroll
            for (int z = 0; z < 3; z++) {
                const uint4 p = S.p[(wid & ~1) + b][z][lane];
                mma_u8s8(acc[z][0], p.x, p.y, p.z, p.w, v0.x, v0.y);
                mma_u8s8(acc[z][1], p.x, p.y, p.z, p.w, v0.z, v0.w);
                mma_u8s8(acc[z][2], p.x, p.y, p.z, p.w, v1.x, v1.y);
                mma_u8s8(acc[z][3], p.x, p.y, p.z, p.w, v1.z, v1.w);
            }
        };
        auto pass2 = [&](auto slow) {
            pass(true, [&](const SmTile& T, int kt) {
                const int kb = kt + blk * 32;
                if (kb <= w_p1 && kb + 31 >= w_l0) {
                    if (kb + 31 <= w_p0 && kb >= w_l1) weights(T, kb, slow, std::true_type());
                    else weights(T, kb, slow, std::false_type());
                }
                const bool b0 = kt <= w_p1 && kt + 31 >= w_l0, b1 = kt + 32 <= w_p1 && kt + 63 >= w_l0;
                if (b0 || b1) asm volatile("bar.sync %0, 64;" ::"r"(1 + pair) : "memory");   // both warps of the pair
                if (b0) add(T, 0);
                if (b1) add(T, 1);
            });
        };
        if (slow) pass2(std::true_type());
        else pass2(std::false_type());
#pragma unroll
        for (int o = 1; o < 4; o <<= 1) {
            za += __shfl_xor_sync(0xffffffffu, za, o);
            zb += __shfl_xor_sync(0xffffffffu, zb, o);
        }
        if (j == 0) {
            S.z[wid][g] = za;
            S.z[wid][g + 8] = zb;
        }
        // a lane's 8 sums of each of its rows; a cluster's CTAs lay theirs out (in place of the tiles) a row at a time and
        // each finishes some of them
        int64_t* const part = reinterpret_cast<int64_t*>(S.tile);     // [warp][8][32 lanes]
        auto sum = [&](int c, int t, int y) {
            return (int64_t)acc[0][t][2 * y + c] + (int64_t)acc[1][t][2 * y + c] * 256 + (int64_t)acc[2][t][2 * y + c] * 65536;
        };
        if (cs > 1) cluster_sync();                                   // the tiles are done with, S.z is complete
        else __syncthreads();
        uint32_t e[2];
        int sh[2];
#pragma unroll
        for (int y = 0; y < 2; y++) {
            int64_t z = 0;
            for (int k = 0; k < cs; k++)
#pragma unroll
                for (int w = 0; w < 2; w++) {
                    if (cs > 1) z += ld_dsmem(mapa(saddr(&S.z[2 * pair + w][g + 8 * y]), (uint32_t)k));
                    else z += S.z[2 * pair + w][g + 8 * y];
                }
            const bool none = (y ? lb > pb : la > pa) || z == 0;
            const int64_t F = 65536ll * ((y ? mb : ma) + STORE_W_SHIFT) - log2fix(none ? 1 : z, a.LOG2);
            e[y] = none ? 0 : (uint32_t)__ldg(a.EXP2 + (F & 0xFFFF));
            sh[y] = 19 - (int)(F >> 16);                              // less one, and 4 digits more: the tiles hold 16 c
        }
#pragma unroll
        for (int y = 0; y < 2; y++) {
            const int r = y ? rb : ra;
            if (cs > 1) {
#pragma unroll
                for (int x = 0; x < 8; x++) part[(wid * 8 + x) * 32 + lane] = sum(x >> 2, x & 3, y);
                cluster_sync();
            }
            int64_t* const out = a.out + ((size_t)(run.r0 + i0 + r) * H + h) * 64 + 16 * j + 4 * (wid & 1);
            // columns 2j, 2j + 1 of tile t: dims 16j + t, 16j + 8 + t
            int64_t o[8];
#pragma unroll
            for (int x = 0; x < 8; x++) {
                o[x] = 0;
                if (cs == 1) {
                    o[x] = sum(x >> 2, x & 3, y);
                } else if ((x >> 1) % cs == rank) {
                    for (int m = 0; m < cs; m++) o[x] += ld_dsmem(mapa(saddr(&part[(wid * 8 + x) * 32 + lane]), (uint32_t)m));
                }
                o[x] *= (int64_t)e[y];                                 // at most 2^46 2^17
            }
            if (sh[y] >= 0) {
#pragma unroll
                for (int x = 0; x < 8; x++) o[x] = ((o[x] >> sh[y]) + 1) >> 1;
            } else {
#pragma unroll
                for (int x = 0; x < 8; x++) o[x] = (int64_t)((uint64_t)o[x] << (-1 - sh[y]));
            }
            if (r < nr) {
#pragma unroll
                for (int x = 0; x < 8; x += 2) {
                    if (cs > 1 && (x >> 1) % cs != rank) continue;
                    int64_t* const to = out + 8 * (x >> 2) + (x & 3);
                    if (wide & 2) {
                        *reinterpret_cast<longlong2*>(to) = make_longlong2(o[x], o[x + 1]);
                    } else {
                        to[0] = o[x];
                        to[1] = o[x + 1];
                    }
                }
            }
            if (cs > 1) cluster_sync();                                // the others have read this CTA's sums
        }
    }
}

// ---- launches -------------------------------------------------------------------------------------------------------
namespace {
template <typename... KArgs, typename... Args>
cudaError_t store_launch(StoreLaunch how, void (*kernel)(KArgs...), dim3 grid, int threads, size_t smem, int cluster, Args... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = how.stream;
    cudaLaunchAttribute at[2];
    int n = 0;
    if (cluster > 1) {
        at[n].id = cudaLaunchAttributeClusterDimension;
        at[n].val.clusterDim.x = cluster;
        at[n].val.clusterDim.y = 1;
        at[n++].val.clusterDim.z = 1;
    }
    if (how.pdl) {
        at[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        at[n++].val.programmaticStreamSerializationAllowed = 1;
    }
    cfg.attrs = at;
    cfg.numAttrs = n;
    return cudaLaunchKernelEx(&cfg, kernel, ((KArgs)args)...);
}
bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }
bool pairs(const StoreVec& v) { return aligned16(v.x) && v.ld % 2 == 0 && v.hs % 2 == 0; }   // every pair of dims in one load
}  // namespace

namespace {
// rows a warp: one where streams give few (a decode step: more warps, the least latency), else eight
constexpr int SW_ROWS = 8;
dim3 row_grid(const Store4& st, const StoreRows& rw, int u) {
    return dim3((unsigned)(((int64_t)((rw.max_rows + u - 1) / u) * 2 * st.H + SW_WARPS - 1) / SW_WARPS), rw.n_streams);
}
}  // namespace

cudaError_t store_write(const Store4& st, const StoreRows& rw, int layer, const StoreVec& k, const StoreVec& v, uint32_t* err,
                        StoreLaunch how, uint64_t* stamp) {
    if (rw.n_streams == 0 || rw.rows == 0) return cudaSuccess;
    const int wide = pairs(k) && pairs(v);
    const bool few = rw.max_rows < SW_ROWS;
    const int64_t items = few ? (int64_t)rw.max_rows * 2 * st.H : (int64_t)((rw.max_rows + SW_ROWS - 1) / SW_ROWS) * 4 * 2 * st.H;
    const dim3 grid((unsigned)((items + SW_WARPS * 4 - 1) / (SW_WARPS * 4)), rw.n_streams);
    return few ? store_launch(how, k_store_write<1>, grid, SW_WARPS * 32, 0, 1, st, rw, layer, k, v, wide, err, stamp)
               : store_launch(how, k_store_write<2>, grid, SW_WARPS * 32, 0, 1, st, rw, layer, k, v, wide, err, stamp);
}

cudaError_t store_read(const Store4& st, const StoreRows& rw, int layer, int64_t* k, int64_t* v, uint32_t* err, StoreLaunch how) {
    if (rw.n_streams == 0 || rw.rows == 0) return cudaSuccess;
    const int wide = aligned16(k) && aligned16(v);
    if (rw.max_rows < SW_ROWS)
        return store_launch(how, k_store_read<1>, row_grid(st, rw, 1), SW_WARPS * 32, 0, 1, st, rw, layer, k, v, wide, err);
    return store_launch(how, k_store_read<SW_ROWS>, row_grid(st, rw, SW_ROWS), SW_WARPS * 32, 0, 1, st, rw, layer, k, v, wide, err);
}

// the few-row kernel is quicker up to so many rows a stream (4 streams on 2,000 positions: 12 rows 21 us, the many-row kernel 38;
// 32 rows 50 and 40), and of more rows while there is little to do in all: (row, head)s times their blocks of 32 keys and a
// start of SF_START more, an SM (in stores that just hold them: one prompt of 64 rows 8.8 and 14.3 us, of 256 13.5 and 20.6,
// 2 x 48 rows on 700 19 and 27; past it 8 x 32 rows on 500 32.6 and 29.7, 16 prompts of 64 19.2 and 16.4)
constexpr int SM_FROM_ROWS = 20, SF_START = 3, SF_LITTLE = 340;
constexpr int SM_FIXED = 4, SM_SPLIT = 6;
constexpr int SM_SMEM_MOST = 200 * 1024;
constexpr int SF_MOST_KEYS = 8192;   // of a CTA: 40 KB of shared memory
// The rules from here on go by the positions that a row may see, the store's context (or the window), since what the streams
// hold is on the device: in a store much larger than its streams they choose for keys that are not there (64 x 160 in a store of
// 160, 1,024, 2,048 and 32,768 positions, calls in a graph: 5.4, 6.5, 10 and 62 us; 512 x 192: 17, 18, 62 and 487).
// A warp a unit where units are many and short: from SF_WARP_UNITS an SM on up to 1,024 keys (20 KB a CTA; 200 x 160, 16 an SM:
// 10.1 us against 13.6); an arrival (not a step) also below that, where the blocks of 32 keys are at most twice the units an SM
// less five, a line through the crossings measured (64 x 160, 5 an SM of 5 blocks: 5.8 against 6.1, 64 x 256 7.7 against 6.9;
// 140 x 256, 11 an SM of 8: 9.5 against 13.3, 100 x 900 30 against 23; a step's one warp would put the row's own key and value
// first: 64 x 160 in the engine 0.605 ms a step against 0.581)
constexpr int SF_WARP_UNITS = 12, SF_WARP_BLOCKS = 32;
// blocks of 32 keys a warp from which they come through the ring, three on their way: 100 x 900 (8 blocks) 26.6 us straight into
// registers, 22.8 through the ring, 512 x 192 (6) 22.3 and 21.1, 4 x 32,768 (16) 30.8 and 29.3; but 200 x 160 (5) 10.1 and 11.0,
// 16 x 1,024 (4) 7.1 and 8.1: a copy into shared memory and the load from it come later than a load
constexpr int SF_RING_FROM = 6;
// blocks of 32 keys a CTA from which it has 8 warps: 32 where there are few CTAs (16 x 1,024, 192 of them: 7.1 us against 8.2
// with four; 20 x 1,024, 240: 8.9 against 8.2), else 48, where the ring begins (64 x 1,024 20.7 against 16.4 with four)
constexpr int SF_LONG = 32, SF_LONG_MANY = SF_RING_FROM * 8, SF_VERY_LONG = 64;

size_t few_smem(int warps, int keys, bool ring) { return (ring ? warps * SF_RING * sizeof(SfBlock) : 0) + (size_t)keys * SF_BYTES; }
size_t many_smem(int alen) { return sizeof(SmShared) + (size_t)(alen + 1) * 4; }

namespace {
// the most shared memory that a launch of these asks for
template <int NW>
cudaError_t few_room() {
    cudaError_t e = cudaSuccess;
    for (auto f : {k_store_attend_few<NW, false, false>, k_store_attend_few<NW, false, true>, k_store_attend_few<NW, true, false>,
                   k_store_attend_few<NW, true, true>})
        if (e == cudaSuccess)
            e = cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)few_smem(16, SF_MOST_KEYS, true));
    return e;
}

cudaError_t make_plan(int device, int alen, StorePlan& plan) {
    cudaError_t e = cudaDeviceGetAttribute(&plan.sms, cudaDevAttrMultiProcessorCount, device);
    for (auto room : {few_room<1>, few_room<4>, few_room<8>, few_room<16>})
        if (e == cudaSuccess) e = room();
    if (e == cudaSuccess)
        e = cudaFuncSetAttribute(k_store_attend_many, cudaFuncAttributeMaxDynamicSharedMemorySize, SM_SMEM_MOST);
    if (e != cudaSuccess) return e;
    int fit = 0;
    e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&fit, k_store_attend_many, SM_THREADS, many_smem(alen));
    if (e != cudaSuccess) return e;
    plan.many[1] = fit * plan.sms;
    for (int cs = 2; cs <= STORE_MAX_CLUSTER; cs++) {
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3(cs);
        cfg.blockDim = dim3(SM_THREADS);
        cfg.dynamicSmemBytes = many_smem(alen);
        cudaLaunchAttribute at[1];
        at[0].id = cudaLaunchAttributeClusterDimension;
        at[0].val.clusterDim.x = cs;
        at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
        cfg.attrs = at;
        cfg.numAttrs = 1;
        if (cudaOccupancyMaxActiveClusters(&plan.many[cs], k_store_attend_many, &cfg) != cudaSuccess) {
            plan.many[cs] = 0;
            cudaGetLastError();
        }
    }
    return cudaSuccess;
}

// the plans made so far: a few devices and table lengths a process
std::mutex g_plan_mu;
struct PlanAt { int device, alen; StorePlan plan; };
std::vector<PlanAt> g_plans;
}  // namespace

cudaError_t store_init(int alen, StorePlan& plan) {
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e != cudaSuccess) return e;
    std::lock_guard<std::mutex> lock(g_plan_mu);
    for (const PlanAt& p : g_plans)
        if (p.device == device && p.alen == alen) {
            plan = p.plan;
            return cudaSuccess;
        }
    e = make_plan(device, alen, plan);
    if (e == cudaSuccess) g_plans.push_back(PlanAt{device, alen, plan});
    return e;
}

namespace {
// NW warps a (row, head) (a CTA of four for one warp), `each` blocks of 32 keys a CTA at most
template <int NW, bool PUT>
cudaError_t few_launch(const StoreAttend& a, StoreLaunch how, int wide, dim3 grid, int each, int cs) {
    const int chunk = each * 32, warps = NW == 1 ? 4 : NW;
    const bool ring = each >= NW * SF_RING_FROM;
    return store_launch(how, ring ? k_store_attend_few<NW, PUT, true> : k_store_attend_few<NW, PUT, false>, grid, warps * 32,
                        few_smem(warps, NW == 1 ? chunk * 4 : chunk, ring), cs, a, chunk, cs, wide);
}

// blocks of 32 positions that a row may see
int few_blocks(const StoreAttend& a) {
    const int blocks = (a.st.lim + 31) / 32;
    return a.window > 0 && a.window < a.st.lim ? std::min(blocks, (a.window + 30) / 32 + 1) : blocks;
}

template <bool PUT>
cudaError_t attend_few(const StoreAttend& a, StoreLaunch how, int wide) {
    const int blocks = few_blocks(a);
    const int64_t units = (int64_t)a.rw.n_streams * a.rw.max_rows * a.st.H;
    const int sms = how.plan->sms;
    if (blocks <= SF_WARP_BLOCKS && (units >= (int64_t)SF_WARP_UNITS * sms || (!PUT && (int64_t)(blocks + 5) * sms <= 2 * units)))
        return few_launch<1, PUT>(a, how, wide, dim3((unsigned)(((int64_t)a.rw.max_rows * a.st.H + 3) / 4), a.rw.n_streams), blocks, 1);
    // a cluster costs about 1.3 us (its barriers), a warp's block of 32 keys 0.5 (from L2) to 1.2 us (from HBM): the keys are
    // split where that leaves half the SMs idle, and while there is a long run of keys for every CTA of two an SM
    int cs = 1;
    while (cs < STORE_MAX_CLUSTER && ((units * cs * 2 <= sms && blocks >= SF_LONG && blocks >= cs * 8) ||
                                      (units * cs < sms * 2 && blocks >= cs * SF_VERY_LONG) ||
                                      blocks * 32 > cs * SF_MOST_KEYS))
        cs *= 2;
    const int each = (blocks + cs - 1) / cs;
    const dim3 grid((unsigned)((int64_t)a.rw.max_rows * a.st.H * cs), a.rw.n_streams);
    if (each >= SF_VERY_LONG && units * cs <= sms) return few_launch<16, PUT>(a, how, wide, grid, each, cs);   // one CTA an SM
    if (each >= SF_LONG_MANY || (each >= SF_LONG && units * cs * 2 < sms * 3)) return few_launch<8, PUT>(a, how, wide, grid, each, cs);
    return few_launch<4, PUT>(a, how, wide, grid, each, cs);
}
int wide_bits(const StoreAttend& a) {
    return pairs(a.q) | aligned16(a.out) << 1 | pairs(a.k) << 2 | pairs(a.v) << 3;
}
}  // namespace

cudaError_t store_step(const StoreAttend& a, StoreLaunch how) {
    if (a.rw.n_streams == 0 || a.rw.rows == 0) return cudaSuccess;
    return attend_few<true>(a, how, wide_bits(a));
}

cudaError_t store_attend(const StoreAttend& a, StoreLaunch how) {
    if (a.rw.n_streams == 0 || a.rw.rows == 0) return cudaSuccess;
    const int wide = wide_bits(a);
    const int64_t items = (int64_t)((a.rw.max_rows + SM_ROWS - 1) / SM_ROWS) * a.st.H * a.rw.n_streams;
    const int64_t work = (int64_t)a.rw.n_streams * a.rw.max_rows * a.st.H * (few_blocks(a) + SF_START);
    if (a.rw.max_rows > SM_FROM_ROWS && work > (int64_t)SF_LITTLE * how.plan->sms && items < INT32_MAX) {
        const int tiles = (a.rw.max_rows + SM_ROWS - 1) / SM_ROWS;
        const size_t smem = many_smem(a.alen);
        // fewer items than half of what the GPU holds: their keys split over clusters, in two tiles a CTA at least, by the
        // time that a split would take (waves x tiles a CTA, an item's start and end counted as SM_FIXED tiles, a cluster's
        // barriers and sums as SM_SPLIT more: 2 x 256 rows on 8,000 positions 263 us whole, 182 on clusters of five; 8 x 64
        // on 500 30 us whole, 33 on pairs)
        const int keys = a.window > 0 ? std::min(a.st.lim, std::min(a.window, a.st.lim) + SM_ROWS) : a.st.lim;
        const int all = (keys + SM_KEYS - 1) / SM_KEYS;
        int cs = 1;
        int64_t least = INT64_MAX;
        for (int k = 1; k <= STORE_MAX_CLUSTER && (k == 1 || (k * 2 <= all && items * 2 <= how.plan->many[1])); k++) {
            const int fit = how.plan->many[k];
            if (fit < 1) continue;
            const int64_t t = (items + fit - 1) / fit * ((all + k - 1) / k + SM_FIXED + (k > 1 ? SM_SPLIT : 0));
            if (t < least) {
                least = t;
                cs = k;
            }
        }
        const dim3 grid((unsigned)(std::min<int64_t>(items, std::max(how.plan->many[cs], 1)) * cs));
        return store_launch(how, k_store_attend_many, grid, SM_THREADS, smem, cs, a, tiles, cs, wide);
    }
    return attend_few<false>(a, how, wide);
}

}  // namespace b2

// =====================================================================================================================
// C ABI
// =====================================================================================================================
using namespace b2;

struct b2_store {
    b2_store_config cfg{};
    int device = 0;
    std::string err;
    Store4 st{};
    int32_t *ARR = nullptr, *LOG2 = nullptr, *EXP2 = nullptr;
    int alen = 0;
    StorePlan plan;
    uint32_t* d_err = nullptr;
    void* own = nullptr;      // the memory, where the library allocated it
};

namespace {

int sfail(b2_store* h, int code, const char* fmt, ...) {
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof buf, fmt, ap);
    va_end(ap);
    if (h) h->err = buf;
    return code;
}

// the store's device current for the length of a call, the caller's back afterwards
struct OnDevice {
    int before = -1;
    cudaError_t e;
    explicit OnDevice(int device) {
        e = cudaGetDevice(&before);
        if (e == cudaSuccess && before != device) e = cudaSetDevice(device);
        else before = -1;
    }
    ~OnDevice() {
        if (before >= 0) cudaSetDevice(before);
    }
};

#define SCK(call)                                                                                     \
    do {                                                                                              \
        cudaError_t e_ = (call);                                                                      \
        if (e_ != cudaSuccess) {                                                                      \
            cudaGetLastError(); /* nothing is left behind for the next call's check */                \
            return sfail(h, B2_ERR_CUDA, "%s: %s", #call, cudaGetErrorString(e_));                    \
        }                                                                                             \
    } while (0)

// a table's entries as 32 bits; where one lies outside [lo, hi], an error that names it
int table32(b2_store* h, int32_t* to, const int64_t* from, int64_t n, int64_t lo, int64_t hi, const char* name) {
    int64_t least = from[0], most = from[0];
    for (int64_t i = 0; i < n; i++) {
        least = std::min(least, from[i]);
        most = std::max(most, from[i]);
        to[i] = (int32_t)from[i];
    }
    if (least >= lo && most <= hi) return B2_OK;
    return sfail(h, B2_ERR_VALUE, "b2_store_create: %s holds %lld .. %lld, its entries lie in [%lld, %lld]", name, (long long)least,
                 (long long)most, (long long)lo, (long long)hi);
}

void store_release(b2_store* h) {
    if (h->own) cudaFree(h->own);
    h->own = nullptr;
    h->d_err = nullptr;
}

// the store's one piece of memory: the arrays, then (16-byte aligned) four error words and the tables
constexpr size_t TABLE_WORDS = 4 + 2 * 65536;
size_t store_bytes(const b2_store_config& c, int64_t n_arrival, Store4* st = nullptr, void* at = nullptr, size_t* tables = nullptr) {
    Store4 tmp;
    const size_t n = (store_layout(st ? *st : tmp, c.n_slots, c.n_layer, c.n_head, c.max_ctx, at) + 15) / 16 * 16;
    if (tables) *tables = n;
    return n + (TABLE_WORDS + (size_t)n_arrival) * sizeof(int32_t);
}

bool config_ok(const b2_store_config* c, int64_t n_arrival) {
    return c && n_arrival >= 1 && n_arrival <= STORE_MAX_ALEN && c->n_slots >= 1 && c->n_slots <= 65535 && c->n_layer >= 1 &&
           c->n_layer <= 1024 && c->n_head >= 1 && c->n_head <= 1024 && c->max_ctx >= 1 && c->max_ctx <= STORE_MAX_CTX;
}

int store_build(b2_store* h, const int64_t* arrival, int64_t n_arrival, const int64_t* log2, const int64_t* exp2, void* memory) {
    const b2_store_config& c = h->cfg;
    if (arrival[0] < 1) return sfail(h, B2_ERR_VALUE, "b2_store_create: arrival[0] = %lld (at least 1)", (long long)arrival[0]);
    std::vector<int32_t> t(TABLE_WORDS + (size_t)n_arrival, 0);
    int rc;
    if ((rc = table32(h, t.data() + 4, log2, 65536, 0, 65536, "log2")) ||
        (rc = table32(h, t.data() + 4 + 65536, exp2, 65536, 65536, 131071, "exp2")) ||
        (rc = table32(h, t.data() + TABLE_WORDS, arrival, n_arrival, 0, STORE_MAX_ARR, "arrival")))
        return rc;
    SCK(store_init((int)n_arrival, h->plan));
    uint8_t* mem = (uint8_t*)memory;
    if (!mem) {
        const size_t bytes = store_bytes(c, n_arrival);
        const cudaError_t e = cudaMalloc(&h->own, bytes);
        if (e != cudaSuccess) {
            cudaGetLastError();
            h->own = nullptr;
            return sfail(h, B2_ERR_NOMEM, "b2_store_create: cudaMalloc(%zu bytes): %s", bytes, cudaGetErrorString(e));
        }
        mem = (uint8_t*)h->own;
    }
    size_t tables = 0;
    store_bytes(c, n_arrival, &h->st, mem, &tables);
    SCK(cudaDeviceSynchronize());        // given memory may still be in use by earlier work
    SCK(cudaMemset(mem, 0, tables));
    int32_t* const d = (int32_t*)(mem + tables);
    SCK(cudaMemcpy(d, t.data(), sizeof(int32_t) * t.size(), cudaMemcpyHostToDevice));
    SCK(cudaDeviceSynchronize());
    h->LOG2 = d + 4;
    h->EXP2 = h->LOG2 + 65536;
    h->ARR = d + TABLE_WORDS;
    h->alen = (int)n_arrival;
    h->d_err = (uint32_t*)d;
    return B2_OK;
}

// the arguments that every call on rows has
int check_rows(b2_store* h, const char* what, int32_t layer, const int32_t* cu, const int32_t* pos, int32_t n_streams,
               int32_t rows, int32_t max_rows) {
    const b2_store_config& c = h->cfg;
    if (layer < 0 || layer >= c.n_layer) return sfail(h, B2_ERR_ARG, "%s: layer %d of %d", what, layer, c.n_layer);
    if (n_streams < 0 || n_streams > c.n_slots) return sfail(h, B2_ERR_ARG, "%s: n_streams %d of %d slots", what, n_streams, c.n_slots);
    if (rows < 0 || max_rows < 0) return sfail(h, B2_ERR_ARG, "%s: rows %d, max_rows %d", what, rows, max_rows);
    if (!cu && (rows != n_streams || max_rows != (rows ? 1 : max_rows)))
        return sfail(h, B2_ERR_ARG, "%s: without cu every stream gives one row (rows %d, n_streams %d, max_rows %d)", what, rows,
                     n_streams, max_rows);
    if (rows && (!pos || !n_streams || !max_rows))
        return sfail(h, B2_ERR_ARG, "%s: %d rows of %d streams, max_rows %d, pos %p", what, rows, n_streams, max_rows, (const void*)pos);
    return B2_OK;
}

// a bound past the context says no more than the context
StoreRows call_rows(const b2_store* h, const int32_t* cu, const int32_t* pos, int32_t n_streams, int32_t rows, int32_t max_rows) {
    return StoreRows{cu, pos, n_streams, rows, std::min(max_rows, h->cfg.max_ctx)};
}

// nothing that is thrown (memory for a message, a table) passes the C boundary
template <class F>
int guarded(b2_store* h, F f) {
    try {
        return f();
    } catch (const std::bad_alloc&) {
        return B2_ERR_NOMEM;
    } catch (const std::exception& e) {
        return sfail(h, B2_ERR_ARG, "%s", e.what());
    }
}

}  // namespace

extern "C" {

const char* b2_store_last_error(const b2_store* h) { return h ? h->err.c_str() : "null store"; }

int64_t b2_store_size(const b2_store_config* cfg, int64_t n_arrival) {
    return config_ok(cfg, n_arrival) ? (int64_t)store_bytes(*cfg, n_arrival) : -1;
}

int b2_store_create(const b2_store_config* cfg, int device, const int64_t* arrival, int64_t n_arrival, const int64_t* log2,
                    const int64_t* exp2, void* memory, b2_store** out) {
    if (!out) return B2_ERR_ARG;
    *out = nullptr;
    if (!config_ok(cfg, n_arrival) || !arrival || !log2 || !exp2 || ((uintptr_t)memory & 31)) return B2_ERR_ARG;
    OnDevice on(device);
    if (on.e != cudaSuccess) {
        cudaGetLastError();
        return B2_ERR_CUDA;
    }
    b2_store* h = new (std::nothrow) b2_store();
    if (!h) return B2_ERR_NOMEM;
    const int rc = guarded(h, [&] {
        h->cfg = *cfg;
        h->device = device;
        return store_build(h, arrival, n_arrival, log2, exp2, memory);
    });
    *out = h;      // on an error the store holds its message; b2_store_destroy frees it all the same
    if (rc) store_release(h);
    return rc;
}

int b2_store_write(b2_store* h, int32_t layer, const int64_t* k, int64_t ldk, const int64_t* v, int64_t ldv, const int32_t* cu,
                   const int32_t* pos, int32_t n_streams, int32_t rows, int32_t max_rows, void* stream) {
    if (!h || !h->d_err) return B2_ERR_ARG;
    return guarded(h, [&] {
        int rc = check_rows(h, "b2_store_write", layer, cu, pos, n_streams, rows, max_rows);
        if (rc) return rc;
        const int64_t d = 64ll * h->cfg.n_head;
        if (rows && (!k || !v || ldk < d || ldv < d))
            return sfail(h, B2_ERR_ARG, "b2_store_write: k %p (stride %lld), v %p (stride %lld), rows of %lld", (const void*)k,
                         (long long)ldk, (const void*)v, (long long)ldv, (long long)d);
        OnDevice on(h->device);
        SCK(on.e);
        SCK(store_write(h->st, call_rows(h, cu, pos, n_streams, rows, max_rows), layer, StoreVec{k, ldk, 64}, StoreVec{v, ldv, 64}, h->d_err,
                        StoreLaunch{(cudaStream_t)stream, true, &h->plan}));
        return (int)B2_OK;
    });
}

int b2_store_read(b2_store* h, int32_t layer, const int32_t* cu, const int32_t* pos, int32_t n_streams, int32_t rows,
                  int32_t max_rows, int64_t* k, int64_t* v, void* stream) {
    if (!h || !h->d_err) return B2_ERR_ARG;
    return guarded(h, [&] {
        int rc = check_rows(h, "b2_store_read", layer, cu, pos, n_streams, rows, max_rows);
        if (rc) return rc;
        if (rows && !k && !v) return sfail(h, B2_ERR_ARG, "b2_store_read: neither k nor v asked for");
        OnDevice on(h->device);
        SCK(on.e);
        SCK(store_read(h->st, call_rows(h, cu, pos, n_streams, rows, max_rows), layer, k, v, h->d_err,
                       StoreLaunch{(cudaStream_t)stream, true, &h->plan}));
        return (int)B2_OK;
    });
}

int b2_store_attend(b2_store* h, int32_t layer, const int64_t* q, int64_t ldq, const int32_t* cu, const int32_t* pos,
                    const int32_t* first, int32_t n_streams, int32_t rows, int32_t max_rows, int32_t window, int64_t* out,
                    void* stream) {
    if (!h || !h->d_err) return B2_ERR_ARG;
    return guarded(h, [&] {
        int rc = check_rows(h, "b2_store_attend", layer, cu, pos, n_streams, rows, max_rows);
        if (rc) return rc;
        if (window < 0 || (rows && (!q || !out || ldq < 64ll * h->cfg.n_head)))
            return sfail(h, B2_ERR_ARG, "b2_store_attend: q %p (stride %lld), out %p, window %d", (const void*)q, (long long)ldq,
                         (const void*)out, window);
        OnDevice on(h->device);
        SCK(on.e);
        StoreAttend a{h->st, call_rows(h, cu, pos, n_streams, rows, max_rows), layer, StoreVec{q, ldq, 64}, first, window, h->ARR, h->alen,
                      h->LOG2, h->EXP2, out, nullptr, h->d_err};
        SCK(store_attend(a, StoreLaunch{(cudaStream_t)stream, true, &h->plan}));
        return (int)B2_OK;
    });
}

int b2_store_step(b2_store* h, int32_t layer, const int64_t* q, int64_t ldq, const int64_t* k, int64_t ldk, const int64_t* v,
                  int64_t ldv, const int32_t* pos, const int32_t* first, int32_t n_streams, int32_t window, int64_t* out,
                  void* stream) {
    if (!h || !h->d_err) return B2_ERR_ARG;
    return guarded(h, [&] {
        int rc = check_rows(h, "b2_store_step", layer, nullptr, pos, n_streams, n_streams, n_streams ? 1 : 0);
        if (rc) return rc;
        const int64_t d = 64ll * h->cfg.n_head;
        if (window < 0 || (n_streams && (!q || !k || !v || !out || ldq < d || ldk < d || ldv < d)))
            return sfail(h, B2_ERR_ARG, "b2_store_step: q %p (stride %lld), k %p (%lld), v %p (%lld), out %p, window %d", (const void*)q,
                         (long long)ldq, (const void*)k, (long long)ldk, (const void*)v, (long long)ldv, (const void*)out, window);
        OnDevice on(h->device);
        SCK(on.e);
        StoreAttend a{h->st, StoreRows{nullptr, pos, n_streams, n_streams, 1}, layer, StoreVec{q, ldq, 64}, first, window, h->ARR,
                      h->alen, h->LOG2, h->EXP2, out, nullptr, h->d_err};
        a.k = StoreVec{k, ldk, 64};
        a.v = StoreVec{v, ldv, 64};
        SCK(store_step(a, StoreLaunch{(cudaStream_t)stream, true, &h->plan}));
        return (int)B2_OK;
    });
}

int b2_store_sync(b2_store* h) {
    if (!h || !h->d_err) return B2_ERR_ARG;
    return guarded(h, [&] {
        OnDevice on(h->device);
        SCK(on.e);
        SCK(cudaDeviceSynchronize());
        uint32_t e = 0;
        SCK(cudaMemcpy(&e, h->d_err, sizeof e, cudaMemcpyDeviceToHost));
        if (!e) return (int)B2_OK;
        SCK(cudaMemset(h->d_err, 0, sizeof(uint32_t)));
        if (e & DERR_ROWS)
            return sfail(h, B2_ERR_ARG, "a stream's rows did not fit the call: cu decreasing, past rows, or more than max_rows "
                         "(device check, bits 0x%x)", e);
        if (e & DERR_POS) return sfail(h, B2_ERR_CTX, "a position passed the store's context (device check, bits 0x%x)", e);
        return sfail(h, B2_ERR_DEVICE, "device check, bits 0x%x", e);
    });
}

void b2_store_destroy(b2_store* h) {
    if (!h) return;
    {
        OnDevice on(h->device);
        cudaDeviceSynchronize();
        store_release(h);
    }
    delete h;
}

}  // extern "C"
