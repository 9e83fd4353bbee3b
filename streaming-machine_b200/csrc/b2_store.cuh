// b2_store.cuh -- the key/value store held in 4 bits: its layout on the device, its arithmetic and the launches that
// write rows into it, read them back and run the arrival over it (b2_store.cu; the C ABI's b2_store_* and the engine's
// "store_bits" 4).
//
// Per (slot, layer, head) the positions are contiguous (stride ctx, a multiple of 32):
//   k  [pos][32 bytes]  64 codes, two per byte (the lower dimension in the low digits). The two halves' words lie in
//                       turn: word 2j is dims 8j .. 8j + 7, word 2j + 1 dims 32 + 8j .., so that one 8-byte load holds
//                       the same place of both halves
//   ks [pos][2]         the halves' shifts
//   v  [pos][32 bytes]  64 codes, word j is dims 8j .. 8j + 7
//   vs [pos]            the value's shift
// 67 bytes a position and head; the 16-bit store (struct KV) takes 396.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include "b2_epi.cuh"

namespace b2 {

struct Store4 {
    uint8_t* k;
    int8_t* ks;
    uint8_t* v;
    int8_t* vs;
    int L, H, ctx;     // ctx: the positions' stride
    int lim;           // positions a stream may hold
};

// a call's rows: stream i (slot slot0 + i) gives rows cu[i] .. cu[i + 1] - 1 (cu == nullptr: row i), its first at
// position pos[i]
struct StoreRows {
    const int32_t* cu = nullptr;
    const int32_t* pos = nullptr;
    int n_streams = 0, rows = 0, max_rows = 0;
    int slot0 = 0;
};

// int64 rows of heads: row r's head h at x + r * ld + h * hs
struct StoreVec {
    const int64_t* x;
    int64_t ld;
    int hs;
};

struct StoreAttend {
    Store4 st;
    StoreRows rw;
    int layer;
    StoreVec q;
    const int32_t* first;  // optional [n_streams]: the first position that a stream still sees
    int window;            // 0, or how many positions a row sees (its own the last)
    const int32_t* ARR;
    int alen;
    const int32_t* LOG2;
    const int32_t* EXP2;
    int64_t* out;          // [rows][H][64]
    uint64_t* or_out;      // store_step, optional [rows]: OR of |out| per row (the next bank's to16 shift)
    uint32_t* err;
    uint64_t* stamp = nullptr;   // b2_profile mode 2
    // store_step: the rows' own keys and values, held first (one row a stream); Pythia's turn of q and k before it, where
    // COS is given ([positions][8] at 2^-30)
    StoreVec k{nullptr, 0, 0}, v{nullptr, 0, 0};
    const int32_t *COS = nullptr, *SIN = nullptr;
    bool early = false;    // store_step: the row table and the positions before the rows' own were written two launches before or more
};

// what the launches are sized by, once per device (the current one) and arrival table; to be called before the first launch
constexpr int STORE_MAX_CLUSTER = 8;
struct StorePlan {
    int sms = 0;                               // the device's SM count
    int many[STORE_MAX_CLUSTER + 1] = {0};     // clusters of 1 .. 8 CTAs of the many-row arrival that fit at once (0: none)
};
cudaError_t store_init(int alen, StorePlan& plan);

// how the launches below are made: on `stream`, as programmatic dependent launches where pdl is set
struct StoreLaunch {
    cudaStream_t stream;
    bool pdl;
    const StorePlan* plan;
};

cudaError_t store_write(const Store4& st, const StoreRows& rw, int layer, const StoreVec& k, const StoreVec& v, uint32_t* err,
                        StoreLaunch how, uint64_t* stamp = nullptr);
cudaError_t store_read(const Store4& st, const StoreRows& rw, int layer, int64_t* k, int64_t* v, uint32_t* err, StoreLaunch how);
cudaError_t store_attend(const StoreAttend& a, StoreLaunch how);
cudaError_t store_step(const StoreAttend& a, StoreLaunch how);   // a.rw.max_rows = 1

constexpr int64_t STORE_TOP = 1ll << 47;          // magnitudes are held below this
constexpr int32_t STORE_LIM = (1 << 30) - 1;      // scores are held between -STORE_LIM and STORE_LIM
constexpr int STORE_MAX_SHIFT = 44;               // 2^47 in 4 bits
constexpr int STORE_MAX_CTX = 65536;              // 255 x 128 x 65,536 < 2^31: the tensor cores' sums stay in 32 bits
constexpr int32_t STORE_MAX_ARR = 1 << 24;        // the arrival table's largest entry (the converter's ARR[0])
constexpr int STORE_MAX_ALEN = 32768;             // its entries: a copy has to fit shared memory (the converter's has 17,745)
constexpr int STORE_W_SHIFT = 1;                  // a weight is the table's entry halved: its top byte stays below 129

// the store's arrays in one piece of memory: its size, and the pointers into it
inline size_t store_layout(Store4& st, int n_slots, int L, int H, int max_ctx, void* at) {
    st.L = L;
    st.H = H;
    st.lim = max_ctx;
    st.ctx = (max_ctx + 31) / 32 * 32;
    const size_t n = (size_t)n_slots * L * H * st.ctx;     // a multiple of 32: every array starts on 32 bytes
    st.k = (uint8_t*)at;
    st.v = st.k + n * 32;
    st.ks = (int8_t*)(st.v + n * 32);
    st.vs = st.ks + n * 2;
    return n * 67;
}

#ifdef __CUDACC__
// x 2^-s to nearest, halves up, s >= 0: with no carry past the word (base2.py:18-22 wherever that does not overflow)
B2_DEV int32_t rnd32(int32_t x, int s) { return s > 0 ? ((x >> (s - 1)) + 1) >> 1 : x; }
B2_DEV int64_t rnd64(int64_t x, int s) { return s > 0 ? ((x >> (s - 1)) + 1) >> 1 : x; }
B2_DEV uint32_t mag32(int32_t x) { return x < 0 ? 0u - (uint32_t)x : (uint32_t)x; }
B2_DEV int64_t store_clamp(int64_t x) { return x < -STORE_TOP ? -STORE_TOP : (x > STORE_TOP - 1 ? STORE_TOP - 1 : x); }
B2_DEV int store_code(int64_t x, int s) {
    const int64_t c = rnd64(x, s);
    return c < -8 ? -8 : (c > 7 ? 7 : (int)c);
}
// where the key codes of dims 2i, 2i + 1 lie in their 32 bytes (i = 0 .. 31), and back
B2_DEV int key_byte(int i) { return ((i & 12) << 1) | ((i & 16) >> 2) | (i & 3); }
B2_DEV int key_pair(int m) { return ((m & 4) << 2) | ((m & 24) >> 1) | (m & 3); }

// the score: dot 2^-r rounded (r = 28 - u - S), held between -STORE_LIM and STORE_LIM; |dot| <= 2^26
B2_DEV int32_t store_score(int32_t dot, int r) {
    if (r >= 0) return rnd32(dot, r);
    const int up = -r < 31 ? -r : 31;
    const int32_t lim = STORE_LIM >> up;
    if (dot > lim) return STORE_LIM;
    if (dot < -lim) return -STORE_LIM;
    return (int32_t)((uint32_t)dot << (up & 31));
}

// the rows of a stream by its entries of the row table; false: nothing to do (no rows, or an entry that does not fit the
// call, which is flagged)
struct StoreRun { int r0, n, p0; };
B2_DEV bool store_run(const StoreRows& w, int r0, int r1, int p0, int lim, StoreRun& run, uint32_t* err) {
    run.r0 = r0;
    run.n = 0;
    run.p0 = p0;
    if (r0 < 0 || r1 < r0 || r1 > w.rows || r1 - r0 > w.max_rows) {
        set_err(err, DERR_ROWS);
        return false;
    }
    if (r1 == r0) return false;
    if (p0 < 0 || p0 > lim - (r1 - r0)) {
        set_err(err, DERR_POS);
        return false;
    }
    run.n = r1 - r0;
    return true;
}
B2_DEV bool store_run(const StoreRows& w, int s, int lim, StoreRun& run, uint32_t* err) {
    return store_run(w, w.cu ? w.cu[s] : s, w.cu ? w.cu[s + 1] : s + 1, w.pos[s], lim, run, err);
}
#endif

}  // namespace b2
