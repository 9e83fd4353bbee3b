// b2_store.cu -- the key/value store held in 4 bits: the kernels that write rows into it, read them back and run the
// arrival over it, and the C ABI's b2_store_* (include/base2.h has the formulas).
#include <stdarg.h>
#include <stdio.h>
#include <string.h>

#include <exception>
#include <new>
#include <string>
#include <vector>

#include "../../include/base2.h"
#include "b2_store.cuh"

namespace b2 {

// ---------------------------------------------------------------------------------------------------------------------
// write: a warp holds one head row (64 int64, two a lane). The shift is the bit length of the largest magnitude less 3:
// a warp maximum of bit lengths, over each half of 32 dims for keys, over all 64 for values.
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

__global__ void __launch_bounds__(SW_WARPS * 32) k_store_write(Store4 st, StoreRows rw, int layer, const int64_t* __restrict__ K,
                                                               int64_t ldk, const int64_t* __restrict__ V, int64_t ldv,
                                                               int wide, uint32_t* err) {
    griddep_wait();
    griddep_launch();
    const int s = blockIdx.y, lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
    StoreRun run;
    if (!store_run(rw, s, st.lim, run, err)) return;
    const int item = blockIdx.x * SW_WARPS + wid;            // (row of the stream, key or value, head)
    const int i = item / (2 * st.H), part = item - i * 2 * st.H, h = part < st.H ? part : part - st.H;
    if (i >= run.n) return;
    const bool key = part < st.H;
    const int64_t* x = key ? K + (size_t)(run.r0 + i) * ldk : V + (size_t)(run.r0 + i) * ldv;
    int64_t a, b;
    load_pair(x + h * 64 + 2 * lane, wide, a, b);
    a = store_clamp(a);
    b = store_clamp(b);
    const uint32_t t = (uint32_t)bitlen_u(mag(a) > mag(b) ? mag(a) : mag(b));
    const int whole = max((int)__reduce_max_sync(0xffffffffu, t) - 3, 0);
    int sh = min(whole, STORE_MAX_SHIFT);
    if (key) {                                               // lanes 0 .. 15 hold dims 0 .. 31
        const uint32_t half = __reduce_max_sync(lane < 16 ? 0xffffu : 0xffff0000u, t);
        sh = max(min(max((int)half - 3, 0), STORE_MAX_SHIFT), sh - 3);
    }
    const uint8_t c = (uint8_t)((store_code(a, sh) & 15) | (store_code(b, sh) << 4));
    const size_t e = kv_index(s, layer, h, run.p0 + i, st.L, st.H, st.ctx);
    if (key) {
        st.k[e * 32 + key_byte(lane)] = c;
        if ((lane & 15) == 0) st.ks[e * 2 + (lane >> 4)] = (int8_t)sh;
    } else {
        st.v[e * 32 + lane] = c;
        if (lane == 0) st.vs[e] = (int8_t)sh;
    }
}

// read: the values that the codes stand for, c 2^s; a warp a head row, as above
__global__ void __launch_bounds__(SW_WARPS * 32) k_store_read(Store4 st, StoreRows rw, int layer, int64_t* __restrict__ K,
                                                              int64_t* __restrict__ V, int wide, uint32_t* err) {
    griddep_wait();
    griddep_launch();
    const int s = blockIdx.y, lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
    StoreRun run;
    if (!store_run(rw, s, st.lim, run, err)) return;
    const int item = blockIdx.x * SW_WARPS + wid;
    const int i = item / (2 * st.H), part = item - i * 2 * st.H, h = part < st.H ? part : part - st.H;
    if (i >= run.n) return;
    const bool key = part < st.H;
    int64_t* out = key ? K : V;
    if (!out) return;
    const size_t e = kv_index(s, layer, h, run.p0 + i, st.L, st.H, st.ctx);
    const int c = key ? (int)(int8_t)st.k[e * 32 + key_byte(lane)] : (int)(int8_t)st.v[e * 32 + lane];
    const int sh = key ? st.ks[e * 2 + (lane >> 4)] : st.vs[e];
    const int lo = (int)((uint32_t)c << 28) >> 28, hi = c >> 4;
    const int64_t a = (int64_t)((uint64_t)(int64_t)lo << sh), b = (int64_t)((uint64_t)(int64_t)hi << sh);
    int64_t* o = out + ((size_t)(run.r0 + i) * st.H + h) * 64 + 2 * lane;
    if (wide) {
        *reinterpret_cast<longlong2*>(o) = make_longlong2(a, b);
    } else {
        o[0] = a;
        o[1] = b;
    }
}

// ---------------------------------------------------------------------------------------------------------------------
// the arrival, one CTA of 8 warps per (row, head): a warp takes a key at a time, two dims a lane.
//   pass 1  every visible key's score: the largest; the largest value shift
//   pass 2  the scores again, a = ARR[start - score], Z = sum a, num = sum rnd(a, 1 + M - vs) c
// ---------------------------------------------------------------------------------------------------------------------
constexpr int SA_WARPS = 8;

B2_DEV int32_t key_dot(const Store4& st, size_t e, int lane, int q0, int q1, int& S) {
    const int c = (int)(int8_t)st.k[e * 32 + key_byte(lane)];
    const int lo = (int)((uint32_t)c << 28) >> 28, hi = c >> 4;
    const int s0 = st.ks[e * 2], s1 = st.ks[e * 2 + 1];
    S = max(s0, s1);
    const int up = (lane < 16 ? s0 : s1) - S + 3;
    return __reduce_add_sync(0xffffffffu, (lo * q0 + hi * q1) << up);
}

__global__ void __launch_bounds__(SA_WARPS * 32) k_store_attend(StoreAttend a) {
    griddep_wait();
    griddep_launch();
    const int i = blockIdx.x, h = blockIdx.y, s = blockIdx.z;
    const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
    __shared__ int64_t s_num[SA_WARPS][64], s_z[SA_WARPS];
    __shared__ int32_t s_max[SA_WARPS], s_shift[SA_WARPS];
    StoreRun run;
    if (!store_run(a.rw, s, a.st.lim, run, a.err) || i >= run.n) return;
    const int H = a.st.H, row = run.r0 + i, p = run.p0 + i;
    int lo = a.window > 0 ? max(0, p - a.window + 1) : 0;
    if (a.first) lo = max(lo, a.first[s]);
    int64_t* out = a.out + ((size_t)row * H + h) * 64;
    if (lo > p) {
        if (threadIdx.x < 64) out[threadIdx.x] = 0;
        return;
    }
    const int64_t* q = a.q + (size_t)row * a.ldq + h * 64 + 2 * lane;
    const int64_t x0 = store_clamp(q[0]), x1 = store_clamp(q[1]);
    const uint64_t m0 = mag(x0), m1 = mag(x1);
    const int u = max((int)__reduce_max_sync(0xffffffffu, (uint32_t)bitlen_u(m0 > m1 ? m0 : m1)) - 14, 0);
    const int q0 = (int)rnd64(x0, u), q1 = (int)rnd64(x1, u);
    const size_t base = kv_index(s, a.layer, h, 0, a.st.L, H, a.st.ctx);
    int32_t start = -STORE_LIM - 1;
    int M = 0, S;
    for (int j = lo + wid; j <= p; j += SA_WARPS) {
        const int32_t dot = key_dot(a.st, base + j, lane, q0, q1, S);
        start = max(start, store_score(dot, 28 - u - S));
        M = max(M, (int)a.st.vs[base + j]);
    }
    if (lane == 0) { s_max[wid] = start; s_shift[wid] = M; }
    __syncthreads();
    for (int k = 0; k < SA_WARPS; k++) {
        start = max(start, s_max[k]);
        M = max(M, s_shift[k]);
    }
    int64_t n0 = 0, n1 = 0, z = 0;
    for (int j = lo + wid; j <= p; j += SA_WARPS) {
        const int32_t dot = key_dot(a.st, base + j, lane, q0, q1, S);
        const int32_t d = start - store_score(dot, 28 - u - S);
        if (d >= a.alen) continue;
        const int32_t w = __ldg(a.ARR + d);
        z += w;
        const int64_t wr = rnd32(w, min(STORE_W_SHIFT + M - a.st.vs[base + j], 26));
        const int c = (int)(int8_t)a.st.v[(base + j) * 32 + lane];
        n0 += wr * ((int)((uint32_t)c << 28) >> 28);
        n1 += wr * (c >> 4);
    }
    s_num[wid][2 * lane] = n0;
    s_num[wid][2 * lane + 1] = n1;
    if (lane == 0) s_z[wid] = z;
    __syncthreads();
    if (wid) return;
    n0 = n1 = z = 0;
    for (int k = 0; k < SA_WARPS; k++) {
        n0 += s_num[k][2 * lane];
        n1 += s_num[k][2 * lane + 1];
        z += s_z[k];
    }
    const int64_t F = 65536ll * (M + STORE_W_SHIFT) - log2fix(z, a.LOG2);
    const int64_t y0 = power(n0, F, a.EXP2), y1 = power(n1, F, a.EXP2);
    out[2 * lane] = y0;
    out[2 * lane + 1] = y1;
    if (a.or_out) {
        const uint64_t o = warp_or64(mag(y0) | mag(y1));
        if (lane == 0) atomicOr((unsigned long long*)&a.or_out[row], (unsigned long long)o);
    }
}

// ---- launches -------------------------------------------------------------------------------------------------------
namespace {
template <typename... KArgs, typename... Args>
cudaError_t store_launch(StoreLaunch how, void (*kernel)(KArgs...), dim3 grid, int threads, size_t smem, Args... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = how.stream;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = how.pdl ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kernel, ((KArgs)args)...);
}
bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }
}  // namespace

cudaError_t store_write(const Store4& st, const StoreRows& rw, int layer, const int64_t* k, int64_t ldk, const int64_t* v,
                        int64_t ldv, uint32_t* err, StoreLaunch how) {
    if (rw.n_streams == 0 || rw.rows == 0) return cudaSuccess;
    const int wide = aligned16(k) && aligned16(v) && ldk % 2 == 0 && ldv % 2 == 0;
    const dim3 grid((unsigned)(((int64_t)rw.max_rows * 2 * st.H + SW_WARPS - 1) / SW_WARPS), rw.n_streams);
    return store_launch(how, k_store_write, grid, SW_WARPS * 32, 0, st, rw, layer, k, ldk, v, ldv, wide, err);
}

cudaError_t store_read(const Store4& st, const StoreRows& rw, int layer, int64_t* k, int64_t* v, uint32_t* err, StoreLaunch how) {
    if (rw.n_streams == 0 || rw.rows == 0) return cudaSuccess;
    const int wide = aligned16(k) && aligned16(v);
    const dim3 grid((unsigned)(((int64_t)rw.max_rows * 2 * st.H + SW_WARPS - 1) / SW_WARPS), rw.n_streams);
    return store_launch(how, k_store_read, grid, SW_WARPS * 32, 0, st, rw, layer, k, v, wide, err);
}

cudaError_t store_attend(const StoreAttend& a, StoreLaunch how) {
    if (a.rw.n_streams == 0 || a.rw.rows == 0) return cudaSuccess;
    const dim3 grid(a.rw.max_rows, a.st.H, a.rw.n_streams);
    return store_launch(how, k_store_attend, grid, SA_WARPS * 32, 0, a);
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
    uint32_t* d_err = nullptr;
    std::vector<void*> allocs;
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
        if (e_ != cudaSuccess) return sfail(h, B2_ERR_CUDA, "%s: %s", #call, cudaGetErrorString(e_)); \
    } while (0)

template <class T>
int salloc(b2_store* h, T** p, size_t n) {
    void* q = nullptr;
    const cudaError_t e = cudaMalloc(&q, n * sizeof(T));
    if (e != cudaSuccess) {
        cudaGetLastError();      // an allocation that failed leaves nothing behind for the next call's check
        return sfail(h, B2_ERR_NOMEM, "cudaMalloc(%zu bytes): %s", n * sizeof(T), cudaGetErrorString(e));
    }
    h->allocs.push_back(q);
    *p = (T*)q;
    return B2_OK;
}

int upload32(b2_store* h, int32_t** dst, const int64_t* src, int64_t n, int64_t lo, int64_t hi, const char* name) {
    std::vector<int32_t> t((size_t)n);
    for (int64_t i = 0; i < n; i++) {
        if (src[i] < lo || src[i] > hi)
            return sfail(h, B2_ERR_VALUE, "b2_store_create: %s[%lld] = %lld outside [%lld, %lld]", name, (long long)i,
                         (long long)src[i], (long long)lo, (long long)hi);
        t[(size_t)i] = (int32_t)src[i];
    }
    const int rc = salloc(h, dst, (size_t)n);
    if (rc) return rc;
    SCK(cudaMemcpy(*dst, t.data(), sizeof(int32_t) * n, cudaMemcpyHostToDevice));
    return B2_OK;
}

void store_release(b2_store* h) {
    for (void* p : h->allocs) cudaFree(p);
    h->allocs.clear();
}

int store_build(b2_store* h, const int64_t* arrival, int64_t n_arrival, const int64_t* log2, const int64_t* exp2) {
    const b2_store_config& c = h->cfg;
    int rc;
    if (arrival[0] < 1) return sfail(h, B2_ERR_VALUE, "b2_store_create: arrival[0] = %lld (at least 1)", (long long)arrival[0]);
    if ((rc = upload32(h, &h->ARR, arrival, n_arrival, 0, STORE_MAX_ARR, "arrival")) ||
        (rc = upload32(h, &h->LOG2, log2, 65536, 0, 65536, "log2")) ||
        (rc = upload32(h, &h->EXP2, exp2, 65536, 65536, 131072, "exp2")))
        return rc;
    h->alen = (int)n_arrival;
    if ((rc = store_alloc(h->st, c.n_slots, c.n_layer, c.n_head, c.max_ctx, [&](void** p, size_t n) {
             uint8_t* q = nullptr;
             const int r = salloc(h, &q, n);
             *p = q;
             return r;
         })))
        return rc;
    if ((rc = salloc(h, &h->d_err, 4))) return rc;
    SCK(cudaMemset(h->d_err, 0, 4 * sizeof(uint32_t)));
    SCK(cudaDeviceSynchronize());
    return B2_OK;
}

// the arguments that every call on rows has
int check_rows(b2_store* h, const char* what, int32_t layer, const int32_t* cu, const int32_t* pos, int32_t n_streams,
               int32_t rows, int32_t max_rows) {
    const b2_store_config& c = h->cfg;
    if (layer < 0 || layer >= c.n_layer) return sfail(h, B2_ERR_ARG, "%s: layer %d of %d", what, layer, c.n_layer);
    if (n_streams < 0 || n_streams > c.n_slots) return sfail(h, B2_ERR_ARG, "%s: n_streams %d of %d slots", what, n_streams, c.n_slots);
    if (rows < 0 || max_rows < 0 || max_rows > c.max_ctx)
        return sfail(h, B2_ERR_ARG, "%s: rows %d, max_rows %d (context %d)", what, rows, max_rows, c.max_ctx);
    if (!cu && (rows != n_streams || max_rows != (rows ? 1 : max_rows)))
        return sfail(h, B2_ERR_ARG, "%s: without cu every stream gives one row (rows %d, n_streams %d, max_rows %d)", what, rows,
                     n_streams, max_rows);
    if (rows && (!pos || !n_streams || !max_rows))
        return sfail(h, B2_ERR_ARG, "%s: %d rows of %d streams, max_rows %d, pos %p", what, rows, n_streams, max_rows, (const void*)pos);
    return B2_OK;
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

int b2_store_create(const b2_store_config* cfg, int device, const int64_t* arrival, int64_t n_arrival, const int64_t* log2,
                    const int64_t* exp2, b2_store** out) {
    if (!out) return B2_ERR_ARG;
    *out = nullptr;
    if (!cfg || !arrival || !log2 || !exp2 || n_arrival < 1 || n_arrival > (1 << 20)) return B2_ERR_ARG;
    if (cfg->n_slots < 1 || cfg->n_slots > 65535 || cfg->n_layer < 1 || cfg->n_layer > 1024 || cfg->n_head < 1 ||
        cfg->n_head > 1024 || cfg->max_ctx < 1 || cfg->max_ctx > STORE_MAX_CTX)
        return B2_ERR_ARG;
    OnDevice on(device);
    if (on.e != cudaSuccess) return B2_ERR_CUDA;
    b2_store* h = new (std::nothrow) b2_store();
    if (!h) return B2_ERR_NOMEM;
    const int rc = guarded(h, [&] {
        h->cfg = *cfg;
        h->device = device;
        return store_build(h, arrival, n_arrival, log2, exp2);
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
        SCK(store_write(h->st, StoreRows{cu, pos, n_streams, rows, max_rows}, layer, k, ldk, v, ldv, h->d_err,
                        StoreLaunch{(cudaStream_t)stream, false}));
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
        SCK(store_read(h->st, StoreRows{cu, pos, n_streams, rows, max_rows}, layer, k, v, h->d_err,
                       StoreLaunch{(cudaStream_t)stream, false}));
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
        StoreAttend a{h->st, StoreRows{cu, pos, n_streams, rows, max_rows}, layer, q, ldq, first, window, h->ARR, h->alen,
                      h->LOG2, h->EXP2, out, nullptr, h->d_err};
        SCK(store_attend(a, StoreLaunch{(cudaStream_t)stream, false}));
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
