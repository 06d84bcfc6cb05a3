// devops.h — the operators on device tensors that stand outside the ggml graph: MXFP4 products
// and expert routing (k_mx4.hip, k_moe.hip, devops_capi.cpp).
//
// These sources need no ggml header: they are linked into the plugin beside the rest and, alone,
// into libmi355x-ops.so for hosts that only call the flat ABI.  Nothing here aborts: a launcher
// returns the HIP status of its launch and the C entry hands it on.
#pragma once

#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>
#include <tuple>
#include <type_traits>

namespace mi355x_ops {

// element types of the flat ABI (the ggml_type numbers)
enum elem_type { ELEM_F32 = 0, ELEM_F16 = 1, ELEM_BF16 = 30 };

constexpr int MX4_BLOCK = 32;    // elements that share one exponent
constexpr int MX4_PLANE = 256;   // elements whose eight exponents lie side by side
constexpr int MOE_MAX_EXPERTS = 1024;
constexpr int MOE_MAX_USED = 16;

// MXFP4 rows: codes [rows][K / 2], element 2 i in the low half of byte i; scales
// [ceil(K / 256)][rows][8].  Bytes of a scale plane that lie past K are never used.
struct mx4_mat {
    const uint8_t * codes;
    const uint8_t * scales;
    int64_t rows;
    int64_t K;
};

// the sorted pairs of a routing step: pairs [offsets[e], offsets[e + 1]) belong to expert e
struct moe_view {
    const int32_t * order;     // [pairs] pair (token * used + slot) at a sorted place, -1 behind offsets[n_expert]
    const int32_t * offsets;   // [n_expert + 1]
    int64_t pairs;
    int n_expert;
    int used;                  // slots per token; 0: the product's rows are in sorted order already
};

hipError_t mx4_quantize(int type, const void * x, int64_t ldx, int64_t rows, int64_t K, uint8_t * codes, uint8_t * scales,
                        hipStream_t st);
hipError_t mx4_dequantize(const mx4_mat & m, int type, void * y, hipStream_t st);
// y [T][M] = W . x, or by experts with a view: sorted row p of y [pairs][M] is expert e(p)'s W times x
// row order[p] / used (or p)
struct mx4_needs {
    bool quantized;   // x has to come as MXFP4; few rows of floats go to mx4_product_float
    int64_t part;     // bytes of workspace for sums, beside x's
};
mx4_needs mx4_product_needs(const mx4_mat & w, int64_t x_rows, const moe_view * v);
hipError_t mx4_product(const mx4_mat & w, const mx4_mat & x, const moe_view * v, int ytype, void * y, void * part, hipStream_t st);
hipError_t mx4_product_float(const mx4_mat & w, int xtype, const void * x, int64_t ldx, int64_t x_rows, const moe_view * v,
                             int ytype, void * y, hipStream_t st);

size_t moe_sort_workspace(int64_t pairs, int n_expert);
hipError_t moe_sort(const void * ids, int id_bytes, int64_t pairs, int n_expert, int32_t * order, int32_t * rank,
                    int32_t * offsets, void * work, hipStream_t st);
hipError_t moe_gather(int type, const void * x, int64_t ldx, int64_t T, int64_t D, int used, const int32_t * order,
                      const int32_t * rank, void * xs, hipStream_t st);
hipError_t moe_combine(int type, const void * ys, int64_t ldys, int64_t T, int64_t D, int used, const int32_t * rank,
                       const float * w, void * y, hipStream_t st);
hipError_t moe_combine_back(int type, const void * dy, int64_t lddy, const void * ys, int64_t ldys, int64_t T, int64_t D,
                            int used, const int32_t * order, const int32_t * rank, const float * w, void * dys, float * dw,
                            hipStream_t st);

// A launch counts its threads in 32 bits along each axis.  Groups of `waves` waves, which may be more
// than that, lie along x and z: group group_id() of row_groups(n, y, waves), some of them past n.
constexpr int64_t MAX_WAVES = ((int64_t) 1 << 32) / 64 - 1;
static inline dim3 row_groups(int64_t n, int64_t y, int waves = 4) {
    const int64_t z = (n + MAX_WAVES / waves - 1) / (MAX_WAVES / waves);
    return dim3((unsigned) ((n + z - 1) / z), (unsigned) y, (unsigned) z);
}

// A launch and its own status.  hipGetLastError would also name an earlier failure, of any HIP call that the
// thread made, and take it from whoever has yet to ask; it is asked only to clear what this launch left.
template <class... P, class... A>
static inline hipError_t launch(void (*kernel)(P...), dim3 grid, unsigned threads, size_t lds, hipStream_t st, A... args) {
    std::tuple<P...> values(args...);
    return std::apply(
        [&](auto &... v) {
            void * at[] = {(void *) &v...};
            const hipError_t e = hipLaunchKernel((const void *) kernel, grid, dim3(threads), at, lds, st);
            if (e != hipSuccess) (void) hipGetLastError();
            return e;
        },
        values);
}

// ---- device side -----------------------------------------------------------------------------
__device__ __forceinline__ int64_t group_id() { return (int64_t) blockIdx.z * gridDim.x + blockIdx.x; }

template <class T> __device__ __forceinline__ float to_f32(T v) { return (float) v; }
template <class T> __device__ __forceinline__ T from_f32(float v) { return (T) v; }   // to nearest, ties to even

// N elements.  16 bytes of them are moved by get and put as one access, at any address that the
// element allows: gfx950's memory instructions need no more, so rows may lie anywhere.
template <class T, int N> struct pack { T v[N]; };
typedef int words16 __attribute__((ext_vector_type(4), aligned(2)));

template <class T, int N> __device__ __forceinline__ pack<T, N> get(const T * p) {
    static_assert(sizeof(T) * N == 16);
    const words16 w = *(const words16 *) p;
    return __builtin_bit_cast(pack<T, N>, w);
}

// STREAM: past the caches' replacement order, for outputs larger than the Infinity Cache
constexpr int64_t STREAM_BYTES = (int64_t) 256 << 20;
template <bool STREAM, class T, int N> __device__ __forceinline__ void put(T * p, const pack<T, N> & v) {
    static_assert(sizeof(T) * N == 16);
    const words16 w = __builtin_bit_cast(words16, v);
    if constexpr (STREAM) __builtin_nontemporal_store(w, (words16 *) p);
    else *(words16 *) p = w;
}

// a type as a template argument out of a run-time number: f(T{}) with T = float, _Float16 or __bf16
template <class F> static inline hipError_t with_type(int type, F && f) {
    switch (type) {
        case ELEM_F32: return f(float{});
        case ELEM_F16: return f(_Float16{});
        case ELEM_BF16: return f(__bf16{});
        default: return hipErrorInvalidValue;
    }
}

}  // namespace mi355x_ops
