// dense_tiles.h — matrix-core tiles of the policy network's products.
//
// A product is C[m][n] = sum over k of P(m, k) Q(n, k).  A workgroup makes a
// BM x BN tile of C in steps of KB bytes of k (128: 64 bfloat16 or 32 fp32; or
// half of that), which go from memory straight to LDS, some steps ahead of the
// products.
//
// A side lies in memory along k ("rows": p[m ld + k]) or along its own index
// ("columns": p[k ld + m]).  Either way it moves in 16-byte words, a wavefront
// 64 of them to consecutive places of LDS, so the place that a word gets is
// chosen by which word a lane asks for.  A word's place in its row is exchanged
// (xor) by the row, so that the lanes that LDS serves together are on different
// banks.  A side of columns is turned when it is read back: 16-bit
// elements by the transposing LDS read, 32-bit ones one at a time.
//
// Products are 32 x 32 tiles.  A lane l has index l % 32 of both sides and of
// the result the rows 8 (r / 4) + 4 (l / 32) + r % 4 of its column in register
// r.  Q is the first operand, so registers run along n, which is contiguous in
// every result, and a lane stores neighbours.
//
// The order of k inside a step differs between lanes' words and the sum's
// order, alike on both sides; sums are fp32, one chain a value.
#ifndef MDNAV_DENSE_TILES_H
#define MDNAV_DENSE_TILES_H

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace dense {

typedef __bf16 bf16;
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

template <class T> constexpr uint32_t per_word() { return 16 / sizeof(T); }

// What lanes past the end of k load.
__device__ __attribute__((aligned(16))) const uint32_t zero_word[4] = {0, 0, 0, 0};

// One side of a product, from one matrix or two of the same shape.
struct Side {
    const char *p, *p2;
    int64_t ld;      // bytes between rows (along k) or between k (columns)
    uint32_t count;  // m or n
};

// 64 words from each lane's address to LDS at `to` + 16 lane.  The compiler
// knows neither of the load nor of what it writes: whoever reads the words
// waits (landed()) and passes a barrier first.
__device__ __forceinline__ void to_lds(const char* from, uint32_t to) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(to), "v"(from) : "m0");
}
// The same from a base that all lanes share and a lane's offset, to `to` + `more`.
__device__ __forceinline__ void to_lds(const char* base, uint32_t off, uint32_t to, uint32_t more) {
    asm volatile("s_add_u32 m0, %0, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(to), "v"(off), "s"(base), "i"(more) : "m0", "scc");
}
// All but the last N loads have landed, all LDS reads are back; then every wavefront of the workgroup.
template <int N> __device__ __forceinline__ void landed() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"i"(N) : "memory");
}

template <class T> struct Frag;
template <> struct Frag<bf16> { bf16x8 t; };
template <> struct Frag<float> { f32x4 t; };

__device__ __forceinline__ void mma(f32x16& acc, const Frag<bf16>& a, const Frag<bf16>& b) {
    acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.t, b.t, acc, 0, 0, 0);
}
__device__ __forceinline__ void mma(f32x16& acc, const Frag<float>& a, const Frag<float>& b) {
#pragma unroll
    for (int i = 0; i < 4; i++) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(a.t[i], b.t[i], acc, 0, 0, 0);
}

__device__ __forceinline__ bf16x4 transposed4(uint32_t at) {
    typedef __attribute__((address_space(3))) s16x4 lds4;
    return __builtin_bit_cast(bf16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(uintptr_t)at));
}
template <class V> __device__ __forceinline__ V lds_at(uint32_t at) {
    typedef __attribute__((address_space(3))) const V lds;
    return *(lds*)(uintptr_t)at;
}

// A side's part of one stage: R rows of a step, R a multiple of 32.  W: wavefronts of the workgroup, T2: from two matrices
// (half of the rows from each, rows only).  A step has KB / 32 places of two words of k, one to each half of a wavefront.
template <class T, int R, int W, int KB, bool COLUMNS, bool T2> struct Staged;

template <class T, int R, int W, int KB, bool T2> struct Staged<T, R, W, KB, false, T2> {
    static constexpr int WORDS = KB / 16, LOADS = R * WORDS / (64 * W), BYTES = R * KB;
    static_assert(LOADS >= 1 && (!T2 || LOADS % 2 == 0), "");
    uint32_t off[LOADS];
    const char *p0, *p1;
    uint32_t word;  // of the step, this lane's

    // 256 / KB rows fill the 64 banks.
    static __device__ __forceinline__ uint32_t exchange(uint32_t row) { return row / (256 / KB) % WORDS; }
    // From row r0; rows past the last repeat it (their results are not stored).
    __device__ __forceinline__ void init(const Side& a, uint32_t r0, uint32_t wave, uint32_t lane) {
        p0 = a.p + int64_t(r0) * a.ld;
        p1 = a.p2 + int64_t(r0) * a.ld;
        static_assert(W % 2 == 0, "");
        constexpr uint32_t ROWS = 64 / WORDS;
        word = (lane % WORDS) ^ exchange(wave * ROWS + lane / WORDS);  // (the same in all loads: ROWS W rows change nothing)
#pragma unroll
        for (int i = 0; i < LOADS; i++) {
            const uint32_t row = (i * W + wave) * ROWS + lane / WORDS;
            const uint32_t in = T2 && i >= LOADS / 2 ? row - R / 2 : row, left = a.count - 1 - r0;
            off[i] = (in < left ? in : left) * uint32_t(a.ld) + 16 * word;
        }
    }
    // Load i of the step at k0.
    __device__ __forceinline__ void load(int i, uint32_t to, uint32_t k0, uint32_t wave, bool second) const {
        to_lds(((T2 ? i >= LOADS / 2 : second) ? p1 : p0) + uint64_t(k0) * sizeof(T), off[i], to + wave * 1024, i * W * 1024);
    }
    // The same of the last step of a sum, which does not fill it.
    __device__ __forceinline__ void load_end(int i, uint32_t to, uint32_t k0, uint32_t k_end, uint32_t wave, bool second) const {
        const char* from = ((T2 ? i >= LOADS / 2 : second) ? p1 : p0) + uint64_t(k0) * sizeof(T) + off[i];
        to_lds(k0 + word * per_word<T>() < k_end ? from : reinterpret_cast<const char*>(zero_word), to + (i * W + wave) * 1024);
    }
    // A lane's operands: of the 32 rows from `row`, its word of place kk of the step.
    struct Reader {
        uint32_t at[KB / 32];
        __device__ __forceinline__ void init(uint32_t lane) {
#pragma unroll
            for (uint32_t kk = 0; kk < KB / 32; kk++) at[kk] = (lane & 31) * KB + (((2 * kk + (lane >> 5)) ^ exchange(lane & 31)) << 4);
        }
        __device__ __forceinline__ Frag<T> get(uint32_t base, uint32_t row, int kk) const {
            return {lds_at<decltype(Frag<T>::t)>(base + at[kk] + row * KB)};
        }
    };
};

template <class T, int R, int W, int KB> struct Staged<T, R, W, KB, true, false> {
    static constexpr int WORDS = R * sizeof(T) / 16, KS = 64 / WORDS;
    static constexpr int LOADS = R * KB / (1024 * W), BYTES = R * KB;
    static_assert(LOADS >= 1 && WORDS <= 64, "");
    uint32_t off[LOADS];
    const char *p0, *p1;
    int64_t ld;
    uint32_t k_in;  // this lane's k in its first load; each further load is KS W later

    static __device__ __forceinline__ uint32_t exchange(uint32_t k) {
        if (sizeof(T) == 4) return ((k >> 2) & 1) << 3;
        return R >= 128 ? (k & 3) << 2 : ((k >> 1) & 1) << 2;
    }
    __device__ __forceinline__ void init(const Side& a, uint32_t r0, uint32_t wave, uint32_t lane) {
        p0 = a.p + int64_t(r0) * sizeof(T);
        p1 = a.p2 + int64_t(r0) * sizeof(T);
        ld = a.ld;
        k_in = wave * KS + lane / WORDS;
#pragma unroll
        for (int i = 0; i < LOADS; i++) {
            const uint32_t k = i * W * KS + k_in, word = (lane % WORDS) ^ exchange(k), last = (a.count - 1 - r0) / per_word<T>();
            off[i] = k * uint32_t(a.ld) + 16 * (word < last ? word : last);
        }
    }
    __device__ __forceinline__ void load(int i, uint32_t to, uint32_t k0, uint32_t wave, bool second) const {
        to_lds((second ? p1 : p0) + int64_t(k0) * ld, off[i], to + wave * 1024, i * W * 1024);
    }
    __device__ __forceinline__ void load_end(int i, uint32_t to, uint32_t k0, uint32_t k_end, uint32_t wave, bool second) const {
        const char* from = (second ? p1 : p0) + int64_t(k0) * ld + off[i];
        to_lds(k0 + i * W * KS + k_in < k_end ? from : reinterpret_cast<const char*>(zero_word), to + (i * W + wave) * 1024);
    }
    struct Reader {
        uint32_t lane;
        __device__ __forceinline__ void init(uint32_t l) { lane = l; }
        __device__ __forceinline__ Frag<T> get(uint32_t base, uint32_t row, int kk) const {
            if constexpr (sizeof(T) == 2) {
                const uint32_t j = lane & 15, word = (row / 8 + 2 * ((lane >> 4) & 1) + ((j & 3) >> 1)) ^ exchange(j >> 2);
                const uint32_t at = base + (8 * (lane >> 5) + (j >> 2)) * (2 * R) + word * 16 + (j & 1) * 8 + kk * 32 * R;
                const bf16x4 lo = transposed4(at), hi = transposed4(at + 8 * R);
                return {__builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7)};
            } else {
                const uint32_t h = lane >> 5, c = lane & 31, word = (row / 4 + c / 4) ^ (h << 3);
                const uint32_t at = base + h * (16 * R) + word * 16 + (c & 3) * 4 + kk * 32 * R;
                return {f32x4{lds_at<float>(at), lds_at<float>(at + 4 * R), lds_at<float>(at + 8 * R), lds_at<float>(at + 12 * R)}};
            }
        }
    };
};

}  // namespace dense

#endif
