// Probe: what the fp32 multiply-adds of hv_gemm_fp8_kernel's block scales cost beside its matrix instructions (gfx950).
// A wave's block of the reduction: 32 v_mfma_f32_16x16x128_f8f6f4 from a zero accumulator (8 row tiles x 4 column tiles) and
// 128 v_fma_f32 that add their results to the sums with the block's factor.  Modes:
//   0 MFMA alone (accumulating in the instruction)       1 FMA alone
//   2 the kernel's order: row tile j's four MFMAs, then the sixteen FMAs of row tile j - 1, a fence
//   3 the same instructions interleaved: one MFMA, then four FMAs of row tile j - 1, a fence
// One workgroup of W waves per CU, W = 4 (one wave per SIMD) and 8 (two, as the 256 x 256 tile has); prints shader cycles per
// block of the reduction per SIMD (s_memtime of wave 0, mean over the workgroups) and per MFMA.
//   hipcc --offload-arch=gfx950 -O3 -std=c++17 -Xclang -target-feature -Xclang -packed-fp32-ops tools/probes/fp8_scale_fma.hip -o tools/bin/fp8_scale_fma
#include <hip/hip_runtime.h>
#include <cstdio>
#include <vector>
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));

template <int MODE>
__global__ __launch_bounds__(512, 2) void probe(float* out, unsigned long long* cycles, int iters) {
    i32x8 w[4], x[2];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j][i] = 0x38383838 + (int)(threadIdx.x & 3) * 0x01010101 + j;
        x[0][i] = x[1][i] = 0x30303030 + (int)(threadIdx.x & 7) * 0x01010101;
    }
    f32x4 acc[8][4], part[2][4];
    const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[j][i] = zero;
#pragma unroll
    for (int i = 0; i < 4; ++i) part[0][i] = part[1][i] = f32x4{1.f, 2.f, 3.f, (float)threadIdx.x};
    const float f = 1e-3f * (float)(threadIdx.x & 15);
    __syncthreads();
    const unsigned long long t0 = __builtin_amdgcn_s_memtime();
    for (int it = 0; it < iters; ++it) {
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int now = j & 1, old = now ^ 1, at = (j + 7) & 7;
            asm volatile("" : "+v"(x[now][0]));  // (no instruction: equal products are not merged)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (MODE == 0) acc[j][i] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w[i], x[now], acc[j][i], 0, 0, 0, 0, 0, 0);
                if (MODE >= 2) part[now][i] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w[i], x[now], zero, 0, 0, 0, 0, 0, 0);
                if (MODE == 1 || MODE == 3) {
#pragma unroll
                    for (int r = 0; r < 4; ++r) acc[at][i][r] = __builtin_fmaf(part[old][i][r], f, acc[at][i][r]);
                }
                if (MODE == 3) __builtin_amdgcn_sched_barrier(0);
            }
            if (MODE == 2) {
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int r = 0; r < 4; ++r) acc[at][i][r] = __builtin_fmaf(part[old][i][r], f, acc[at][i][r]);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    const unsigned long long t1 = __builtin_amdgcn_s_memtime();
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) s += acc[j][i][0] + acc[j][i][1] + acc[j][i][2] + acc[j][i][3];
    out[blockIdx.x * blockDim.x + threadIdx.x] = s;
    if (threadIdx.x == 0) cycles[blockIdx.x] = t1 - t0;
}

template <int MODE>
static void run(const char* name, int waves) {
    const int blocks = 256, threads = waves * 64, iters = 4000;
    float* out;
    unsigned long long* cycles;
    if (hipMalloc(&out, sizeof(float) * blocks * threads) != hipSuccess || hipMalloc(&cycles, sizeof(*cycles) * blocks) != hipSuccess) exit(1);
    hipEvent_t e0, e1;
    (void)hipEventCreate(&e0), (void)hipEventCreate(&e1);
    probe<MODE><<<blocks, threads>>>(out, cycles, 100);
    (void)hipEventRecord(e0);
    probe<MODE><<<blocks, threads>>>(out, cycles, iters);
    (void)hipEventRecord(e1);
    if (hipDeviceSynchronize() != hipSuccess) exit(2);
    float ms;
    (void)hipEventElapsedTime(&ms, e0, e1);
    std::vector<unsigned long long> h(blocks);
    if (hipMemcpy(h.data(), cycles, sizeof(h[0]) * blocks, hipMemcpyDeviceToHost) != hipSuccess) exit(3);
    double mean = 0;
    for (auto c : h) mean += (double)c / blocks;
    const int per_simd = waves / 4;  // waves that share a SIMD
    printf("%-46s %d waves/CU: %7.1f s_memtime ticks and %7.1f ns per block of the reduction per SIMD wave, %5.1f ns per MFMA\n", name, waves,
           mean / iters / per_simd, ms * 1e6 / iters / per_simd, ms * 1e6 / iters / per_simd / 32);
    (void)hipFree(out), (void)hipFree(cycles);
}

int main() {
    for (int waves : {4, 8}) {
        run<0>("32 MFMA alone", waves);
        run<1>("128 FMA alone", waves);
        run<2>("4 MFMA, then 16 FMA of the row tile before", waves);
        run<3>("1 MFMA, then 4 FMA of the row tile before", waves);
    }
    return 0;
}
