// Short reciprocals and quotients against the ones of CUDA: every float from 1 up to 2^118, and random quotients of 2^-100 <= a <= 1 and 1 <= x <= 2^20, a quarter each
// with ordinary mantissas, with divisors just below and just above a power of two, and with a and x a few places apart.  Prints the numbers of differences and of pairs.
#include <cstdint>
#include <cstdio>

#include "division.cuh"

__global__ void reciprocals(unsigned long long* bad) {
    const uint64_t first = 0x3f800000u, end = static_cast<uint64_t>(127 + 118) << 23;
    unsigned long long n = 0;
    for (uint64_t u = first + blockIdx.x * static_cast<uint64_t>(blockDim.x) + threadIdx.x; u < end; u += static_cast<uint64_t>(gridDim.x) * blockDim.x) {
        const float x = __uint_as_float(static_cast<uint32_t>(u));
        n += __float_as_uint(ep::reciprocal(x)) != __float_as_uint(__frcp_rn(x));
    }
    if (n != 0) atomicAdd(bad, n);
}

__global__ void quotients(unsigned long long* bad, int rounds) {
    uint64_t s = (blockIdx.x * static_cast<uint64_t>(blockDim.x) + threadIdx.x) * 0x9E3779B97F4A7C15ull + 12345;
    unsigned long long n = 0;
    for (int i = 0; i < rounds; ++i) {
        s = s * 6364136223846793005ull + 1442695040888963407ull;
        uint64_t h = (s ^ (s >> 29)) * 0xBF58476D1CE4E5B9ull;
        h ^= h >> 32;
        uint32_t a_bits = h & 0x7fffff, x_bits = (h >> 23) & 0x7fffff;
        if (i % 4 == 1) x_bits |= 0x7fff00;
        if (i % 4 == 2) x_bits &= 0xff;
        if (i % 4 == 3) a_bits = (x_bits + static_cast<uint32_t>(h & 7) - 4) & 0x7fffff;
        const uint32_t a_exponent = 27 + ((h >> 46) & 0x3ff) % 100, x_exponent = 127 + ((h >> 56) & 0xff) % 20;
        const float a = __uint_as_float(a_exponent << 23 | a_bits), x = __uint_as_float(x_exponent << 23 | x_bits);
        n += __float_as_uint(ep::quotient(a, x, ep::reciprocal(x))) != __float_as_uint(__fdiv_rn(a, x));
    }
    if (n != 0) atomicAdd(bad, n);
}

int main() {
    constexpr int kCtas = 592, kThreads = 256, kRounds = 40000;
    unsigned long long* device = nullptr;
    unsigned long long bad[2] = {1, 1};
    cudaError_t err = cudaMalloc(&device, sizeof(bad));
    if (err == cudaSuccess) err = cudaMemset(device, 0, sizeof(bad));
    if (err == cudaSuccess) {
        reciprocals<<<kCtas, kThreads>>>(device);
        quotients<<<kCtas, kThreads>>>(device + 1, kRounds);
        err = cudaMemcpy(bad, device, sizeof(bad), cudaMemcpyDeviceToHost);
    }
    std::printf("%s %llu %llu %lld\n", cudaGetErrorName(err), bad[0], bad[1], static_cast<long long>(kCtas) * kThreads * kRounds);
    return err != cudaSuccess;
}
