// Division of indexes by sizes that the host knows before a launch.
#pragma once

// Division by a number known on the host, by multiplication (Granlund and Montgomery): exact for n < 2^31.
struct Divisor {
  int d;
  unsigned m, shift;
};
inline Divisor divisor(int d) {
  unsigned l = 0;
  while ((1ll << l) < d)
    l++;
  return Divisor{d, (unsigned)(((1ull << 32) * ((1ull << l) - (unsigned)d)) / (unsigned)d + 1), l};
}
// n / by, and n becomes the rest.
__host__ __device__ __forceinline__ int divide(int &n, const Divisor &by) {
#ifdef __CUDA_ARCH__
  const unsigned high = __umulhi((unsigned)n, by.m);
#else
  const unsigned high = (unsigned)(((unsigned long long)(unsigned)n * by.m) >> 32);
#endif
  const int q = (int)((high + (unsigned)n) >> by.shift);
  n -= q * by.d;
  return q;
}
