// TEST INFRASTRUCTURE: the six functions psk_oracle.c takes from the reference's C library, for a machine that has
// neither the reference's sources nor the library built from them: psk_libm.cuh compiled for the host (the same
// algorithms; tests/test_libm_host.py compares the bits where the reference is there). See oracle/Makefile.
#include "../presk_b200/csrc/psk_libm.cuh"

extern "C" {
float presk_expf(float x) { return psk::lm_expf(x); }
float presk_logf(float x) { return psk::lm_logf(x); }
float presk_tanhf(float x) { return psk::lm_tanhf(x); }
float presk_erff(float x) { return psk::lm_erff(x); }
float presk_sinf(float x) { int declined = 0; return psk::lm_sinf(x, &declined); }
float presk_cosf(float x) { int declined = 0; return psk::lm_cosf(x, &declined); }
}
