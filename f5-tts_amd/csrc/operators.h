// operators.h — launchers of the operators with entry points of their own (rotary positions, sliding-window attention).  The argument
// structs are the ABI's (include/f5hip.h); the checks are in operators_api.cpp, the launchers take arguments that passed them.
#pragma once
#include "../../include/f5hip.h"
#include "common.h"

typedef __bf16 bf16;

// why the arguments are refused, or null
const char* check_rotary(const f5hip_rotary_args& a);
const char* check_window_attention(const f5hip_window_attention_args& a);

// frequencies (64 bits, R / 2 of them) scaled for longer contexts, in place; why they are refused, or null
const char* scale_rotary_frequencies(double* f, int rot_dim, int scaling, double factor, int64_t original_length, double low, double high, double* amplitude);

constexpr int64_t ROTARY_THREADS = 0x7fffff00;  // most of a sequence: the kernel numbers them in 32 bits
int64_t rotary_threads(const f5hip_rotary_args& a);  // of a sequence, of arguments that passed the other checks
hipError_t launch_rotary(const f5hip_rotary_args& a, hipStream_t s);
int64_t window_attention_workspace(const f5hip_window_attention_args& a);
hipError_t launch_window_attention(const f5hip_window_attention_args& a, hipStream_t s);
