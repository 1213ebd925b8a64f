// Element types of the tree-round operators: conversion of bf16 / fp16 / fp32 values, and
// 16-byte vector loads of eight 2-byte values.
#pragma once

#include <cuda_fp16.h>

#include <type_traits>

#include "common.cuh"

namespace dspark {

template <typename T>
struct Elem;

template <>
struct Elem<bf16> {
  static constexpr uint32_t kExpMask = 0x7F80u;
  static __device__ __forceinline__ float to_f(bf16 v) { return __bfloat162float(v); }
  static __device__ __forceinline__ bf16 from_f(float v) { return __float2bfloat16_rn(v); }
  static __device__ __forceinline__ float2 unpack(uint32_t w) {
    return make_float2(bf16_lo(w), bf16_hi(w));
  }
  static __device__ __forceinline__ uint32_t pack(float a, float b) { return pack_bf16x2(a, b); }
};

template <>
struct Elem<__half> {
  static constexpr uint32_t kExpMask = 0x7C00u;
  static __device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
  static __device__ __forceinline__ __half from_f(float v) { return __float2half_rn(v); }
  static __device__ __forceinline__ float2 unpack(uint32_t w) {
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
  }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
};

template <>
struct Elem<float> {
  static __device__ __forceinline__ float to_f(float v) { return v; }
  static __device__ __forceinline__ float from_f(float v) { return v; }
  static __device__ __forceinline__ float2 unpack(uint32_t w) {  // one value to a word
    return make_float2(__uint_as_float(w), 0.f);
  }
};

}  // namespace dspark
