//! Mirror of include/llmini_b200_fp4.h: the 4-bit operators beside the requantised weights.  Same names, same field order; a
//! test reads both files.  The reference has no counterpart as a call (its forward GEMMs are kernels of the model crate).
use std::ffi::c_void;

pub type CUstream = *mut c_void;

pub const B2_TYPE_F32: u32 = 0;
pub const B2_TYPE_BF16: u32 = 1;
pub const B2_TYPE_F16: u32 = 2;
pub const B2_NVFP4_MAXIMA: usize = 1024;

#[repr(C)]
#[derive(Clone, Copy)]
pub struct b2_matrix {
    pub data: *mut c_void,
    pub ld: u64,
    pub rows: u32,
    pub cols: u32,
    pub r#type: u32,
    pub reserved: u32,
}

#[repr(C)]
#[derive(Clone, Copy)]
pub struct b2_nvfp4_operand {
    pub bytes: *mut u8,
    pub scales: *mut u8,
    pub scale: *mut f32,
    pub row_bytes: u64,
    pub rows: u32,
    pub cols: u32,
    pub scale_count: u32,
    pub reserved: u32,
}

#[repr(C)]
#[derive(Clone, Copy)]
pub struct b2_nvfp4_linear_gradients {
    pub grad: b2_matrix,
    pub x: b2_matrix,
    pub weight_t: b2_nvfp4_operand,
    pub grad_x: b2_matrix,
    pub grad_weight: b2_matrix,
    pub grad_rows: b2_nvfp4_operand,
    pub grad_columns: b2_nvfp4_operand,
    pub x_columns: b2_nvfp4_operand,
    pub d_maxima: *mut f32,
    pub accumulate: u32,
    pub reserved: u32,
}

#[repr(C)]
#[derive(Clone, Copy)]
pub struct b2_nvfp4_cache {
    pub bytes: *mut u8,
    pub scales: *mut u8,
    pub exponents: *mut u8,
    pub pages: u32,
    pub page_size: u32,
    pub heads: u32,
    pub dim: u32,
}

#[repr(C)]
#[derive(Clone, Copy)]
pub struct b2_vectors {
    pub data: *mut c_void,
    pub sequence_stride: u64,
    pub token_stride: u64,
    pub head_stride: u64,
    pub r#type: u32,
    pub reserved: u32,
}

extern "C" {
    pub fn b2_nvfp4_quantize_rows(x: *const b2_matrix, out: *const b2_nvfp4_operand, stream: CUstream) -> i32;
    pub fn b2_nvfp4_quantize_columns(x: *const b2_matrix, out: *const b2_nvfp4_operand, d_maxima: *mut f32, stream: CUstream) -> i32;
    pub fn b2_nvfp4_decode(r#in: *const b2_nvfp4_operand, scale_layout: u32, out: *const b2_matrix, stream: CUstream) -> i32;
    pub fn b2_nvfp4_matmul(a: *const b2_nvfp4_operand, b: *const b2_nvfp4_operand, c: *const b2_matrix, d_bias: *const f32, accumulate: u32, stream: CUstream) -> i32;
    pub fn b2_nvfp4_linear_forward(x: *const b2_matrix, weight: *const b2_nvfp4_operand, y: *const b2_matrix, d_bias: *const f32, scratch: *const b2_nvfp4_operand, stream: CUstream) -> i32;
    pub fn b2_nvfp4_linear_backward(args: *const b2_nvfp4_linear_gradients, stream: CUstream) -> i32;
    pub fn b2_nvfp4_status(stream: CUstream) -> i32;
    pub fn b2_nvfp4_cache_write(caches: *const b2_nvfp4_cache, tokens: *const b2_vectors, count: u32, d_slots: *const i64, token_count: u32, stream: CUstream) -> i32;
    pub fn b2_nvfp4_cache_read(caches: *const b2_nvfp4_cache, out: *const b2_vectors, count: u32, d_table: *const i32, table_width: u32, d_lengths: *const i32, sequences: u32, max_tokens: u32, stream: CUstream) -> i32;
}
