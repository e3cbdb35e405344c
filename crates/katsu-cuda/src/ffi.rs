// GENERATED by gen_ffi.py from include/katsu_cuda.h -- do not edit by hand.
// Not compiled in the repository that carries the kernels: its build image has no Rust toolchain.
#![allow(dead_code)]
use std::os::raw::{c_char, c_void};

/// Opaque katsu_cuda_ctx: one device, one stream.
#[repr(C)]
pub struct Ctx {
    _private: [u8; 0],
}
/// Opaque katsu_cuda_event.
#[repr(C)]
pub struct Event {
    _private: [u8; 0],
}

pub const KATSU_OK: i32 = 0;
pub const KATSU_ERR_INVALID_ARG: i32 = 1;
pub const KATSU_ERR_ALLOC: i32 = 2;
pub const KATSU_ERR_CUDA: i32 = 3;
pub const KATSU_ERR_NCCL: i32 = 4;
pub const KATSU_ERR_TIMEOUT: i32 = 5;
pub const KATSU_ERR_NO_DEVICE: i32 = 6;
pub const KATSU_ERR_UNSUPPORTED: i32 = 7;
pub const KATSU_MODE_3XTF32: i32 = 0;
pub const KATSU_MODE_TF32: i32 = 1;
pub const KATSU_MODE_FP32: i32 = 2;
pub const KATSU_NORM_RMS: i32 = 0;
pub const KATSU_NORM_LAYER: i32 = 1;
pub const KATSU_BLOCK_DX: i32 = 1;
pub const KATSU_BLOCK_DH: i32 = 2;
pub const KATSU_BLOCK_DGATE: i32 = 4;
pub const KATSU_BLOCK_DPOST_W: i32 = 8;
pub const KATSU_BLOCK_DPOST_B: i32 = 16;
pub const KATSU_BLOCK_DPRE_W: i32 = 32;
pub const KATSU_BLOCK_DPRE_B: i32 = 64;
pub const KATSU_INT8_MAX_K: i32 = 133144;
pub const KATSU_DISTILL_MAX_TOP: i32 = 1024;
pub const KATSU_LOGITS_MAX_BIASES: i32 = 1024;
pub const KATSU_COMM_ID_BYTES: usize = 128;
pub const KATSU_SUM_STATIC_MAX_COUNT: usize = 1 << 30;

extern "C" {
    pub fn katsu_cuda_device_count(out_count: *mut i32) -> i32;
    pub fn katsu_cuda_init(device: i32, out_ctx: *mut *mut Ctx) -> i32;
    pub fn katsu_cuda_shutdown(ctx: *mut Ctx) -> i32;
    pub fn katsu_cuda_set_precision(ctx: *mut Ctx, mode: i32) -> i32;
    pub fn katsu_cuda_get_precision(ctx: *mut Ctx, out_mode: *mut i32) -> i32;
    pub fn katsu_cuda_last_error_string() -> *const c_char;
    pub fn katsu_cuda_launch_count(ctx: *mut Ctx, out_count: *mut u64) -> i32;
    pub fn katsu_cuda_stream(ctx: *mut Ctx, out_stream: *mut *mut c_void) -> i32;
    pub fn katsu_cuda_alloc(ctx: *mut Ctx, count: usize, out_ptr: *mut *mut f32) -> i32;
    pub fn katsu_cuda_alloc_uninit(ctx: *mut Ctx, count: usize, out_ptr: *mut *mut f32) -> i32;
    pub fn katsu_cuda_free(ctx: *mut Ctx, ptr: *mut f32) -> i32;
    pub fn katsu_cuda_zero(ctx: *mut Ctx, dst: *mut f32, count: usize) -> i32;
    pub fn katsu_cuda_fill(ctx: *mut Ctx, dst: *mut f32, value: f32, count: usize) -> i32;
    pub fn katsu_cuda_h2d(ctx: *mut Ctx, dst_device: *mut f32, src_host: *const f32, count: usize) -> i32;
    pub fn katsu_cuda_d2h(ctx: *mut Ctx, dst_host: *mut f32, src_device: *const f32, count: usize) -> i32;
    pub fn katsu_cuda_d2h_async(ctx: *mut Ctx, dst_host: *mut f32, src_device: *const f32, count: usize) -> i32;
    pub fn katsu_cuda_d2d(ctx: *mut Ctx, dst_device: *mut f32, src_device: *const f32, count: usize) -> i32;
    pub fn katsu_cuda_host_alloc(ctx: *mut Ctx, count: usize, out_ptr: *mut *mut f32) -> i32;
    pub fn katsu_cuda_host_free(ctx: *mut Ctx, ptr: *mut f32) -> i32;
    pub fn katsu_cuda_sync(ctx: *mut Ctx) -> i32;
    pub fn katsu_cuda_conv2d_fwd(ctx: *mut Ctx, x: *const f32, w: *const f32, y: *mut f32, n: usize, c: usize, h: usize, wd: usize, k: usize, r: usize, s: usize, stride: usize, pad: usize) -> i32;
    pub fn katsu_cuda_conv2d_bwd(ctx: *mut Ctx, x: *const f32, w: *const f32, g: *const f32, dx: *mut f32, dw: *mut f32, n: usize, c: usize, h: usize, wd: usize, k: usize, r: usize, s: usize, stride: usize, pad: usize, accumulate: i32) -> i32;
    pub fn katsu_cuda_conv2d_bwd_scaled(ctx: *mut Ctx, x: *const f32, w: *const f32, g: *const f32, gscale: *const f32, gfactor: f32, dx: *mut f32, dw: *mut f32, n: usize, c: usize, h: usize, wd: usize, k: usize, r: usize, s: usize, stride: usize, pad: usize, accumulate: i32) -> i32;
    pub fn katsu_cuda_conv2d_fwd_bias_relu(ctx: *mut Ctx, x: *const f32, w: *const f32, bias: *const f32, y: *mut f32, n: usize, c: usize, h: usize, wd: usize, k: usize, r: usize, s: usize, stride: usize, pad: usize, relu: i32) -> i32;
    pub fn katsu_cuda_conv2d_staged_floats(ctx: *mut Ctx, n: usize, c: usize, h: usize, wd: usize, k: usize, r: usize, s: usize, stride: usize, pad: usize, floats: *mut usize) -> i32;
    pub fn katsu_cuda_conv2d_stage(ctx: *mut Ctx, x: *const f32, staged: *mut f32, n: usize, c: usize, h: usize, wd: usize) -> i32;
    pub fn katsu_cuda_conv2d_fwd_staged(ctx: *mut Ctx, x: *const f32, x_staged: *const f32, w: *const f32, bias: *const f32, y: *mut f32, n: usize, c: usize, h: usize, wd: usize, k: usize, r: usize, s: usize, stride: usize, pad: usize, relu: i32) -> i32;
    pub fn katsu_cuda_conv2d_bwd_staged(ctx: *mut Ctx, x: *const f32, x_staged: *const f32, w: *const f32, g: *const f32, gscale: *const f32, gfactor: f32, dx: *mut f32, dw: *mut f32, n: usize, c: usize, h: usize, wd: usize, k: usize, r: usize, s: usize, stride: usize, pad: usize, accumulate: i32) -> i32;
    pub fn katsu_cuda_bias_relu_bwd(ctx: *mut Ctx, y_act: *const f32, g: *const f32, dg: *mut f32, dbias: *mut f32, n: usize, k: usize, plane: usize, relu: i32, accumulate_bias: i32) -> i32;
    pub fn katsu_cuda_sgd_step(ctx: *mut Ctx, w: *mut f32, dw: *const f32, lr: f32, count: usize) -> i32;
    pub fn katsu_cuda_matmul_fwd(ctx: *mut Ctx, a: *const f32, b: *const f32, c: *mut f32, m: usize, k: usize, n: usize) -> i32;
    pub fn katsu_cuda_matmul_bwd(ctx: *mut Ctx, a: *const f32, b: *const f32, g: *const f32, da: *mut f32, db: *mut f32, m: usize, k: usize, n: usize, accumulate: i32) -> i32;
    pub fn katsu_cuda_block_norm_fwd(ctx: *mut Ctx, x: *const f32, h: *const f32, gate: *const f32, gate_rows: usize, post_w: *const f32, post_b: *const f32, pre_w: *const f32, pre_b: *const f32, scale: f32, eps: f32, kind: i32, r: *mut f32, n: *mut f32, rows: usize, cols: usize) -> i32;
    pub fn katsu_cuda_block_norm_bwd(ctx: *mut Ctx, r: *const f32, h: *const f32, gate: *const f32, gate_rows: usize, post_w: *const f32, post_b: *const f32, pre_w: *const f32, scale: f32, eps: f32, kind: i32, dr: *const f32, dn: *const f32, dx: *mut f32, dh: *mut f32, dgate: *mut f32, dpost_w: *mut f32, dpost_b: *mut f32, dpre_w: *mut f32, dpre_b: *mut f32, rows: usize, cols: usize, accumulate: i32) -> i32;
    pub fn katsu_cuda_int8_row_bytes(k: usize, out_bytes: *mut usize) -> i32;
    pub fn katsu_cuda_int8_quantize_weights(ctx: *mut Ctx, w: *const f32, q: *mut i8, scale: *mut f32, k: usize, n: usize) -> i32;
    pub fn katsu_cuda_int8_quantize_rows(ctx: *mut Ctx, x: *const f32, q: *mut i8, scale: *mut f32, m: usize, k: usize) -> i32;
    pub fn katsu_cuda_int8_matmul(ctx: *mut Ctx, xq: *const i8, xs: *const f32, wq: *const i8, ws: *const f32, bias: *const f32, y: *mut f32, m: usize, k: usize, n: usize) -> i32;
    pub fn katsu_cuda_int8_linear(ctx: *mut Ctx, x: *const f32, wq: *const i8, ws: *const f32, bias: *const f32, y: *mut f32, m: usize, k: usize, n: usize) -> i32;
    pub fn katsu_cuda_grad_norm(ctx: *mut Ctx, grads: *const *const f32, counts: *const usize, tensors: usize, norm: *mut f32) -> i32;
    pub fn katsu_cuda_clip_grads(ctx: *mut Ctx, grads: *const *const f32, out: *const *mut f32, counts: *const usize, tensors: usize, max_norm: f32, norm: *mut f32) -> i32;
    pub fn katsu_cuda_sgd_step_clipped(ctx: *mut Ctx, weights: *const *mut f32, grads: *const *const f32, counts: *const usize, tensors: usize, lr: f32, max_norm: f32, norm: *mut f32) -> i32;
    pub fn katsu_cuda_embed_fwd(ctx: *mut Ctx, table: *const f32, tokens: *const i32, scale: f32, y: *mut f32, count: usize, vocab: usize, cols: usize) -> i32;
    pub fn katsu_cuda_int8_embed(ctx: *mut Ctx, q: *const i8, rows_scale: *const f32, tokens: *const i32, scale: f32, y: *mut f32, count: usize, vocab: usize, cols: usize) -> i32;
    pub fn katsu_cuda_embed_bwd(ctx: *mut Ctx, tokens: *const i32, dy: *const f32, scale: f32, dtable: *mut f32, count: usize, vocab: usize, cols: usize, accumulate: i32) -> i32;
    pub fn katsu_cuda_distill_fwd(ctx: *mut Ctx, logits: *const f32, teacher: *const f32, index: *const i32, labels: *const i32, weight: *const f32, temperature: f32, soft: f32, hard: f32, loss: *mut f32, rows: usize, vocab: usize, top: usize) -> i32;
    pub fn katsu_cuda_distill_bwd(ctx: *mut Ctx, logits: *const f32, teacher: *const f32, index: *const i32, labels: *const i32, weight: *const f32, temperature: f32, soft: f32, hard: f32, g: *const f32, loss: *mut f32, dlogits: *mut f32, rows: usize, vocab: usize, top: usize, accumulate: i32) -> i32;
    pub fn katsu_cuda_adjust_logits(ctx: *mut Ctx, logits: *const f32, history: *const i32, prompts: *const i32, lengths: *const i32, repetition: *const f32, presence: *const f32, frequency: *const f32, bias_tokens: *const i32, bias: *const f32, allowed: *const u32, out: *mut f32, rows: usize, vocab: usize, history_cols: usize, biases: usize) -> i32;
    pub fn katsu_cuda_add(ctx: *mut Ctx, a: *const f32, b: *const f32, out: *mut f32, count: usize) -> i32;
    pub fn katsu_cuda_mul(ctx: *mut Ctx, a: *const f32, b: *const f32, out: *mut f32, count: usize) -> i32;
    pub fn katsu_cuda_sum(ctx: *mut Ctx, a: *const f32, out: *mut f32, count: usize) -> i32;
    pub fn katsu_cuda_sum_static(ctx: *mut Ctx, a: *const f32, out: *mut f32, count: usize) -> i32;
    pub fn katsu_cuda_sumsq(ctx: *mut Ctx, a: *const f32, out: *mut f32, count: usize) -> i32;
    pub fn katsu_cuda_square_vjp(ctx: *mut Ctx, dst: *mut f32, src: *const f32, s: *const f32, count: usize, accumulate: i32) -> i32;
    pub fn katsu_cuda_axpy_acc(ctx: *mut Ctx, dst: *mut f32, g: *const f32, count: usize) -> i32;
    pub fn katsu_cuda_mul_acc(ctx: *mut Ctx, dst: *mut f32, g: *const f32, other: *const f32, count: usize) -> i32;
    pub fn katsu_cuda_bcast_acc(ctx: *mut Ctx, dst: *mut f32, g: *const f32, count: usize) -> i32;
    pub fn katsu_cuda_comm_unique_id(out_id: *mut u8) -> i32;
    pub fn katsu_cuda_comm_init(ctx: *mut Ctx, id: *const u8, n_ranks: i32, rank: i32) -> i32;
    pub fn katsu_cuda_comm_destroy(ctx: *mut Ctx) -> i32;
    pub fn katsu_cuda_allreduce_sum(ctx: *mut Ctx, buf: *mut f32, count: usize) -> i32;
    pub fn katsu_cuda_selftest_wait_timeout(ctx: *mut Ctx, cycles: u64) -> i32;
    pub fn katsu_cuda_selftest_mailbox_allreduce(ctx: *mut Ctx, buf: *mut f32, ranks: i32, count: usize, absent: i32, cycles: u64) -> i32;
    pub fn katsu_cuda_event_create(ctx: *mut Ctx, out_event: *mut *mut Event) -> i32;
    pub fn katsu_cuda_event_record(ctx: *mut Ctx, event: *mut Event) -> i32;
    pub fn katsu_cuda_event_elapsed_ms(ctx: *mut Ctx, start: *mut Event, stop: *mut Event, out_ms: *mut f32) -> i32;
    pub fn katsu_cuda_event_destroy(ctx: *mut Ctx, event: *mut Event) -> i32;
    pub fn katsu_cuda_wait_event(ctx: *mut Ctx, event: *mut Event) -> i32;
    pub fn katsu_cuda_flush_l2(ctx: *mut Ctx) -> i32;
}
