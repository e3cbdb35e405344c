//! katsu-cuda: safe Rust over the C ABI of libkatsu_cuda.so (include/katsu_cuda.h), the sm_100a
//! replacement for katsu-core's dense loops (Conv2D forward / backward_buffers, matmul and its
//! VJP, the streaming ops that keep the autograd graph on the device).
//!
//! This is the only crate of the workspace that contains `unsafe`; katsu-core keeps
//! `#![forbid(unsafe_code)]` (crates/katsu-core/src/lib.rs:2) and calls the functions below.
//!
//! NOT COMPILED in the repository that carries the kernels (no Rust toolchain in its build image).
//! The same boundary is exercised there by the C++ mirror of katsu-core (katsu_b200/csrc/host) and
//! by ctypes tests; `ffi.rs` is generated from the header and checked against it by a test.
//!
//! Threading: `Context` is `!Send + !Sync` (it holds a raw pointer), matching katsu-core's
//! `Rc`-based, single-threaded `Tensor` (crates/katsu-core/src/tensor.rs:95-99).  One context is
//! one device and one stream; calls are asynchronous and ordered on it; `sync`, `DeviceBuf::to_host`
//! and `Event::elapsed_ms` wait.

pub mod ffi;

use std::ffi::CStr;
use std::fmt;
use std::marker::PhantomData;
use std::ptr;
use std::rc::Rc;

/// A failed call: the status code of include/katsu_cuda.h and the library's message.
#[derive(Debug, Clone, PartialEq, Eq)]
pub struct CudaError {
    pub code: i32,
    pub message: String,
}

impl CudaError {
    /// katsu-core maps this to `TensorError::Allocation`, everything else to `TensorError::Device`.
    pub fn is_allocation(&self) -> bool {
        self.code == ffi::KATSU_ERR_ALLOC
    }
    /// A bounded device-side wait gave up; results queued since the last check are undefined.
    pub fn is_timeout(&self) -> bool {
        self.code == ffi::KATSU_ERR_TIMEOUT
    }
}

impl fmt::Display for CudaError {
    fn fmt(&self, f: &mut fmt::Formatter<'_>) -> fmt::Result {
        write!(f, "katsu_cuda error {}: {}", self.code, self.message)
    }
}

impl std::error::Error for CudaError {}

fn check(code: i32) -> Result<(), CudaError> {
    if code == ffi::KATSU_OK {
        return Ok(());
    }
    // SAFETY: the library returns a pointer to a NUL-terminated thread-local buffer.
    let message = unsafe { CStr::from_ptr(ffi::katsu_cuda_last_error_string()) }.to_string_lossy().into_owned();
    Err(CudaError { code, message })
}

/// Arithmetic mode of the contraction kernels.
#[derive(Debug, Clone, Copy, PartialEq, Eq)]
pub enum Precision {
    /// Tensor cores, split precision (hi*hi + lo*hi + hi*lo): FP32-grade accuracy.  Default.
    ThreeXTf32,
    /// Tensor cores, one TF32 pass (relative error about 1e-3).
    Tf32,
    /// CUDA cores only.
    Fp32,
}

struct RawContext(*mut ffi::Ctx);

impl Drop for RawContext {
    fn drop(&mut self) {
        // SAFETY: created by katsu_cuda_init, dropped once (Rc), no buffer outlives it (they hold an Rc).
        unsafe { ffi::katsu_cuda_shutdown(self.0) };
    }
}

/// One device, one stream.  Cheap to clone (reference counted); buffers keep their context alive.
#[derive(Clone)]
pub struct Context {
    raw: Rc<RawContext>,
}

impl Context {
    pub fn device_count() -> Result<usize, CudaError> {
        let mut n = 0i32;
        check(unsafe { ffi::katsu_cuda_device_count(&mut n) })?;
        Ok(n.max(0) as usize)
    }

    pub fn new(device: usize) -> Result<Self, CudaError> {
        let mut raw = ptr::null_mut();
        check(unsafe { ffi::katsu_cuda_init(device as i32, &mut raw) })?;
        Ok(Self { raw: Rc::new(RawContext(raw)) })
    }

    fn ptr(&self) -> *mut ffi::Ctx {
        self.raw.0
    }

    pub fn set_precision(&self, mode: Precision) -> Result<(), CudaError> {
        let raw = match mode {
            Precision::ThreeXTf32 => ffi::KATSU_MODE_3XTF32,
            Precision::Tf32 => ffi::KATSU_MODE_TF32,
            Precision::Fp32 => ffi::KATSU_MODE_FP32,
        };
        check(unsafe { ffi::katsu_cuda_set_precision(self.ptr(), raw) })
    }

    /// Waits for everything queued; `Err(timeout)` once if a device-side wait gave up since the last check.
    pub fn sync(&self) -> Result<(), CudaError> {
        check(unsafe { ffi::katsu_cuda_sync(self.ptr()) })
    }

    pub fn launch_count(&self) -> Result<u64, CudaError> {
        let mut n = 0u64;
        check(unsafe { ffi::katsu_cuda_launch_count(self.ptr(), &mut n) })?;
        Ok(n)
    }
}

/// Owned device buffer of f32: the device variant of `TensorNode.data`
/// (crates/katsu-core/src/tensor.rs:101-107).  Freed (stream-ordered) on drop.
pub struct DeviceBuf {
    ctx: Context,
    ptr: *mut f32,
    len: usize,
    _not_send: PhantomData<*mut f32>,
}

impl DeviceBuf {
    /// Zero-filled, like `zeros_buffer` (tensor.rs:120-125).
    pub fn zeros(ctx: &Context, len: usize) -> Result<Self, CudaError> {
        let mut ptr = ptr::null_mut();
        check(unsafe { ffi::katsu_cuda_alloc(ctx.ptr(), len, &mut ptr) })?;
        Ok(Self { ctx: ctx.clone(), ptr, len, _not_send: PhantomData })
    }

    pub fn from_host(ctx: &Context, data: &[f32]) -> Result<Self, CudaError> {
        let buf = Self::zeros(ctx, data.len())?;
        check(unsafe { ffi::katsu_cuda_h2d(ctx.ptr(), buf.ptr, data.as_ptr(), data.len()) })?;
        ctx.sync()?; // `data` is pageable and may be dropped by the caller right away
        Ok(buf)
    }

    /// Synchronous copy back: what `Tensor::data()` / `Tensor::grad()` fill their host mirror with.
    pub fn to_host(&self) -> Result<Vec<f32>, CudaError> {
        let mut out = vec![0.0f32; self.len];
        check(unsafe { ffi::katsu_cuda_d2h(self.ctx.ptr(), out.as_mut_ptr(), self.ptr, self.len) })?;
        Ok(out)
    }

    pub fn len(&self) -> usize {
        self.len
    }
    pub fn is_empty(&self) -> bool {
        self.len == 0
    }
    pub fn as_ptr(&self) -> *const f32 {
        self.ptr
    }
    pub fn as_mut_ptr(&mut self) -> *mut f32 {
        self.ptr
    }
    pub fn context(&self) -> &Context {
        &self.ctx
    }
}

impl Drop for DeviceBuf {
    fn drop(&mut self) {
        // SAFETY: allocated by katsu_cuda_alloc on this context; freeing is ordered behind queued work.
        unsafe { ffi::katsu_cuda_free(self.ctx.ptr(), self.ptr) };
    }
}

fn opt_mut(buf: Option<&mut DeviceBuf>) -> *mut f32 {
    buf.map_or(ptr::null_mut(), |b| b.ptr)
}

fn opt_const(buf: Option<&DeviceBuf>) -> *const f32 {
    buf.map_or(ptr::null(), |b| b.ptr as *const f32)
}

/// Output of `Geometry::new` (crates/katsu-core/src/conv2d.rs:183-224); katsu-core validates, this
/// crate only carries the numbers across.
#[derive(Debug, Clone, Copy)]
pub struct ConvGeometry {
    pub batch: usize,
    pub cin: usize,
    pub h: usize,
    pub w: usize,
    pub cout: usize,
    pub kh: usize,
    pub kw: usize,
    pub oh: usize,
    pub ow: usize,
    pub stride: usize,
    pub padding: usize,
}

impl ConvGeometry {
    fn x_len(&self) -> usize {
        self.batch * self.cin * self.h * self.w
    }
    fn w_len(&self) -> usize {
        self.cout * self.cin * self.kh * self.kw
    }
    fn y_len(&self) -> usize {
        self.batch * self.cout * self.oh * self.ow
    }
}

fn length(what: &str, buf: &DeviceBuf, expected: usize) -> Result<(), CudaError> {
    if buf.len == expected {
        Ok(())
    } else {
        Err(CudaError { code: ffi::KATSU_ERR_INVALID_ARG, message: format!("{what}: expected {expected} elements, got {}", buf.len) })
    }
}

/// The visit closure of `Conv2D::forward` (conv2d.rs:95-103, 232-262); y is overwritten.
/// `bias` / `relu` are additions that ride in the kernel's epilogue.
pub fn conv2d_forward(ctx: &Context, x: &DeviceBuf, w: &DeviceBuf, bias: Option<&DeviceBuf>, relu: bool, y: &mut DeviceBuf,
                      g: &ConvGeometry) -> Result<(), CudaError> {
    length("x", x, g.x_len())?;
    length("w", w, g.w_len())?;
    length("y", y, g.y_len())?;
    if let Some(b) = bias {
        length("bias", b, g.cout)?;
    }
    check(unsafe {
        ffi::katsu_cuda_conv2d_fwd_bias_relu(ctx.ptr(), x.ptr, w.ptr, opt_const(bias), y.ptr, g.batch, g.cin, g.h, g.w, g.cout,
                                             g.kh, g.kw, g.stride, g.padding, relu as i32)
    })
}

/// Size in floats of the channels-innermost copy of x that this geometry's kernels read in the context's
/// current precision mode; 0 when they read x directly.
pub fn conv2d_staged_len(ctx: &Context, g: &ConvGeometry) -> Result<usize, CudaError> {
    let mut floats: usize = 0;
    check(unsafe {
        ffi::katsu_cuda_conv2d_staged_floats(ctx.ptr(), g.batch, g.cin, g.h, g.w, g.cout, g.kh, g.kw, g.stride, g.padding,
                                             &mut floats)
    })?;
    Ok(floats)
}

/// Writes that copy.  `Conv2D` holds its input from forward to backward (conv2d.rs:104-107, 130-136); holding
/// this copy beside it lets both calls skip their own staging pass.
pub fn conv2d_stage(ctx: &Context, x: &DeviceBuf, staged: &mut DeviceBuf, g: &ConvGeometry) -> Result<(), CudaError> {
    length("x", x, g.x_len())?;
    length("staged", staged, conv2d_staged_len(ctx, g)?)?;
    check(unsafe { ffi::katsu_cuda_conv2d_stage(ctx.ptr(), x.ptr, staged.ptr, g.batch, g.cin, g.h, g.w) })
}

/// `conv2d_forward` reading x through its staged copy (bit-identical to the plain call).
pub fn conv2d_forward_staged(ctx: &Context, x: &DeviceBuf, staged: Option<&DeviceBuf>, w: &DeviceBuf, bias: Option<&DeviceBuf>,
                             relu: bool, y: &mut DeviceBuf, g: &ConvGeometry) -> Result<(), CudaError> {
    length("x", x, g.x_len())?;
    length("w", w, g.w_len())?;
    length("y", y, g.y_len())?;
    check(unsafe {
        ffi::katsu_cuda_conv2d_fwd_staged(ctx.ptr(), x.ptr, opt_const(staged), w.ptr, opt_const(bias), y.ptr, g.batch, g.cin,
                                          g.h, g.w, g.cout, g.kh, g.kw, g.stride, g.padding, relu as i32)
    })
}

/// `conv2d_backward` reading x through its staged copy (dW).
pub fn conv2d_backward_staged(ctx: &Context, x: &DeviceBuf, staged: Option<&DeviceBuf>, w: &DeviceBuf, grad: &DeviceBuf,
                              scale: Option<GradScale<'_>>, dx: Option<&mut DeviceBuf>, dw: Option<&mut DeviceBuf>,
                              g: &ConvGeometry, accumulate: bool) -> Result<(), CudaError> {
    length("x", x, g.x_len())?;
    length("w", w, g.w_len())?;
    length("grad", grad, g.y_len())?;
    let (scalar, factor) = scale.map_or((ptr::null(), 1.0), |s| (opt_const(s.scalar), s.factor));
    check(unsafe {
        ffi::katsu_cuda_conv2d_bwd_staged(ctx.ptr(), x.ptr, opt_const(staged), w.ptr, grad.ptr, scalar, factor, opt_mut(dx),
                                          opt_mut(dw), g.batch, g.cin, g.h, g.w, g.cout, g.kh, g.kw, g.stride, g.padding,
                                          accumulate as i32)
    })
}

/// Scale of the upstream gradient handed to `conv2d_backward`: the gradient is `factor * scalar[0] * g`
/// without being stored (what the VJP of `sum(y * y)` sends: g = y, factor 2, scalar = the loss adjoint).
pub struct GradScale<'a> {
    pub scalar: Option<&'a DeviceBuf>,
    pub factor: f32,
}

/// One `backward_buffers` (conv2d.rs:269-292).  `dx` / `dw` may be `None`; `accumulate` adds to their
/// contents, which folds in the `pending[parent] += grad` pass of tensor.rs:383-390.
pub fn conv2d_backward(ctx: &Context, x: &DeviceBuf, w: &DeviceBuf, grad: &DeviceBuf, scale: Option<GradScale<'_>>,
                       dx: Option<&mut DeviceBuf>, dw: Option<&mut DeviceBuf>, g: &ConvGeometry, accumulate: bool)
                       -> Result<(), CudaError> {
    length("x", x, g.x_len())?;
    length("w", w, g.w_len())?;
    length("grad", grad, g.y_len())?;
    if let Some(b) = dx.as_deref() {
        length("dx", b, g.x_len())?;
    }
    if let Some(b) = dw.as_deref() {
        length("dw", b, g.w_len())?;
    }
    let (scalar, factor) = scale.map_or((ptr::null(), 1.0), |s| (opt_const(s.scalar), s.factor));
    check(unsafe {
        ffi::katsu_cuda_conv2d_bwd_scaled(ctx.ptr(), x.ptr, w.ptr, grad.ptr, scalar, factor, opt_mut(dx), opt_mut(dw), g.batch,
                                          g.cin, g.h, g.w, g.cout, g.kh, g.kw, g.stride, g.padding, accumulate as i32)
    })
}

/// VJP of the bias / ReLU epilogue: `dg` = grad where `y_act > 0` (else 0), `dbias[k]` (+)= its sum.
pub fn bias_relu_backward(ctx: &Context, y_act: &DeviceBuf, grad: &DeviceBuf, dg: Option<&mut DeviceBuf>,
                          dbias: Option<&mut DeviceBuf>, g: &ConvGeometry, relu: bool, accumulate_bias: bool)
                          -> Result<(), CudaError> {
    length("y", y_act, g.y_len())?;
    length("grad", grad, g.y_len())?;
    check(unsafe {
        ffi::katsu_cuda_bias_relu_bwd(ctx.ptr(), y_act.ptr, grad.ptr, opt_mut(dg), opt_mut(dbias), g.batch, g.cout, g.oh * g.ow,
                                      relu as i32, accumulate_bias as i32)
    })
}

/// `Tensor::matmul` (tensor.rs:264-273): c[m,n] = a[m,k] @ b[k,n].
pub fn matmul(ctx: &Context, a: &DeviceBuf, b: &DeviceBuf, c: &mut DeviceBuf, m: usize, k: usize, n: usize)
              -> Result<(), CudaError> {
    length("a", a, m * k)?;
    length("b", b, k * n)?;
    length("c", c, m * n)?;
    check(unsafe { ffi::katsu_cuda_matmul_fwd(ctx.ptr(), a.ptr, b.ptr, c.ptr, m, k, n) })
}

/// Matmul VJP (tensor.rs:418-445): da (+)= g @ b^T, db (+)= a^T @ g.
pub fn matmul_backward(ctx: &Context, a: &DeviceBuf, b: &DeviceBuf, grad: &DeviceBuf, da: Option<&mut DeviceBuf>,
                       db: Option<&mut DeviceBuf>, m: usize, k: usize, n: usize, accumulate: bool) -> Result<(), CudaError> {
    length("a", a, m * k)?;
    length("b", b, k * n)?;
    length("grad", grad, m * n)?;
    check(unsafe {
        ffi::katsu_cuda_matmul_bwd(ctx.ptr(), a.ptr, b.ptr, grad.ptr, opt_mut(da), opt_mut(db), m, k, n, accumulate as i32)
    })
}

macro_rules! same_len {
    ($($buf:expr),+ ; $len:expr) => { $( length(stringify!($buf), $buf, $len)?; )+ };
}

/// `Tensor::add` / `Tensor::mul` (tensor.rs:226-233).
pub fn add(ctx: &Context, a: &DeviceBuf, b: &DeviceBuf, out: &mut DeviceBuf) -> Result<(), CudaError> {
    same_len!(b, out; a.len);
    check(unsafe { ffi::katsu_cuda_add(ctx.ptr(), a.ptr, b.ptr, out.ptr, a.len) })
}
pub fn mul(ctx: &Context, a: &DeviceBuf, b: &DeviceBuf, out: &mut DeviceBuf) -> Result<(), CudaError> {
    same_len!(b, out; a.len);
    check(unsafe { ffi::katsu_cuda_mul(ctx.ptr(), a.ptr, b.ptr, out.ptr, a.len) })
}
/// `Tensor::sum` (tensor.rs:243-247) into a one-element buffer.
pub fn sum(ctx: &Context, a: &DeviceBuf, out: &mut DeviceBuf) -> Result<(), CudaError> {
    length("out", out, 1)?;
    check(unsafe { ffi::katsu_cuda_sum(ctx.ptr(), a.ptr, out.ptr, a.len) })
}
/// sum(a * a) in one pass, bit-identical to `mul` then `sum`.
pub fn sum_of_squares(ctx: &Context, a: &DeviceBuf, out: &mut DeviceBuf) -> Result<(), CudaError> {
    length("out", out, 1)?;
    check(unsafe { ffi::katsu_cuda_sumsq(ctx.ptr(), a.ptr, out.ptr, a.len) })
}
/// Both Mul VJP edges of y * y under a broadcast adjoint `scalar[0]` (tensor.rs:392-417).
pub fn square_vjp(ctx: &Context, dst: &mut DeviceBuf, src: &DeviceBuf, scalar: &DeviceBuf, accumulate: bool)
                  -> Result<(), CudaError> {
    same_len!(src; dst.len);
    length("scalar", scalar, 1)?;
    check(unsafe { ffi::katsu_cuda_square_vjp(ctx.ptr(), dst.ptr, src.ptr, scalar.ptr, dst.len, accumulate as i32) })
}
/// dst += g (tensor.rs:353-356, 387-389, 400-408).
pub fn axpy_acc(ctx: &Context, dst: &mut DeviceBuf, g: &DeviceBuf) -> Result<(), CudaError> {
    same_len!(g; dst.len);
    check(unsafe { ffi::katsu_cuda_axpy_acc(ctx.ptr(), dst.ptr, g.ptr, dst.len) })
}
/// dst += g * other (Mul VJP edge, tensor.rs:400-408).
pub fn mul_acc(ctx: &Context, dst: &mut DeviceBuf, g: &DeviceBuf, other: &DeviceBuf) -> Result<(), CudaError> {
    same_len!(g, other; dst.len);
    check(unsafe { ffi::katsu_cuda_mul_acc(ctx.ptr(), dst.ptr, g.ptr, other.ptr, dst.len) })
}
/// dst += g[0] (Sum VJP, tensor.rs:410-417).
pub fn bcast_acc(ctx: &Context, dst: &mut DeviceBuf, g: &DeviceBuf) -> Result<(), CudaError> {
    length("g", g, 1)?;
    check(unsafe { ffi::katsu_cuda_bcast_acc(ctx.ptr(), dst.ptr, g.ptr, dst.len) })
}
/// w -= lr * dw (docs/roadmap.md:21-22).
pub fn sgd_step(ctx: &Context, w: &mut DeviceBuf, dw: &DeviceBuf, lr: f32) -> Result<(), CudaError> {
    same_len!(dw; w.len);
    check(unsafe { ffi::katsu_cuda_sgd_step(ctx.ptr(), w.ptr, dw.ptr, lr, w.len) })
}

/// A norm's weight and bias, one value per channel.
#[derive(Clone, Copy)]
pub struct NormWeights<'a> {
    pub weight: &'a DeviceBuf,
    pub bias: Option<&'a DeviceBuf>,
}

/// Kind and eps of the norms around a block, and the residual scale.
#[derive(Debug, Clone, Copy)]
pub struct BlockNorm {
    pub layer: bool,
    pub eps: f32,
    pub scale: f32,
    pub rows: usize,
    pub cols: usize,
}

impl BlockNorm {
    fn kind(&self) -> i32 {
        if self.layer { ffi::KATSU_NORM_LAYER } else { ffi::KATSU_NORM_RMS }
    }
    fn gate_rows(&self, gate: Option<&DeviceBuf>) -> Result<usize, CudaError> {
        match gate {
            None => Ok(0),
            Some(g) if self.cols != 0 && g.len != 0 && g.len % self.cols == 0 => Ok(g.len / self.cols),
            Some(g) => Err(CudaError {
                code: ffi::KATSU_ERR_INVALID_ARG,
                message: format!("gate: {} elements are no whole rows of {}", g.len, self.cols),
            }),
        }
    }
    fn weights(&self, w: Option<NormWeights<'_>>) -> Result<(*const f32, *const f32), CudaError> {
        if let Some(w) = w {
            length("weight", w.weight, self.cols)?;
            if let Some(b) = w.bias {
                length("bias", b, self.cols)?;
            }
        }
        Ok((opt_const(w.map(|w| w.weight)), opt_const(w.and_then(|w| w.bias))))
    }
}

/// r = x + scale * gate * N(h; post), n = N(r; pre) in one pass; see katsu_cuda_block_norm_fwd for the parts that may be left out.
pub fn block_norm_forward(ctx: &Context, x: &DeviceBuf, h: Option<&DeviceBuf>, gate: Option<&DeviceBuf>,
                          post: Option<NormWeights<'_>>, pre: Option<NormWeights<'_>>, r: Option<&mut DeviceBuf>,
                          n: Option<&mut DeviceBuf>, g: &BlockNorm) -> Result<(), CudaError> {
    let count = g.rows * g.cols;
    for buf in [Some(x), h, r.as_deref(), n.as_deref()].into_iter().flatten() {
        length("x, h, r or n", buf, count)?;
    }
    let ((post_w, post_b), (pre_w, pre_b)) = (g.weights(post)?, g.weights(pre)?);
    let gate_rows = g.gate_rows(gate)?;
    check(unsafe {
        ffi::katsu_cuda_block_norm_fwd(ctx.ptr(), x.ptr, opt_const(h), opt_const(gate), gate_rows, post_w, post_b, pre_w,
                                       pre_b, g.scale, g.eps, g.kind(), opt_mut(r), opt_mut(n), g.rows, g.cols)
    })
}

/// What `block_norm_backward` writes; `None` is skipped.
#[derive(Default)]
pub struct BlockNormGrads<'a> {
    pub x: Option<&'a mut DeviceBuf>,
    pub h: Option<&'a mut DeviceBuf>,
    pub gate: Option<&'a mut DeviceBuf>,
    pub post_weight: Option<&'a mut DeviceBuf>,
    pub post_bias: Option<&'a mut DeviceBuf>,
    pub pre_weight: Option<&'a mut DeviceBuf>,
    pub pre_bias: Option<&'a mut DeviceBuf>,
}

/// Its backward.  `accumulate` is a sum of `ffi::KATSU_BLOCK_*`: those outputs are added to their contents.
pub fn block_norm_backward(ctx: &Context, r: &DeviceBuf, h: Option<&DeviceBuf>, gate: Option<&DeviceBuf>,
                           post: Option<NormWeights<'_>>, pre_weight: Option<&DeviceBuf>, dr: Option<&DeviceBuf>,
                           dn: Option<&DeviceBuf>, out: BlockNormGrads<'_>, g: &BlockNorm, accumulate: i32)
                           -> Result<(), CudaError> {
    let count = g.rows * g.cols;
    for buf in [Some(r), h, dr, dn, out.x.as_deref(), out.h.as_deref()].into_iter().flatten() {
        length("r, h, dr, dn or their gradients", buf, count)?;
    }
    let per_channel = [pre_weight, out.post_weight.as_deref(), out.post_bias.as_deref(), out.pre_weight.as_deref(), out.pre_bias.as_deref()];
    for buf in per_channel.into_iter().flatten() {
        length("weights or their gradients", buf, g.cols)?;
    }
    if let (Some(gate), Some(dgate)) = (gate, out.gate.as_deref()) {
        length("gate gradient", dgate, gate.len)?;
    }
    let (post_w, post_b) = g.weights(post)?;
    let gate_rows = g.gate_rows(gate)?;
    check(unsafe {
        ffi::katsu_cuda_block_norm_bwd(ctx.ptr(), r.ptr, opt_const(h), opt_const(gate), gate_rows, post_w, post_b,
                                       opt_const(pre_weight), g.scale, g.eps, g.kind(), opt_const(dr), opt_const(dn), opt_mut(out.x),
                                       opt_mut(out.h), opt_mut(out.gate), opt_mut(out.post_weight), opt_mut(out.post_bias),
                                       opt_mut(out.pre_weight), opt_mut(out.pre_bias), g.rows, g.cols, accumulate)
    })
}

/// Weights [k, n] in 8 bits with a scale per output channel, laid out once for `int8_linear`.
pub struct Int8Weights {
    q: DeviceBuf,
    scale: DeviceBuf,
    k: usize,
    n: usize,
}

impl Int8Weights {
    pub fn new(ctx: &Context, weights: &DeviceBuf, k: usize, n: usize) -> Result<Self, CudaError> {
        length("weights", weights, k * n)?;
        let mut bytes = 0usize;
        check(unsafe { ffi::katsu_cuda_int8_row_bytes(k, &mut bytes) })?;
        let (q, scale) = (DeviceBuf::zeros(ctx, n * bytes / 4)?, DeviceBuf::zeros(ctx, n)?);
        check(unsafe { ffi::katsu_cuda_int8_quantize_weights(ctx.ptr(), weights.ptr, q.ptr as *mut i8, scale.ptr, k, n) })?;
        Ok(Self { q, scale, k, n })
    }
}

/// y[m, n] = x[m, k] w + bias with the rows of x in 8 bits too (katsu_cuda_int8_linear).
pub fn int8_linear(ctx: &Context, x: &DeviceBuf, w: &Int8Weights, bias: Option<&DeviceBuf>, y: &mut DeviceBuf, m: usize)
                   -> Result<(), CudaError> {
    length("x", x, m * w.k)?;
    length("y", y, m * w.n)?;
    if let Some(b) = bias {
        length("bias", b, w.n)?;
    }
    check(unsafe {
        ffi::katsu_cuda_int8_linear(ctx.ptr(), x.ptr, w.q.ptr as *const i8, w.scale.ptr, opt_const(bias), y.ptr, m, w.k, w.n)
    })
}

/// Tokens (32-bit whole numbers) on the device; what is no token of a vocabulary, negative numbers for one, stands for none.
pub struct TokenBuf {
    words: DeviceBuf,
}

impl TokenBuf {
    pub fn from_host(ctx: &Context, tokens: &[i32]) -> Result<Self, CudaError> {
        let words = DeviceBuf::zeros(ctx, tokens.len())?;
        // h2d copies 4-byte elements as they are; `tokens` may be dropped right away
        check(unsafe { ffi::katsu_cuda_h2d(ctx.ptr(), words.ptr, tokens.as_ptr() as *const f32, tokens.len()) })?;
        ctx.sync()?;
        Ok(Self { words })
    }
    pub fn len(&self) -> usize {
        self.words.len
    }
    pub fn is_empty(&self) -> bool {
        self.words.len == 0
    }
    fn ptr(&self) -> *const i32 {
        self.words.ptr as *const i32
    }
}

fn opt_tokens(tokens: Option<&TokenBuf>) -> *const i32 {
    tokens.map_or(ptr::null(), |t| t.ptr())
}

/// y[i] = scale * table[tokens[i]] for a table [vocab, cols].
pub fn embed_forward(ctx: &Context, table: &DeviceBuf, tokens: &TokenBuf, scale: f32, y: &mut DeviceBuf, vocab: usize, cols: usize)
                     -> Result<(), CudaError> {
    length("table", table, vocab * cols)?;
    length("y", y, tokens.len() * cols)?;
    check(unsafe { ffi::katsu_cuda_embed_fwd(ctx.ptr(), table.ptr, tokens.ptr(), scale, y.ptr, tokens.len(), vocab, cols) })
}

/// dtable[v] (+)= scale * sum of dy[i] over the tokens that are v.
pub fn embed_backward(ctx: &Context, tokens: &TokenBuf, dy: &DeviceBuf, scale: f32, dtable: &mut DeviceBuf, vocab: usize, cols: usize,
                      accumulate: bool) -> Result<(), CudaError> {
    length("dy", dy, tokens.len() * cols)?;
    length("dtable", dtable, vocab * cols)?;
    check(unsafe {
        ffi::katsu_cuda_embed_bwd(ctx.ptr(), tokens.ptr(), dy.ptr, scale, dtable.ptr, tokens.len(), vocab, cols, accumulate as i32)
    })
}

/// `embed_forward` from the 8-bit weights [k, n] of a head that are the table of its n tokens too: y is [tokens, k].
pub fn int8_embed(ctx: &Context, w: &Int8Weights, tokens: &TokenBuf, scale: f32, y: &mut DeviceBuf) -> Result<(), CudaError> {
    length("y", y, tokens.len() * w.k)?;
    check(unsafe {
        ffi::katsu_cuda_int8_embed(ctx.ptr(), w.q.ptr as *const i8, w.scale.ptr, tokens.ptr(), scale, y.ptr, tokens.len(), w.n, w.k)
    })
}

/// Loss against a teacher's top logits (rows of `top`) and against labels, for every row of logits; see katsu_cuda_distill_fwd.
#[derive(Clone, Copy)]
pub struct Distill<'a> {
    pub logits: &'a DeviceBuf,
    /// Logits and their tokens.
    pub teacher: Option<(&'a DeviceBuf, &'a TokenBuf)>,
    pub labels: Option<&'a TokenBuf>,
    pub weight: Option<&'a DeviceBuf>,
    pub temperature: f32,
    pub soft: f32,
    pub hard: f32,
    pub rows: usize,
    pub vocab: usize,
    pub top: usize,
}

impl Distill<'_> {
    fn check(&self) -> Result<(), CudaError> {
        length("logits", self.logits, self.rows * self.vocab)?;
        if let Some((teacher, index)) = self.teacher {
            length("teacher", teacher, self.rows * self.top)?;
            length("index", &index.words, self.rows * self.top)?;
        }
        if let Some(labels) = self.labels {
            length("labels", &labels.words, self.rows)?;
        }
        self.weight.map_or(Ok(()), |w| length("weight", w, self.rows))
    }
    fn top(&self) -> usize {
        self.teacher.map_or(0, |_| self.top)
    }
}

/// loss [rows].
pub fn distill_forward(ctx: &Context, d: &Distill<'_>, loss: &mut DeviceBuf) -> Result<(), CudaError> {
    d.check()?;
    length("loss", loss, d.rows)?;
    check(unsafe {
        ffi::katsu_cuda_distill_fwd(ctx.ptr(), d.logits.ptr, opt_const(d.teacher.map(|t| t.0)), opt_tokens(d.teacher.map(|t| t.1)),
                                    opt_tokens(d.labels), opt_const(d.weight), d.temperature, d.soft, d.hard, loss.ptr, d.rows, d.vocab, d.top())
    })
}

/// dlogits (+)= gradient of the sum of grad * loss; `loss` is written too where it is given, from the same reading of the logits.
pub fn distill_backward(ctx: &Context, d: &Distill<'_>, grad: Option<&DeviceBuf>, loss: Option<&mut DeviceBuf>, dlogits: &mut DeviceBuf,
                        accumulate: bool) -> Result<(), CudaError> {
    d.check()?;
    for buf in [grad, loss.as_deref()].into_iter().flatten() {
        length("grad or loss", buf, d.rows)?;
    }
    length("dlogits", dlogits, d.rows * d.vocab)?;
    check(unsafe {
        ffi::katsu_cuda_distill_bwd(ctx.ptr(), d.logits.ptr, opt_const(d.teacher.map(|t| t.0)), opt_tokens(d.teacher.map(|t| t.1)),
                                    opt_tokens(d.labels), opt_const(d.weight), d.temperature, d.soft, d.hard, opt_const(grad), opt_mut(loss),
                                    dlogits.ptr, d.rows, d.vocab, d.top(), accumulate as i32)
    })
}

/// What `adjust_logits` does to every row of logits; `None` leaves a part out.
#[derive(Clone, Copy, Default)]
pub struct LogitAdjustments<'a> {
    /// Tokens [rows, history_cols], and how many of a row's there are and are its prompt.
    pub history: Option<&'a TokenBuf>,
    pub lengths: Option<&'a TokenBuf>,
    pub prompts: Option<&'a TokenBuf>,
    pub repetition: Option<&'a DeviceBuf>,
    pub presence: Option<&'a DeviceBuf>,
    pub frequency: Option<&'a DeviceBuf>,
    /// Tokens and values [rows, biases].
    pub bias: Option<(&'a TokenBuf, &'a DeviceBuf)>,
    /// Bits in words [rows, (vocab + 31) / 32].
    pub allowed: Option<&'a TokenBuf>,
}

/// out = the logits [rows, vocab] behind penalties, biases and mask (katsu_cuda_adjust_logits).
pub fn adjust_logits(ctx: &Context, logits: &DeviceBuf, a: &LogitAdjustments<'_>, out: &mut DeviceBuf, rows: usize, vocab: usize)
                     -> Result<(), CudaError> {
    length("logits", logits, rows * vocab)?;
    length("out", out, rows * vocab)?;
    for tokens in [a.lengths, a.prompts].into_iter().flatten() {
        length("lengths or prompts", &tokens.words, rows)?;
    }
    for buf in [a.repetition, a.presence, a.frequency].into_iter().flatten() {
        length("penalties", buf, rows)?;
    }
    let of_row = |len: usize| if rows == 0 { 0 } else { len / rows };
    let (cols, biases) = (a.history.map_or(0, |h| of_row(h.len())), a.bias.map_or(0, |b| of_row(b.1.len())));
    if let Some(h) = a.history {
        length("history", &h.words, rows * cols)?;
    }
    if let Some((tokens, values)) = a.bias {
        length("bias", values, rows * biases)?;
        length("bias tokens", &tokens.words, rows * biases)?;
    }
    if let Some(words) = a.allowed {
        length("allowed", &words.words, rows * ((vocab + 31) / 32))?;
    }
    check(unsafe {
        ffi::katsu_cuda_adjust_logits(ctx.ptr(), logits.ptr, opt_tokens(a.history), opt_tokens(a.prompts), opt_tokens(a.lengths),
                                      opt_const(a.repetition), opt_const(a.presence), opt_const(a.frequency), opt_tokens(a.bias.map(|b| b.0)),
                                      opt_const(a.bias.map(|b| b.1)), opt_tokens(a.allowed) as *const u32, out.ptr, rows, vocab, cols, biases)
    })
}

/// The norm over all gradients into a one-element buffer.
pub fn grad_norm(ctx: &Context, grads: &[&DeviceBuf], norm: &mut DeviceBuf) -> Result<(), CudaError> {
    length("norm", norm, 1)?;
    let (g, counts): (Vec<*const f32>, Vec<usize>) = grads.iter().map(|b| (b.ptr as *const f32, b.len)).unzip();
    check(unsafe { ffi::katsu_cuda_grad_norm(ctx.ptr(), g.as_ptr(), counts.as_ptr(), g.len(), norm.ptr) })
}

/// Scales the gradients in place so that their norm is at most `max_norm`; `norm` receives it as it was.
pub fn clip_grads(ctx: &Context, grads: &mut [&mut DeviceBuf], max_norm: f32, norm: &mut DeviceBuf) -> Result<(), CudaError> {
    length("norm", norm, 1)?;
    let out: Vec<*mut f32> = grads.iter().map(|b| b.ptr).collect();
    let g: Vec<*const f32> = out.iter().map(|p| *p as *const f32).collect();
    let counts: Vec<usize> = grads.iter().map(|b| b.len).collect();
    check(unsafe { ffi::katsu_cuda_clip_grads(ctx.ptr(), g.as_ptr(), out.as_ptr(), counts.as_ptr(), g.len(), max_norm, norm.ptr) })
}

/// `clip_grads` and `sgd_step` of all weights in one, the gradients left as they are.
pub fn sgd_step_clipped(ctx: &Context, weights: &mut [&mut DeviceBuf], grads: &[&DeviceBuf], lr: f32, max_norm: f32,
                        norm: &mut DeviceBuf) -> Result<(), CudaError> {
    length("norm", norm, 1)?;
    if weights.len() != grads.len() {
        return Err(CudaError { code: ffi::KATSU_ERR_INVALID_ARG, message: "as many weights as gradients".to_string() });
    }
    for (w, g) in weights.iter().zip(grads) {
        length("gradient", g, w.len)?;
    }
    let w: Vec<*mut f32> = weights.iter().map(|b| b.ptr).collect();
    let (g, counts): (Vec<*const f32>, Vec<usize>) = grads.iter().map(|b| (b.ptr as *const f32, b.len)).unzip();
    check(unsafe {
        ffi::katsu_cuda_sgd_step_clipped(ctx.ptr(), w.as_ptr(), g.as_ptr(), counts.as_ptr(), g.len(), lr, max_norm, norm.ptr)
    })
}

/// Data-parallel gradient exchange: one process per GPU, images sharded over ranks, only parameter
/// gradients cross devices (dW sums over the batch, conv2d.rs:289).
pub struct Comm {
    ctx: Context,
}

impl Comm {
    /// Rank 0 creates the id and ships its bytes to the other ranks by any means.
    pub fn unique_id() -> Result<[u8; ffi::KATSU_COMM_ID_BYTES], CudaError> {
        let mut id = [0u8; ffi::KATSU_COMM_ID_BYTES];
        check(unsafe { ffi::katsu_cuda_comm_unique_id(id.as_mut_ptr()) })?;
        Ok(id)
    }

    pub fn init(ctx: &Context, id: &[u8; ffi::KATSU_COMM_ID_BYTES], n_ranks: usize, rank: usize) -> Result<Self, CudaError> {
        check(unsafe { ffi::katsu_cuda_comm_init(ctx.ptr(), id.as_ptr(), n_ranks as i32, rank as i32) })?;
        Ok(Self { ctx: ctx.clone() })
    }

    /// In-place sum over all ranks of a flat gradient bucket, ordered on the context's stream.
    pub fn allreduce_sum(&self, bucket: &mut DeviceBuf) -> Result<(), CudaError> {
        check(unsafe { ffi::katsu_cuda_allreduce_sum(self.ctx.ptr(), bucket.ptr, bucket.len) })
    }
}

impl Drop for Comm {
    fn drop(&mut self) {
        unsafe { ffi::katsu_cuda_comm_destroy(self.ctx.ptr()) };
    }
}

/// A CUDA event on the context's stream, for timing and for ordering two contexts of one device.
pub struct Event {
    ctx: Context,
    raw: *mut ffi::Event,
}

impl Event {
    pub fn new(ctx: &Context) -> Result<Self, CudaError> {
        let mut raw = ptr::null_mut();
        check(unsafe { ffi::katsu_cuda_event_create(ctx.ptr(), &mut raw) })?;
        Ok(Self { ctx: ctx.clone(), raw })
    }
    pub fn record(&self) -> Result<(), CudaError> {
        check(unsafe { ffi::katsu_cuda_event_record(self.ctx.ptr(), self.raw) })
    }
    /// Makes `waiter`'s later work wait on the device for this event; the host does not block.
    pub fn make_wait(&self, waiter: &Context) -> Result<(), CudaError> {
        check(unsafe { ffi::katsu_cuda_wait_event(waiter.ptr(), self.raw) })
    }
    pub fn elapsed_ms(&self, stop: &Event) -> Result<f32, CudaError> {
        let mut ms = 0.0f32;
        check(unsafe { ffi::katsu_cuda_event_elapsed_ms(self.ctx.ptr(), self.raw, stop.raw, &mut ms) })?;
        Ok(ms)
    }
}

impl Drop for Event {
    fn drop(&mut self) {
        unsafe { ffi::katsu_cuda_event_destroy(self.ctx.ptr(), self.raw) };
    }
}
