//! Raw bindings of `include/nne_cuda.h`: one declaration per exported symbol, nothing else.
//! GENERATED by `gen_ffi.py` from the header - edit the header, then run the generator.
#![allow(non_camel_case_types)]
use std::os::raw::{c_char, c_int, c_uint, c_void};

#[repr(C)]
pub struct nne_ctx {
    _private: [u8; 0],
}
#[repr(C)]
pub struct nne_qlinear {
    _private: [u8; 0],
}
#[repr(C)]
pub struct nne_qlinear4 {
    _private: [u8; 0],
}
#[repr(C)]
pub struct nne_kv_cache {
    _private: [u8; 0],
}
#[repr(C)]
pub struct nne_plan {
    _private: [u8; 0],
}
#[repr(C)]
pub struct nne_shard_group {
    _private: [u8; 0],
}

/// One forward of a fused plan (`nne_plan_item`).
#[repr(C)]
#[derive(Clone, Copy)]
pub struct nne_plan_item {
    pub layer: *mut nne_qlinear,
    pub x: *const f32,
    pub y: *mut f32,
    pub input_op: c_int,
    pub eps: f32,
    pub gamma: *const f32,
    pub x2: *const f32,
    pub residual: *const f32,
}

/// `nne_kv_cache_desc`.
#[repr(C)]
#[derive(Clone, Copy)]
pub struct nne_kv_cache_desc {
    pub k_pages: *mut c_void,
    pub v_pages: *mut c_void,
    pub pages: usize,
    pub page_size: c_int,
    pub kv_heads: c_int,
    pub head_dim: c_int,
    pub dtype: c_int,
    pub rope_dims: c_int,
    pub rope_interleaved: c_int,
    pub rope_base: f64,
    pub rope_freq: *const f64,
}

/// `nne_kv_append`.
#[repr(C)]
#[derive(Clone, Copy)]
pub struct nne_kv_append {
    pub q: *const f32,
    pub k: *const f32,
    pub v: *const f32,
    pub q_out: *mut f32,
    pub q_stride: usize,
    pub k_stride: usize,
    pub v_stride: usize,
    pub tokens: usize,
    pub q_heads: c_int,
    pub eps: f32,
    pub q_gamma: *const f32,
    pub k_gamma: *const f32,
    pub page_table: *const i32,
    pub table_stride: usize,
    pub sequences: c_int,
    pub sequence: *const i32,
    pub index: *const i32,
    pub position: *const i32,
}

/// `nne_tree_attention`.
#[repr(C)]
#[derive(Clone, Copy)]
pub struct nne_tree_attention {
    pub q: *const f32,
    pub out: *mut f32,
    pub q_stride: usize,
    pub out_stride: usize,
    pub tokens: usize,
    pub q_heads: c_int,
    pub sequences: c_int,
    pub max_nodes: c_int,
    pub max_context: c_int,
    pub scale: f32,
    pub node_start: *const i32,
    pub context: *const i32,
    pub visible: *const u64,
    pub page_table: *const i32,
    pub table_stride: usize,
}

/// `nne_sample`.
#[repr(C)]
#[derive(Clone, Copy)]
pub struct nne_sample {
    pub logits: *const f32,
    pub row_stride: usize,
    pub rows: usize,
    pub vocab: usize,
    pub temperature: *const f32,
    pub top_k: *const i32,
    pub top_p: *const f32,
    pub min_p: *const f32,
    pub uniform: *const f32,
    pub tokens: *mut i32,
}

pub const NNE_OK: c_int = 0;
pub const NNE_ERR_INVALID_ARGUMENT: c_int = 1;
pub const NNE_ERR_SHAPE_MISMATCH: c_int = 2;
pub const NNE_ERR_CUDA: c_int = 3;
pub const NNE_ERR_NCCL: c_int = 4;
pub const NNE_ERR_TIMEOUT: c_int = 5;
pub const NNE_ERR_OUT_OF_MEMORY: c_int = 6;
pub const NNE_ERR_UNSUPPORTED: c_int = 7;
pub const NNE_INPUT_PLAIN: c_int = 0;
pub const NNE_INPUT_RMSNORM: c_int = 1;
pub const NNE_INPUT_SILU_MUL: c_int = 2;
pub const NNE_F16: c_int = 1;
pub const NNE_BF16: c_int = 2;
pub const NNE_SHARD_HANDLE_BYTES: usize = 64;

extern "C" {
    pub fn nne_status_string(status: c_int) -> *const c_char;
    pub fn nne_last_error(buf: *mut c_char, n: usize) -> c_int;
    pub fn nne_cuda_ctx_create(device: c_int, out: *mut *mut nne_ctx) -> c_int;
    pub fn nne_cuda_ctx_destroy(ctx: *mut nne_ctx) -> c_int;
    pub fn nne_cuda_ctx_check(ctx: *mut nne_ctx) -> c_int;
    pub fn nne_cuda_ctx_selftest_wait(ctx: *mut nne_ctx, which: c_int, limit_us: c_uint) -> c_int;
    pub fn nne_cuda_ctx_reserve_sms(ctx: *mut nne_ctx, count: c_int) -> c_int;
    pub fn nne_cuda_ctx_info(
        ctx: *const nne_ctx,
        device: *mut c_int,
        sm_count: *mut c_int,
        cc_major: *mut c_int,
        cc_minor: *mut c_int,
        total_mem_bytes: *mut usize,
    ) -> c_int;
    pub fn nne_device_alloc(ctx: *mut nne_ctx, bytes: usize, out_dev: *mut *mut c_void) -> c_int;
    pub fn nne_device_free(ctx: *mut nne_ctx, ptr_dev: *mut c_void) -> c_int;
    pub fn nne_device_upload(
        ctx: *mut nne_ctx,
        dst_dev: *mut c_void,
        src_host: *const c_void,
        bytes: usize,
    ) -> c_int;
    pub fn nne_device_download(
        ctx: *mut nne_ctx,
        dst_host: *mut c_void,
        src_dev: *const c_void,
        bytes: usize,
    ) -> c_int;
    pub fn nne_cuda_ctx_stream(ctx: *mut nne_ctx) -> *mut c_void;
    pub fn nne_quantize_rows(
        ctx: *mut nne_ctx,
        w_host: *const f32,
        rows: usize,
        cols: usize,
        q_host: *mut i8,
        scales_host: *mut f32,
    ) -> c_int;
    pub fn nne_quantize_rows_dev(
        ctx: *mut nne_ctx,
        w_dev: *const f32,
        rows: usize,
        cols: usize,
        q_dev: *mut i8,
        scales_dev: *mut f32,
        stream: *mut c_void,
    ) -> c_int;
    pub fn nne_quantize_tensor(
        ctx: *mut nne_ctx,
        v_host: *const f32,
        n: usize,
        q_host: *mut i8,
        scale_out: *mut f32,
    ) -> c_int;
    pub fn nne_quantize_tensor_dev(
        ctx: *mut nne_ctx,
        v_dev: *const f32,
        n: usize,
        q_dev: *mut i8,
        scale_dev: *mut f32,
        stream: *mut c_void,
    ) -> c_int;
    pub fn nne_dequantize_rows(
        ctx: *mut nne_ctx,
        q_host: *const i8,
        scales_host: *const f32,
        rows: usize,
        cols: usize,
        out_host: *mut f32,
    ) -> c_int;
    pub fn nne_dequantize_rows_dev(
        ctx: *mut nne_ctx,
        q_dev: *const i8,
        scales_dev: *const f32,
        rows: usize,
        cols: usize,
        out_dev: *mut f32,
        stream: *mut c_void,
    ) -> c_int;
    pub fn nne_qlinear_create_from_f32(
        ctx: *mut nne_ctx,
        w_host: *const f32,
        bias_host_or_null: *const f32,
        n: usize,
        k: usize,
        out: *mut *mut nne_qlinear,
    ) -> c_int;
    pub fn nne_qlinear_create_from_f32_dev(
        ctx: *mut nne_ctx,
        w_dev: *const f32,
        bias_dev_or_null: *const f32,
        n: usize,
        k: usize,
        stream: *mut c_void,
        out: *mut *mut nne_qlinear,
    ) -> c_int;
    pub fn nne_qlinear_create_from_i8(
        ctx: *mut nne_ctx,
        q_host: *const i8,
        scales_host: *const f32,
        bias_host_or_null: *const f32,
        n: usize,
        k: usize,
        out: *mut *mut nne_qlinear,
    ) -> c_int;
    pub fn nne_qlinear_destroy(ql: *mut nne_qlinear) -> c_int;
    pub fn nne_qlinear_download(ql: *const nne_qlinear, q_host: *mut i8, scales_host: *mut f32) -> c_int;
    pub fn nne_qlinear_info(
        ql: *const nne_qlinear,
        n: *mut usize,
        k: *mut usize,
        has_bias: *mut c_int,
        q_dev: *mut *const i8,
        scales_dev: *mut *const f32,
        bias_dev: *mut *const f32,
    ) -> c_int;
    pub fn nne_qlinear_memory_bytes(ql: *const nne_qlinear) -> usize;
    pub fn nne_qlinear_forward_host(
        ql: *mut nne_qlinear,
        x_host: *const f32,
        m: usize,
        k: usize,
        y_host: *mut f32,
    ) -> c_int;
    pub fn nne_qlinear_forward_dev(
        ql: *mut nne_qlinear,
        x_dev: *const f32,
        m: usize,
        k: usize,
        y_dev: *mut f32,
        stream: *mut c_void,
    ) -> c_int;
    pub fn nne_qlinear_forward_dev_strided(
        ql: *mut nne_qlinear,
        x_dev: *const f32,
        m: usize,
        k: usize,
        y_dev: *mut f32,
        ldy: usize,
        stream: *mut c_void,
    ) -> c_int;
    pub fn nne_qlinear_forward_dev_static(
        ql: *mut nne_qlinear,
        x_dev: *const f32,
        m: usize,
        k: usize,
        y_dev: *mut f32,
        stream: *mut c_void,
    ) -> c_int;
    pub fn nne_qlinear_plan_create(
        ctx: *mut nne_ctx,
        count: usize,
        layers: *const *mut nne_qlinear,
        x_dev: *const *const f32,
        y_dev: *const *mut f32,
        m: usize,
        out: *mut *mut nne_plan,
    ) -> c_int;
    pub fn nne_qlinear_plan_run(plan: *mut nne_plan, stream: *mut c_void) -> c_int;
    pub fn nne_qlinear_plan_run_host(
        plan: *mut nne_plan,
        x_all_host: *const f32,
        y_all_host: *mut f32,
    ) -> c_int;
    pub fn nne_qlinear_plan_destroy(plan: *mut nne_plan) -> c_int;
    pub fn nne_qlinear_plan_launches(plan: *const nne_plan) -> c_int;
    pub fn nne_rmsnorm_dev(
        ctx: *mut nne_ctx,
        x_dev: *const f32,
        gamma_dev: *const f32,
        eps: f32,
        rows: usize,
        cols: usize,
        y_dev: *mut f32,
        stream: *mut c_void,
    ) -> c_int;
    pub fn nne_silu_mul_dev(
        ctx: *mut nne_ctx,
        gate_dev: *const f32,
        up_dev: *const f32,
        n: usize,
        out_dev: *mut f32,
        stream: *mut c_void,
    ) -> c_int;
    pub fn nne_add_dev(
        ctx: *mut nne_ctx,
        a_dev: *const f32,
        b_dev: *const f32,
        n: usize,
        out_dev: *mut f32,
        stream: *mut c_void,
    ) -> c_int;
    pub fn nne_qlinear_plan_create_fused(
        ctx: *mut nne_ctx,
        count: usize,
        items: *const nne_plan_item,
        m: usize,
        out: *mut *mut nne_plan,
    ) -> c_int;
    pub fn nne_quantize_rows4_dev(
        ctx: *mut nne_ctx,
        w_dev: *const f32,
        rows: usize,
        cols: usize,
        group: usize,
        q_dev: *mut u8,
        scales_dev: *mut f32,
        stream: *mut c_void,
    ) -> c_int;
    pub fn nne_qlinear4_create_from_f32(
        ctx: *mut nne_ctx,
        w_host: *const f32,
        bias_host_or_null: *const f32,
        n: usize,
        k: usize,
        group: usize,
        out: *mut *mut nne_qlinear4,
    ) -> c_int;
    pub fn nne_qlinear4_create_from_f32_dev(
        ctx: *mut nne_ctx,
        w_dev: *const f32,
        bias_dev_or_null: *const f32,
        n: usize,
        k: usize,
        group: usize,
        stream: *mut c_void,
        out: *mut *mut nne_qlinear4,
    ) -> c_int;
    pub fn nne_qlinear4_create_from_i4(
        ctx: *mut nne_ctx,
        q_host: *const u8,
        scales_host: *const f32,
        bias_host_or_null: *const f32,
        n: usize,
        k: usize,
        group: usize,
        out: *mut *mut nne_qlinear4,
    ) -> c_int;
    pub fn nne_qlinear4_create_from_i4_dev(
        ctx: *mut nne_ctx,
        q_dev: *const u8,
        scales_dev: *const f32,
        bias_dev_or_null: *const f32,
        n: usize,
        k: usize,
        group: usize,
        stream: *mut c_void,
        out: *mut *mut nne_qlinear4,
    ) -> c_int;
    pub fn nne_qlinear4_destroy(ql: *mut nne_qlinear4) -> c_int;
    pub fn nne_qlinear4_download(
        ql: *const nne_qlinear4,
        q_host: *mut u8,
        scales_host: *mut f32,
        bias_host: *mut f32,
    ) -> c_int;
    pub fn nne_qlinear4_dequantize(ql: *const nne_qlinear4, w_host: *mut f32) -> c_int;
    pub fn nne_qlinear4_info(
        ql: *const nne_qlinear4,
        n: *mut usize,
        k: *mut usize,
        group: *mut usize,
        has_bias: *mut c_int,
    ) -> c_int;
    pub fn nne_qlinear4_memory_bytes(ql: *const nne_qlinear4) -> usize;
    pub fn nne_qlinear4_forward_host(
        ql: *mut nne_qlinear4,
        x_host: *const f32,
        m: usize,
        k: usize,
        y_host: *mut f32,
    ) -> c_int;
    pub fn nne_qlinear4_forward_dev(
        ql: *mut nne_qlinear4,
        x_dev: *const f32,
        m: usize,
        k: usize,
        y_dev: *mut f32,
        stream: *mut c_void,
    ) -> c_int;
    pub fn nne_qlinear4_forward_dev_strided(
        ql: *mut nne_qlinear4,
        x_dev: *const f32,
        m: usize,
        k: usize,
        y_dev: *mut f32,
        ldy: usize,
        stream: *mut c_void,
    ) -> c_int;
    pub fn nne_kv_cache_create(
        ctx: *mut nne_ctx,
        desc: *const nne_kv_cache_desc,
        out: *mut *mut nne_kv_cache,
    ) -> c_int;
    pub fn nne_kv_cache_destroy(cache: *mut nne_kv_cache) -> c_int;
    pub fn nne_kv_cache_info(
        cache: *const nne_kv_cache,
        k_pages: *mut *mut c_void,
        v_pages: *mut *mut c_void,
        bytes_each: *mut usize,
    ) -> c_int;
    pub fn nne_kv_append_dev(
        cache: *mut nne_kv_cache,
        args: *const nne_kv_append,
        stream: *mut c_void,
    ) -> c_int;
    pub fn nne_tree_attention_dev(
        cache: *mut nne_kv_cache,
        args: *const nne_tree_attention,
        stream: *mut c_void,
    ) -> c_int;
    pub fn nne_sample_dev(ctx: *mut nne_ctx, args: *const nne_sample, stream: *mut c_void) -> c_int;
    pub fn nne_shard_group_create(
        ctx: *mut nne_ctx,
        rank: c_int,
        world: c_int,
        window_bytes: usize,
        out: *mut *mut nne_shard_group,
    ) -> c_int;
    pub fn nne_shard_group_handle(group: *const nne_shard_group, handle_out: *mut c_void) -> c_int;
    pub fn nne_shard_group_connect(group: *mut nne_shard_group, all_handles: *const c_void) -> c_int;
    pub fn nne_shard_group_connect_local(
        group: *mut nne_shard_group,
        all_groups: *const *mut nne_shard_group,
    ) -> c_int;
    pub fn nne_shard_group_window(
        group: *const nne_shard_group,
        base: *mut *mut c_void,
        bytes: *mut usize,
    ) -> c_int;
    pub fn nne_shard_group_wait(group: *mut nne_shard_group, stream: *mut c_void) -> c_int;
    pub fn nne_shard_group_set_nccl(group: *mut nne_shard_group, nccl_comm: *mut c_void) -> c_int;
    pub fn nne_shard_group_destroy(group: *mut nne_shard_group) -> c_int;
    pub fn nne_qlinear_plan_create_sharded(
        group: *mut nne_shard_group,
        count: usize,
        shards: *const *mut nne_qlinear,
        row_begin: *const usize,
        n_total: *const usize,
        x_dev: *const *const f32,
        y_full_dev: *const *mut f32,
        m: usize,
        route: c_int,
        out: *mut *mut nne_plan,
    ) -> c_int;
    pub fn nne_qlinear_kernel_for(ql: *const nne_qlinear, m: usize) -> c_int;
    pub fn nne_launch_count() -> u64;
}
