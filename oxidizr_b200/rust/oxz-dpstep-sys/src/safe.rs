//! The thin safe layer over the raw declarations: what `LitTrainer` calls in place of boostr's `AdamW`, `GradScaler`,
//! `clip_grad_norm` and the communicator's collectives for the work after its micro-batch loop
//! (src/trainer.rs:515-695). Nothing here computes: every decision and all arithmetic is the library's.
//!
//! Mapping onto the reference's call sites:
//!   `FusedAdamW::with_param_groups` (src/trainer.rs:184-193)   -> `DpOptimizer::new` with `DecayRule::no_decay_mask`
//!   `optimizer.set_lr(lr_plan.lr_at(step))` (src/trainer.rs:254) -> `LrPlan::lr_at` + `StepHyper::lr`
//!   `reduce_step_gradients` + `unscale` + `clip_gradients` + target clip + `optimizer.step`
//!       (src/trainer.rs:520-527, 573-587, 635-649)               -> `DpOptimizer::step`, one call
//!   `diagnose_bad_gradients` (src/trainer.rs:990-1020)           -> `DpOptimizer::grad_norms_per_tensor`
//!   `scaler.record_step(overflow)` (src/trainer.rs:666-681)      -> `LossScaler::record_step`
//!   `metrics.judge(step, loss)` (src/trainer.rs:612)             -> `SpikeGuard::judge`
//!   `NcclCommunicator::from_streams` / `abort` (src/dp/launch.rs:82-103) -> `Communicator`
//!   `EpochOrder::row` with `epoch_permutation` (src/data/rows.rs:240-272) -> `Loader::set_row_order`
//!
//! What library-owned buffers cost the Rust side: the flat gradient and working-weight buffers belong to the plan
//! (`DpOptimizer::pointers`). Either the model's parameter tensors are created as views of `work + offsets[i]` (no copy,
//! the step's weights are in place when it returns) and backward writes into `grads + offsets[i]`, or the trainer keeps
//! its own tensors and pays `flatten_grads` (2 x gradient bytes of HBM traffic per step, measured 0.81 ms on the
//! 1.24 B-parameter set) plus one device copy of the weights back per step.
use crate as sys;
use std::ffi::{c_void, CStr, CString};
use std::os::raw::c_char;
use std::ptr;

/// A non-zero status with the library's message: the counterpart of `boostr::error::Error`.
#[derive(Debug, Clone)]
pub struct Error {
    pub status: i32,
    pub message: String,
}

impl std::fmt::Display for Error {
    fn fmt(&self, f: &mut std::fmt::Formatter<'_>) -> std::fmt::Result {
        write!(f, "oxz status {}: {}", self.status, self.message)
    }
}

impl std::error::Error for Error {}

pub type Result<T> = std::result::Result<T, Error>;

fn check(status: i32) -> Result<()> {
    if status == sys::OXZ_OK {
        return Ok(());
    }
    let message = unsafe { CStr::from_ptr(sys::oxz_last_error()) }.to_string_lossy().into_owned();
    Err(Error { status, message })
}

/// One rank's communicator. Dropping it destroys it; `abort` may be called from any thread
/// (src/dp/launch.rs:97-103, 142-150).
pub struct Communicator {
    raw: *mut sys::oxz_comm,
}

unsafe impl Send for Communicator {}
unsafe impl Sync for Communicator {}

impl Communicator {
    pub fn unique_id() -> Result<[u8; 128]> {
        let mut id = [0u8; 128];
        check(unsafe { sys::oxz_comm_unique_id(id.as_mut_ptr()) })?;
        Ok(id)
    }

    pub fn init_rank(device: i32, rank: i32, world: i32, id: &[u8; 128]) -> Result<Self> {
        let mut raw = ptr::null_mut();
        check(unsafe { sys::oxz_comm_init_rank(device, rank, world, id.as_ptr(), &mut raw) })?;
        Ok(Self { raw })
    }

    /// All communicators of a one-process group at once, as `from_streams` does (src/dp/launch.rs:82-95).
    pub fn init_all(devices: &[i32]) -> Result<Vec<Self>> {
        let mut raws = vec![ptr::null_mut(); devices.len()];
        check(unsafe { sys::oxz_comm_init_all(devices.len() as i32, devices.as_ptr(), raws.as_mut_ptr()) })?;
        Ok(raws.into_iter().map(|raw| Self { raw }).collect())
    }

    /// The in-process group with a collective timeout (boostr's `LocalCommunicator::with_timeout`).
    pub fn init_local(devices: &[i32], timeout_seconds: f64) -> Result<Vec<Self>> {
        let mut raws = vec![ptr::null_mut(); devices.len()];
        check(unsafe {
            sys::oxz_comm_init_local(devices.len() as i32, devices.as_ptr(), timeout_seconds, raws.as_mut_ptr())
        })?;
        Ok(raws.into_iter().map(|raw| Self { raw }).collect())
    }

    pub fn abort(&self) -> Result<()> {
        check(unsafe { sys::oxz_comm_abort(self.raw) })
    }

    pub fn barrier(&self) -> Result<()> {
        check(unsafe { sys::oxz_barrier(self.raw) })
    }

    /// The step-weighting collective (src/dp/weighting.rs:63-101): (scored tokens, masked ranks) summed over ranks.
    pub fn sum_counts(&self, scored: i64, masked_ranks: i64) -> Result<(i64, i64)> {
        let mut v = [scored, masked_ranks];
        check(unsafe { sys::oxz_allreduce_i64x2(self.raw, v.as_mut_ptr()) })?;
        Ok((v[0], v[1]))
    }

    pub fn broadcast(&self, device_ptr: *mut c_void, bytes: u64, root: i32) -> Result<()> {
        check(unsafe { sys::oxz_broadcast(self.raw, device_ptr, bytes, root) })
    }

    pub fn as_raw(&self) -> *mut sys::oxz_comm {
        self.raw
    }
}

impl Drop for Communicator {
    fn drop(&mut self) {
        unsafe { sys::oxz_comm_destroy(self.raw) };
    }
}

/// `WeightDecaySpec` (src/weight_decay/rule.rs:49-118).
pub struct DecayRule {
    pub rule: i32,
    pub no_decay_patterns: Vec<CString>,
}

impl DecayRule {
    /// `DecayPlan::param_groups` (src/weight_decay/plan.rs:113-122): 1 = member of the zero-decay group.
    pub fn no_decay_mask(&self, names_and_ranks: &[(&str, u32)]) -> Result<Vec<u8>> {
        let patterns: Vec<*const c_char> = self.no_decay_patterns.iter().map(|p| p.as_ptr() as *const c_char).collect();
        let mut mask = Vec::with_capacity(names_and_ranks.len());
        for (name, rank) in names_and_ranks {
            let name = CString::new(*name).expect("a checkpoint name holds no NUL");
            let mut excluded = 0i32;
            check(unsafe {
                sys::oxz_decay_excludes(
                    self.rule,
                    patterns.as_ptr(),
                    patterns.len() as u32,
                    name.as_ptr(),
                    *rank,
                    &mut excluded,
                )
            })?;
            mask.push(excluded as u8);
        }
        Ok(mask)
    }
}

/// `LrPlan::lr_at` (src/schedule.rs:177-183).
pub fn lr_at(plan: &sys::oxz_lr_plan, step: u64) -> Result<f64> {
    let mut lr = 0.0;
    check(unsafe { sys::oxz_lr_at(plan, step, &mut lr) })?;
    Ok(lr)
}

/// `LossScaler` (src/loss_scale/scaler.rs:13-51) over the library's state machine.
pub struct LossScaler {
    pub config: sys::oxz_scaler_config,
    pub state: sys::oxz_scaler_state,
}

impl LossScaler {
    pub fn new(config: sys::oxz_scaler_config) -> Result<Self> {
        let mut state = sys::oxz_scaler_state { scale: 0.0, consecutive_ok: 0 };
        check(unsafe { sys::oxz_scaler_init(&config, &mut state) })?;
        Ok(Self { config, state })
    }

    pub fn scale(&self) -> f64 {
        self.state.scale
    }

    /// The update at the end of a step (src/trainer.rs:666-681): untouched on a finite-gradient spike skip.
    pub fn record_step(&mut self, overflow: bool, spike_skip: bool) -> Result<()> {
        check(unsafe { sys::oxz_scaler_record_step(&self.config, &mut self.state, overflow as i32, spike_skip as i32) })
    }
}

/// `TrainMetrics::judge` over `SpikeGuard::observe` (src/metrics/state.rs:79-86).
pub struct SpikeGuard {
    pub config: sys::oxz_spike_config,
    pub state: sys::oxz_spike_state,
}

impl SpikeGuard {
    /// true: the step must skip the optimizer.
    pub fn judge(&mut self, index: u64, loss: f64) -> Result<bool> {
        let (mut skip, mut flagged) = (0i32, 0i32);
        check(unsafe { sys::oxz_spike_judge(&self.config, &mut self.state, index, loss, &mut skip, &mut flagged) })?;
        Ok(skip != 0)
    }
}

/// Device addresses of the plan's flat buffers.
pub struct StatePointers {
    pub grads: *mut c_void,
    pub work: *mut c_void,
    pub master: *mut c_void,
    pub exp_avg: *mut c_void,
    pub exp_avg_sq: *mut c_void,
}

/// The optimizer of one rank: boostr's `FusedAdamW` plus the collectives and clips around its step.
pub struct DpOptimizer {
    raw: *mut sys::oxz_plan,
    comm: *mut sys::oxz_comm,
    n_tensors: usize,
}

unsafe impl Send for DpOptimizer {}

impl DpOptimizer {
    /// `numel` keeps `parameter_ids` order (src/trainer.rs:208); `no_decay` comes from `DecayRule::no_decay_mask`.
    pub fn new(
        numel: &[u64],
        no_decay: &[u8],
        grad_dtype: i32,
        param_dtype: i32,
        world: i32,
        rank: i32,
        device: i32,
        comm: Option<&Communicator>,
    ) -> Result<Self> {
        let desc = sys::oxz_plan_desc {
            n_tensors: numel.len() as u64,
            numel: numel.as_ptr(),
            no_decay: no_decay.as_ptr(),
            lr_scale: ptr::null(),
            grad_dtype,
            param_dtype,
            world,
            rank,
            sync_mode: if world == 1 { sys::OXZ_SYNC_SINGLE } else { sys::OXZ_SYNC_P2P },
            device,
            bucket_bytes: 0,
        };
        let mut raw = ptr::null_mut();
        check(unsafe { sys::oxz_plan_create(&desc, &mut raw) })?;
        let comm = comm.map_or(ptr::null_mut(), |c| c.as_raw());
        let this = Self { raw, comm, n_tensors: numel.len() };
        check(unsafe { sys::oxz_state_alloc(this.raw, this.comm) })?;
        Ok(this)
    }

    pub fn pointers(&self) -> Result<StatePointers> {
        let mut p = StatePointers {
            grads: ptr::null_mut(),
            work: ptr::null_mut(),
            master: ptr::null_mut(),
            exp_avg: ptr::null_mut(),
            exp_avg_sq: ptr::null_mut(),
        };
        check(unsafe {
            sys::oxz_state_pointers(self.raw, &mut p.grads, &mut p.work, &mut p.master, &mut p.exp_avg, &mut p.exp_avg_sq)
        })?;
        Ok(p)
    }

    pub fn tensor_offsets(&self) -> Result<Vec<u64>> {
        let mut offsets = vec![0u64; self.n_tensors];
        check(unsafe { sys::oxz_plan_tensor_offsets(self.raw, offsets.as_mut_ptr()) })?;
        Ok(offsets)
    }

    /// `GradStore` -> flat buffer; `None` = this rank has no gradient for the tensor (its span is zero-filled);
    /// `accumulate` adds instead of storing, the micro-batch accumulation of src/trainer.rs:1087-1107.
    pub fn flatten_grads(&mut self, grads: &[Option<*const c_void>], accumulate: bool) -> Result<()> {
        let ptrs: Vec<*const c_void> = grads.iter().map(|g| g.unwrap_or(ptr::null())).collect();
        check(unsafe { sys::oxz_grads_flatten_async(self.raw, ptrs.as_ptr(), accumulate as i32) })
    }

    /// src/trainer.rs:520-661 in one call. `present[i] = 0`: this rank produced no gradient for tensor i; the library
    /// forms the union over ranks. `loss` comes back summed over ranks (the `extras` of `all_reduce_flat_sum`).
    pub fn step(&mut self, hyper: &sys::oxz_hyper, present: Option<&[u8]>, loss: &mut f64) -> Result<sys::oxz_step_result> {
        let mut result = sys::oxz_step_result {
            grad_norm: 0.0,
            reported_norm: 0.0,
            clip_coef: 1.0,
            overflow: 0,
            applied: 0,
            timestep: 0,
        };
        check(unsafe {
            sys::oxz_step(self.raw, self.comm, hyper, present.map_or(ptr::null(), |p| p.as_ptr()), loss, 1, &mut result)
        })?;
        Ok(result)
    }

    /// `grad_norm_for_tensor` for every parameter (src/trainer.rs:933-937); -1 marks a tensor no rank had a gradient for.
    pub fn grad_norms_per_tensor(&mut self, loss_scale: f64, max_grad_value: f64) -> Result<Vec<f64>> {
        let mut norms = vec![0.0f64; self.n_tensors];
        check(unsafe { sys::oxz_grad_norms_per_tensor(self.raw, self.comm, loss_scale, max_grad_value, norms.as_mut_ptr()) })?;
        Ok(norms)
    }

    /// `optimizer_timestep` (src/trainer.rs:906-908).
    pub fn timestep(&self) -> Result<u64> {
        let mut t = 0u64;
        check(unsafe { sys::oxz_state_timestep(self.raw, &mut t) })?;
        Ok(t)
    }

    pub fn set_timestep(&mut self, applied_steps: u64) -> Result<()> {
        check(unsafe { sys::oxz_state_set_timestep(self.raw, applied_steps) })
    }

    /// The optimizer file of a checkpoint set (src/checkpoint_set/optimizer_io.rs:62-74). Collective; rank 0 writes.
    pub fn save(&mut self, path: &str, names: &[&str], shapes: &[Vec<u64>]) -> Result<()> {
        let (c_names, ptrs, ndim, dims) = names_and_shapes(names, shapes);
        let path = CString::new(path).expect("a path holds no NUL");
        let r = check(unsafe {
            sys::oxz_optimizer_save(self.raw, self.comm, path.as_ptr(), ptrs.as_ptr(), ndim.as_ptr(), dims.as_ptr())
        });
        drop(c_names);
        r
    }

    pub fn load(&mut self, path: &str, names: &[&str], shapes: &[Vec<u64>]) -> Result<()> {
        let (c_names, ptrs, ndim, dims) = names_and_shapes(names, shapes);
        let path = CString::new(path).expect("a path holds no NUL");
        let r = check(unsafe { sys::oxz_optimizer_load(self.raw, path.as_ptr(), ptrs.as_ptr(), ndim.as_ptr(), dims.as_ptr()) });
        drop(c_names);
        r
    }
}

impl Drop for DpOptimizer {
    fn drop(&mut self) {
        unsafe { sys::oxz_plan_destroy(self.raw) };
    }
}

fn names_and_shapes(names: &[&str], shapes: &[Vec<u64>]) -> (Vec<CString>, Vec<*const c_char>, Vec<u32>, Vec<u64>) {
    let c_names: Vec<CString> = names.iter().map(|n| CString::new(*n).expect("a checkpoint name holds no NUL")).collect();
    let ptrs = c_names.iter().map(|n| n.as_ptr() as *const c_char).collect();
    let ndim = shapes.iter().map(|s| s.len() as u32).collect();
    let dims = shapes.iter().flatten().copied().collect();
    (c_names, ptrs, ndim, dims)
}

/// The rank-sliced loader (src/data/ranks.rs:25-41, src/data/positioning.rs:44-68).
pub struct Loader {
    raw: *mut sys::oxz_loader,
}

impl Loader {
    pub fn open(path: &str, seq_len: u64, rank_batch_size: u64, rank: u64, world: u64, device: i32) -> Result<Self> {
        let path = CString::new(path).expect("a path holds no NUL");
        let mut raw = ptr::null_mut();
        check(unsafe { sys::oxz_loader_open(path.as_ptr(), seq_len, rank_batch_size, rank, world, 0, 0, device, &mut raw) })?;
        Ok(Self { raw })
    }

    /// `with_row_order(RowOrder::Shuffled { seed })` (src/data/construction.rs:140): hand over
    /// `epoch_permutation(num_rows, seed, epoch)` (src/data/rows.rs:258-263) for the current epoch and the next one.
    pub fn set_row_order(&mut self, epoch: u64, perm: &[u32]) -> Result<()> {
        check(unsafe { sys::oxz_loader_set_row_order(self.raw, epoch, perm.as_ptr(), perm.len() as u64) })
    }

    /// Device pointers to `[rank_batch_size, seq_len]` i64 inputs and targets, valid until the second-next call.
    pub fn next_batch(&mut self, stream: *mut c_void, rows: &mut [u64]) -> Result<(*mut i64, *mut i64)> {
        let (mut inputs, mut targets) = (ptr::null_mut(), ptr::null_mut());
        check(unsafe { sys::oxz_loader_next_batch_async(self.raw, stream, &mut inputs, &mut targets, rows.as_mut_ptr()) })?;
        Ok((inputs, targets))
    }

    pub fn position(&self) -> Result<sys::oxz_data_position> {
        let mut pos = sys::oxz_data_position { epoch: 0, row: 0 };
        check(unsafe { sys::oxz_loader_position(self.raw, &mut pos) })?;
        Ok(pos)
    }

    pub fn seek(&mut self, pos: sys::oxz_data_position) -> Result<()> {
        check(unsafe { sys::oxz_loader_seek(self.raw, pos) })
    }
}

impl Drop for Loader {
    fn drop(&mut self) {
        unsafe { sys::oxz_loader_close(self.raw) };
    }
}

/// The token embedding and its gradient (embed_tokens, src/model.rs:3905-3953). Pointers are device memory.
pub struct TokenEmbedding {
    raw: *mut sys::oxz_embed,
}

impl TokenEmbedding {
    pub fn new(desc: &sys::oxz_embed_desc) -> Result<Self> {
        let mut raw = ptr::null_mut();
        check(unsafe { sys::oxz_embed_create(desc, &mut raw) })?;
        let this = Self { raw };
        check(unsafe { sys::oxz_embed_alloc(this.raw, ptr::null_mut()) })?;
        Ok(this)
    }

    /// # Safety
    /// `ids`, `table` and `out` are device memory of the sizes the description and `n` give.
    pub unsafe fn lookup(&self, ids: *const i64, n: u64, table: *const c_void, out: *mut c_void, stream: *mut c_void) -> Result<()> {
        self.lookup_strided(ids, n, table, out, 0, stream)
    }

    /// # Safety
    /// As `lookup`; the rows of `out` are `out_stride` elements apart (0: without gaps).
    pub unsafe fn lookup_strided(
        &self,
        ids: *const i64,
        n: u64,
        table: *const c_void,
        out: *mut c_void,
        out_stride: u64,
        stream: *mut c_void,
    ) -> Result<()> {
        check(sys::oxz_embed_lookup_async(self.raw, ids, n, table, out, out_stride, stream))
    }

    /// # Safety
    /// As `lookup`; `d_table` is the table's gradient.
    pub unsafe fn grads(
        &mut self,
        ids: *const i64,
        n: u64,
        d_out: *const c_void,
        d_table: *mut c_void,
        accumulate: bool,
        stream: *mut c_void,
    ) -> Result<()> {
        self.grads_strided(ids, n, d_out, 0, d_table, accumulate, stream)
    }

    /// # Safety
    /// As `grads`; the rows of `d_out` are `d_out_stride` elements apart (0: without gaps).
    #[allow(clippy::too_many_arguments)]
    pub unsafe fn grads_strided(
        &mut self,
        ids: *const i64,
        n: u64,
        d_out: *const c_void,
        d_out_stride: u64,
        d_table: *mut c_void,
        accumulate: bool,
        stream: *mut c_void,
    ) -> Result<()> {
        check(sys::oxz_embed_grads_async(self.raw, ids, n, d_out, d_out_stride, d_table, accumulate as i32, stream))
    }
}

impl Drop for TokenEmbedding {
    fn drop(&mut self) {
        unsafe { sys::oxz_embed_destroy(self.raw) };
    }
}

/// Softmax cross entropy over the vocabulary with its gradients (the step loss of src/step_loss.rs over lm_head).
pub struct LossHead {
    raw: *mut sys::oxz_head,
}

impl LossHead {
    pub fn new(desc: &sys::oxz_head_desc) -> Result<Self> {
        let mut raw = ptr::null_mut();
        check(unsafe { sys::oxz_head_create(desc, &mut raw) })?;
        let this = Self { raw };
        check(unsafe { sys::oxz_head_alloc(this.raw, ptr::null_mut()) })?;
        Ok(this)
    }

    /// # Safety
    /// The batch's pointers and the outputs are device memory of the sizes the description and the batch give.
    pub unsafe fn loss(&mut self, batch: &sys::oxz_head_batch, row_loss: *mut f32, totals: *mut f32, stream: *mut c_void) -> Result<()> {
        self.loss_with_stats(batch, row_loss, ptr::null_mut(), totals, stream)
    }

    /// # Safety
    /// As `loss`; `row_stats` receives what `grads` needs of the same batch.
    pub unsafe fn loss_with_stats(
        &mut self,
        batch: &sys::oxz_head_batch,
        row_loss: *mut f32,
        row_stats: *mut f32,
        totals: *mut f32,
        stream: *mut c_void,
    ) -> Result<()> {
        check(sys::oxz_head_loss_async(self.raw, batch, row_loss, row_stats, totals, stream))
    }

    /// # Safety
    /// As `loss`; `row_stats` was written by `loss_with_stats` for the same batch, `grads` names the gradients' memory.
    pub unsafe fn grads(
        &mut self,
        batch: &sys::oxz_head_batch,
        row_stats: *const f32,
        grads: &sys::oxz_head_grads,
        stream: *mut c_void,
    ) -> Result<()> {
        check(sys::oxz_head_grads_async(self.raw, batch, row_stats, grads, stream))
    }

    /// # Safety
    /// As `loss`; `grads` names the gradients' memory.
    pub unsafe fn loss_and_grads(
        &mut self,
        batch: &sys::oxz_head_batch,
        row_loss: *mut f32,
        totals: *mut f32,
        grads: &sys::oxz_head_grads,
        stream: *mut c_void,
    ) -> Result<()> {
        self.loss_and_grads_with_stats(batch, row_loss, ptr::null_mut(), totals, grads, stream)
    }

    /// # Safety
    /// As `loss_and_grads`; `row_stats` receives the rows' statistics as well.
    pub unsafe fn loss_and_grads_with_stats(
        &mut self,
        batch: &sys::oxz_head_batch,
        row_loss: *mut f32,
        row_stats: *mut f32,
        totals: *mut f32,
        grads: &sys::oxz_head_grads,
        stream: *mut c_void,
    ) -> Result<()> {
        check(sys::oxz_head_loss_grads_async(self.raw, batch, row_loss, row_stats, totals, grads, stream))
    }
}

impl Drop for LossHead {
    fn drop(&mut self) {
        unsafe { sys::oxz_head_destroy(self.raw) };
    }
}
