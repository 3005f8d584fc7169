// GENERATED by js/gen_binding.py from include/tfjs_cuda.h -- do not edit by hand.
// Type declarations of the N-API addon (js/binding.cc).
export type Handle = object;  // napi_external: context, graph or event
export type HostBuffer = ArrayBufferView|ArrayBuffer;
export interface Conv2DInfoLike {
  batchSize: number; inHeight: number; inWidth: number; inChannels: number; outHeight: number;
  outWidth: number; outChannels: number; strideHeight: number; strideWidth: number;
  dilationHeight: number; dilationWidth: number; filterHeight: number; filterWidth: number;
  effectiveFilterHeight: number; effectiveFilterWidth: number; dataFormat?: string;
  padInfo: {top: number, bottom: number, left: number, right: number};
}
export interface EpilogueLike {
  bias: number; biasLen: number; activation: number; prelu: number; preluLen: number;
  clipLo: number; clipHi: number;
}
export function hostAlloc(nbytes: number): {status: number, buffer?: ArrayBuffer};  // tfjs_cuda_host_alloc
export function hostFree(buffer: ArrayBuffer): number;  // tfjs_cuda_host_free (through the finalizer)
export function tensorReadPromise<T extends ArrayBufferView>(ctx: Handle, id: number, into: T): Promise<T>;  // tfjs_cuda_tensor_read_async + tfjs_cuda_event_wait
export function ctxCreate(device_ordinal: number): {status: number, out: Handle};  // tfjs_cuda_ctx_create
export function deviceCount(): {status: number, out: number};  // tfjs_cuda_device_count
export function ctxDestroy(ctx: Handle): number;  // tfjs_cuda_ctx_destroy
export function lastError(ctx: Handle): string;  // tfjs_cuda_last_error
export function ctxSetOption(ctx: Handle, key: string, value: number): number;  // tfjs_cuda_ctx_set_option
export function ctxSync(ctx: Handle, timeout_ms: number): number;  // tfjs_cuda_ctx_sync
export function ctxMemory(ctx: Handle): {status: number, num_tensors: number, bytes_in_use: number, bytes_reserved: number, num_buffers_cached: number, num_device_allocs: number};  // tfjs_cuda_ctx_memory
export function ctxTimeBegin(ctx: Handle): number;  // tfjs_cuda_ctx_time_begin
export function ctxTimeEnd(ctx: Handle): {status: number, kernel_ms: number, num_launches: number};  // tfjs_cuda_ctx_time_end
export function profileBegin(ctx: Handle, max_launches: number): number;  // tfjs_cuda_profile_begin
export function profileEnd(ctx: Handle): {status: number, num_launches: number};  // tfjs_cuda_profile_end
export function profileGet(ctx: Handle, index: number): {status: number, name: string, ms: number};  // tfjs_cuda_profile_get
export function ctxLaunchCount(ctx: Handle): number;  // tfjs_cuda_ctx_launch_count
export function ctxStream(ctx: Handle): bigint;  // tfjs_cuda_ctx_stream
export function tensorRegister(ctx: Handle, rank: number, shape: number[], dtype: number): {status: number, out_id: number};  // tfjs_cuda_tensor_register
export function tensorWrite(ctx: Handle, id: number, host: HostBuffer): number;  // tfjs_cuda_tensor_write
export function tensorRead(ctx: Handle, id: number, host: HostBuffer): number;  // tfjs_cuda_tensor_read
export function tensorWriteAsync(ctx: Handle, id: number, host: HostBuffer): number;  // tfjs_cuda_tensor_write_async
export function tensorWait(ctx: Handle, id: number): number;  // tfjs_cuda_tensor_wait
export function tensorReadAsync(ctx: Handle, id: number, host: HostBuffer): {status: number, out_event: Handle};  // tfjs_cuda_tensor_read_async
export function eventQuery(ev: Handle): number;  // tfjs_cuda_event_query
export function eventWait(ev: Handle, timeout_ms: number): number;  // tfjs_cuda_event_wait
export function eventDestroy(ev: Handle): number;  // tfjs_cuda_event_destroy
export function tensorDispose(ctx: Handle, id: number): number;  // tfjs_cuda_tensor_dispose
export function tensorDevicePtr(ctx: Handle, id: number): {status: number, ptr: bigint, nbytes: number};  // tfjs_cuda_tensor_device_ptr
export function tensorShare(ctx: Handle, id: number): {status: number, ptr: bigint, nbytes: number};  // tfjs_cuda_tensor_share
export function tensorRegisterQuantized(ctx: Handle, rank: number, shape: number[], q: Uint8Array, scale: number, min: number): {status: number, out_id: number};  // tfjs_cuda_tensor_register_quantized
export function batchMatmul(ctx: Handle, a: number, b: number, out: number, batch: number, a_d1: number, a_d2: number, b_d1: number, b_d2: number, transpose_a: number, transpose_b: number, epi: EpilogueLike|null): number;  // tfjs_cuda_batch_matmul
export function conv2d(ctx: Handle, x: number, filter: number, out: number, info: Conv2DInfoLike, epi: EpilogueLike|null): number;  // tfjs_cuda_conv2d
export function depthwiseConv2d(ctx: Handle, x: number, filter: number, out: number, info: Conv2DInfoLike, epi: EpilogueLike|null): number;  // tfjs_cuda_depthwise_conv2d
export function separableConv2d(ctx: Handle, x: number, dw_filter: number, pw_filter: number, out: number, dw_info: Conv2DInfoLike, out_channels: number, dw_epi: EpilogueLike|null, pw_epi: EpilogueLike|null): number;  // tfjs_cuda_separable_conv2d
export function conv2dDerInput(ctx: Handle, dy: number, filter: number, dx: number, info: Conv2DInfoLike): number;  // tfjs_cuda_conv2d_der_input
export function conv2dDerFilter(ctx: Handle, x: number, dy: number, dw: number, info: Conv2DInfoLike): number;  // tfjs_cuda_conv2d_der_filter
export function depthwiseConv2dDerInput(ctx: Handle, dy: number, filter: number, dx: number, info: Conv2DInfoLike): number;  // tfjs_cuda_depthwise_conv2d_der_input
export function depthwiseConv2dDerFilter(ctx: Handle, x: number, dy: number, dw: number, info: Conv2DInfoLike): number;  // tfjs_cuda_depthwise_conv2d_der_filter
export function pool2dBackprop(ctx: Handle, dy: number, x: number, dx: number, info: Conv2DInfoLike, is_avg: number): number;  // tfjs_cuda_pool2d_backprop
export function clipBackprop(ctx: Handle, dy: number, x: number, out: number, lo: number, hi: number): number;  // tfjs_cuda_clip_backprop
export function transpose(ctx: Handle, x: number, out: number, rank: number, shape: number[], perm: number[]): number;  // tfjs_cuda_transpose
export function pool2d(ctx: Handle, x: number, out: number, info: Conv2DInfoLike, is_avg: number): number;  // tfjs_cuda_pool2d
export function binary(ctx: Handle, op: number, a: number, a_rank: number, a_shape: number[], b: number, b_rank: number, b_shape: number[], out: number): number;  // tfjs_cuda_binary
export function unary(ctx: Handle, op: number, x: number, out: number, p0: number, p1: number): number;  // tfjs_cuda_unary
export function reduceLast(ctx: Handle, op: number, x: number, out: number, outer: number, inner: number): number;  // tfjs_cuda_reduce_last
export function softmaxLast(ctx: Handle, x: number, out: number, outer: number, inner: number): number;  // tfjs_cuda_softmax_last
export function layerNorm(ctx: Handle, x: number, gamma: number, beta: number, y: number, stats: number, rows: number, width: number, epsilon: number): number;  // tfjs_cuda_layer_norm
export function layerNormBackprop(ctx: Handle, dy: number, x: number, gamma: number, stats: number, dx: number, dgamma: number, dbeta: number, rows: number, width: number): number;  // tfjs_cuda_layer_norm_backprop
export function embeddingLookup(ctx: Handle, table: number, indices: number, out: number, tokens: number, vocab: number, width: number, scale: number): number;  // tfjs_cuda_embedding_lookup
export function embeddingLookupBackprop(ctx: Handle, dy: number, indices: number, dtable: number, tokens: number, vocab: number, width: number, scale: number): number;  // tfjs_cuda_embedding_lookup_backprop
export function distillationLoss(ctx: Handle, logits: number, teacher_logits: number, teacher_indices: number, loss: number, stats: number, rows: number, classes: number, top: number, temperature: number): number;  // tfjs_cuda_distillation_loss
export function distillationLossBackprop(ctx: Handle, dloss: number, logits: number, teacher_logits: number, teacher_indices: number, stats: number, dlogits: number, rows: number, classes: number, top: number, temperature: number): number;  // tfjs_cuda_distillation_loss_backprop
export function cast(ctx: Handle, x: number, out: number): number;  // tfjs_cuda_cast
export function matmulStaticScratch(ctx: Handle, a: bigint|null, b: bigint|null, bias: bigint|null, out: bigint|null, m: number, k: number, n: number, activation: number, clip_lo: number, clip_hi: number): number;  // tfjs_cuda_matmul_static_scratch
export function graphBegin(ctx: Handle): number;  // tfjs_cuda_graph_begin
export function graphEnd(ctx: Handle): {status: number, out: Handle};  // tfjs_cuda_graph_end
export function graphLaunch(ctx: Handle, graph: Handle): number;  // tfjs_cuda_graph_launch
export function graphDestroy(ctx: Handle, graph: Handle): number;  // tfjs_cuda_graph_destroy
