// GENERATED by js/gen_binding.py from include/tfjs_cuda.h -- do not edit by hand.
//
// Node N-API addon for the B200 `cuda` backend of tfjs-core: one function per entry point of
// the C ABI (include/tfjs_cuda.h), pure marshalling.  js/backend_cuda.ts is the only caller.
// Build with node-gyp (js/binding.gyp); links against tfjs-core_b200/libtfjs_cuda.so.
#include <node_api.h>

#include <cstdint>
#include <cstring>
#include <string>
#include <vector>

#include "tfjs_cuda.h"

namespace {

#define NAPI_OK(call)                                                   \
  do {                                                                  \
    if ((call) != napi_ok) {                                            \
      napi_throw_error(env, nullptr, "N-API call failed: " #call);      \
      return nullptr;                                                   \
    }                                                                   \
  } while (0)

constexpr size_t MAX_ARGS = 16;

struct Args {
  napi_env env;
  size_t argc = MAX_ARGS;
  napi_value argv[MAX_ARGS];
  bool ok = true;
  Args(napi_env e, napi_callback_info info) : env(e) {
    if (napi_get_cb_info(env, info, &argc, argv, nullptr, nullptr) != napi_ok) ok = false;
  }
  bool fail(const char* msg) {
    if (ok) napi_throw_type_error(env, nullptr, msg);
    ok = false;
    return false;
  }
  bool is_nullish(size_t i) {
    if (i >= argc) return true;
    napi_valuetype t;
    if (napi_typeof(env, argv[i], &t) != napi_ok) return true;
    return t == napi_undefined || t == napi_null;
  }
  void* handle(size_t i) {  // napi_external -> pointer (null / undefined -> nullptr)
    if (is_nullish(i)) return nullptr;
    void* p = nullptr;
    if (napi_get_value_external(env, argv[i], &p) != napi_ok) fail("expected a native handle");
    return p;
  }
  int64_t integer(size_t i) {
    int64_t v = 0;
    if (i >= argc || napi_get_value_int64(env, argv[i], &v) != napi_ok) fail("expected an integer");
    return v;
  }
  double number(size_t i) {
    double v = 0;
    if (i >= argc || napi_get_value_double(env, argv[i], &v) != napi_ok) fail("expected a number");
    return v;
  }
  std::string string(size_t i) {
    size_t len = 0;
    if (i >= argc || napi_get_value_string_utf8(env, argv[i], nullptr, 0, &len) != napi_ok) {
      fail("expected a string");
      return std::string();
    }
    std::string s(len, '\0');
    napi_get_value_string_utf8(env, argv[i], &s[0], len + 1, &len);
    return s;
  }
  template <typename T>
  std::vector<T> array(size_t i) {
    std::vector<T> out;
    uint32_t n = 0;
    if (i >= argc || napi_get_array_length(env, argv[i], &n) != napi_ok) {
      fail("expected an array of numbers");
      return out;
    }
    out.resize(n);
    for (uint32_t k = 0; k < n; k++) {
      napi_value e;
      int64_t v = 0;
      if (napi_get_element(env, argv[i], k, &e) != napi_ok || napi_get_value_int64(env, e, &v) != napi_ok)
        fail("expected an array of numbers");
      out[k] = (T)v;
    }
    if (out.empty()) out.push_back(0);  // callers pass .data(); keep it non-null for rank 0
    return out;
  }
  // TypedArray / DataView / ArrayBuffer -> (pointer, byte length)
  void* buffer(size_t i, size_t* nbytes) {
    *nbytes = 0;
    if (is_nullish(i)) return nullptr;
    bool is_ta = false, is_ab = false, is_dv = false;
    napi_is_typedarray(env, argv[i], &is_ta);
    void* data = nullptr;
    if (is_ta) {
      napi_typedarray_type type;
      size_t len = 0, off = 0;
      napi_value ab;
      if (napi_get_typedarray_info(env, argv[i], &type, &len, &data, &ab, &off) != napi_ok) fail("bad TypedArray");
      size_t elem = 1;
      switch (type) {
        case napi_int16_array: case napi_uint16_array: elem = 2; break;
        case napi_int32_array: case napi_uint32_array: case napi_float32_array: elem = 4; break;
        case napi_float64_array: case napi_bigint64_array: case napi_biguint64_array: elem = 8; break;
        default: elem = 1;
      }
      *nbytes = len * elem;
      return data;
    }
    napi_is_arraybuffer(env, argv[i], &is_ab);
    if (is_ab) {
      if (napi_get_arraybuffer_info(env, argv[i], &data, nbytes) != napi_ok) fail("bad ArrayBuffer");
      return data;
    }
    napi_is_dataview(env, argv[i], &is_dv);
    if (is_dv) {
      napi_value ab;
      size_t off = 0;
      if (napi_get_dataview_info(env, argv[i], nbytes, &data, &ab, &off) != napi_ok) fail("bad DataView");
      return data;
    }
    fail("expected a TypedArray, DataView or ArrayBuffer");
    return nullptr;
  }
  void* device_pointer(size_t i) {  // BigInt address (null / undefined -> nullptr)
    if (is_nullish(i)) return nullptr;
    uint64_t v = 0;
    bool lossless = true;
    if (napi_get_value_bigint_uint64(env, argv[i], &v, &lossless) != napi_ok) fail("expected a BigInt device address");
    return (void*)(uintptr_t)v;
  }
  int64_t field_i64(napi_value obj, const char* name, bool* present = nullptr) {
    napi_value v;
    int64_t out = 0;
    napi_valuetype t = napi_undefined;
    if (napi_get_named_property(env, obj, name, &v) == napi_ok) napi_typeof(env, v, &t);
    if (present) *present = t == napi_number;
    if (t == napi_number) napi_get_value_int64(env, v, &out);
    return out;
  }
  double field_f64(napi_value obj, const char* name) {
    napi_value v;
    double out = 0;
    napi_valuetype t = napi_undefined;
    if (napi_get_named_property(env, obj, name, &v) == napi_ok) napi_typeof(env, v, &t);
    if (t == napi_number) napi_get_value_double(env, v, &out);
    return out;
  }
  // Conv2DInfo (tfjs-core/src/ops/conv_util.ts:43-64) -> tfjs_conv2d_info.  Only channelsLast is
  // accepted, as the header says; padInfo {top, bottom, left, right} is flattened.
  tfjs_conv2d_info conv_info(size_t i) {
    tfjs_conv2d_info c;
    memset(&c, 0, sizeof(c));
    if (is_nullish(i)) {
      fail("convInfo is required");
      return c;
    }
    napi_value o = argv[i];
    napi_value fmt;
    if (napi_get_named_property(env, o, "dataFormat", &fmt) == napi_ok) {
      napi_valuetype t;
      napi_typeof(env, fmt, &t);
      if (t == napi_string) {
        char buf[32];
        size_t len = 0;
        napi_get_value_string_utf8(env, fmt, buf, sizeof(buf), &len);
        if (strcmp(buf, "channelsLast") != 0) fail("the cuda backend takes channelsLast (NHWC) convolutions only");
      }
    }
#define F(name) c.name = (int32_t)field_i64(o, #name)
    F(batchSize); F(inHeight); F(inWidth); F(inChannels); F(outHeight); F(outWidth); F(outChannels);
    F(strideHeight); F(strideWidth); F(dilationHeight); F(dilationWidth); F(filterHeight); F(filterWidth);
    F(effectiveFilterHeight); F(effectiveFilterWidth);
#undef F
    napi_value pad;
    napi_valuetype pt = napi_undefined;
    if (napi_get_named_property(env, o, "padInfo", &pad) == napi_ok) napi_typeof(env, pad, &pt);
    if (pt == napi_object) {
      c.padTop = (int32_t)field_i64(pad, "top");
      c.padBottom = (int32_t)field_i64(pad, "bottom");
      c.padLeft = (int32_t)field_i64(pad, "left");
      c.padRight = (int32_t)field_i64(pad, "right");
    }
    return c;
  }
  // {bias, biasLen, activation, prelu, preluLen, clipLo, clipHi} | null -> tfjs_epilogue
  bool epilogue(size_t i, tfjs_epilogue* e) {
    memset(e, 0, sizeof(*e));
    if (is_nullish(i)) return false;
    napi_value o = argv[i];
    e->bias = field_i64(o, "bias");
    e->bias_len = field_i64(o, "biasLen");
    e->activation = (int32_t)field_i64(o, "activation");
    e->prelu = field_i64(o, "prelu");
    e->prelu_len = field_i64(o, "preluLen");
    e->clip_lo = (float)field_f64(o, "clipLo");
    e->clip_hi = (float)field_f64(o, "clipHi");
    return true;
  }
};

struct Result {  // {status, ...outs}
  napi_env env;
  napi_value obj;
  Result(napi_env e, int status) : env(e) {
    napi_create_object(env, &obj);
    set_i64("status", status);
  }
  void set(const char* k, napi_value v) { napi_set_named_property(env, obj, k, v); }
  void set_i64(const char* k, int64_t v) { napi_value n; napi_create_int64(env, v, &n); set(k, n); }
  void set_f64(const char* k, double v) { napi_value n; napi_create_double(env, v, &n); set(k, n); }
  void set_str(const char* k, const char* s) { napi_value n; napi_create_string_utf8(env, s ? s : "", NAPI_AUTO_LENGTH, &n); set(k, n); }
  void set_ptr(const char* k, const void* p) { napi_value n; napi_create_bigint_uint64(env, (uint64_t)(uintptr_t)p, &n); set(k, n); }
  void set_handle(const char* k, void* p) {
    napi_value n;
    if (p) napi_create_external(env, p, nullptr, nullptr, &n); else napi_get_null(env, &n);
    set(k, n);
  }
};

napi_value status_value(napi_env env, int64_t status) {
  napi_value n;
  napi_create_int64(env, status, &n);
  return n;
}

// ---- hand-written entry points ---------------------------------------------------------------

// hostAlloc(nbytes) -> {status, buffer}: pinned host memory as an external ArrayBuffer; the
// finalizer returns it with tfjs_cuda_host_free when the ArrayBuffer is collected.
void FreePinned(napi_env, void* data, void*) { tfjs_cuda_host_free(data); }
napi_value HostAlloc(napi_env env, napi_callback_info info) {
  Args a(env, info);
  const int64_t nbytes = a.integer(0);
  if (!a.ok) return nullptr;
  void* p = nullptr;
  const int rc = tfjs_cuda_host_alloc(&p, (size_t)nbytes);
  Result r(env, rc);
  if (rc == TFJS_CUDA_OK) {
    napi_value ab;
    NAPI_OK(napi_create_external_arraybuffer(env, p, (size_t)nbytes, FreePinned, nullptr, &ab));
    r.set("buffer", ab);
  }
  return r.obj;
}
// hostFree(buffer): detaches the ArrayBuffer, which runs the finalizer above.
napi_value HostFree(napi_env env, napi_callback_info info) {
  Args a(env, info);
  if (!a.ok || a.argc < 1) return nullptr;
  NAPI_OK(napi_detach_arraybuffer(env, a.argv[0]));
  return status_value(env, TFJS_CUDA_OK);
}

// tensorReadPromise(ctx, id, typedArray) -> Promise<typedArray>: KernelBackend.read
// (tfjs-core/src/backends/backend.ts:95-97).  The copy is enqueued on the calling thread
// (tfjs_cuda_tensor_read_async); only the wait for its event runs on a worker thread, which
// touches the event and nothing else of the context, so the one-thread-per-context rule holds
// and the event loop is never blocked (precedent: the fence + promise of
// tfjs-core/src/backends/webgl/backend_webgl.ts:425-499).
struct ReadJob {
  napi_async_work work = nullptr;
  napi_deferred deferred = nullptr;
  napi_ref target = nullptr;  // keeps the destination TypedArray alive until the copy has landed
  tfjs_cuda_event* event = nullptr;
  int status = 0;
};
void ReadExecute(napi_env, void* data) {
  ReadJob* job = (ReadJob*)data;
  job->status = tfjs_cuda_event_wait(job->event, -1);
}
void ReadComplete(napi_env env, napi_status, void* data) {
  ReadJob* job = (ReadJob*)data;
  tfjs_cuda_event_destroy(job->event);
  napi_value target;
  napi_get_reference_value(env, job->target, &target);
  if (job->status == TFJS_CUDA_OK) {
    napi_resolve_deferred(env, job->deferred, target);
  } else {
    napi_value msg, err;
    napi_create_string_utf8(env, "cuda backend: asynchronous read failed", NAPI_AUTO_LENGTH, &msg);
    napi_create_error(env, nullptr, msg, &err);
    napi_reject_deferred(env, job->deferred, err);
  }
  napi_delete_reference(env, job->target);
  napi_delete_async_work(env, job->work);
  delete job;
}
napi_value TensorReadPromise(napi_env env, napi_callback_info info) {
  Args a(env, info);
  tfjs_cuda_ctx* ctx = (tfjs_cuda_ctx*)a.handle(0);
  const int64_t id = a.integer(1);
  size_t nbytes = 0;
  void* host = a.buffer(2, &nbytes);
  if (!a.ok) return nullptr;
  ReadJob* job = new ReadJob();
  const int rc = tfjs_cuda_tensor_read_async(ctx, id, host, nbytes, &job->event);
  if (rc != TFJS_CUDA_OK) {
    delete job;
    napi_throw_error(env, nullptr, tfjs_cuda_last_error(ctx));
    return nullptr;
  }
  napi_value promise, name;
  NAPI_OK(napi_create_promise(env, &job->deferred, &promise));
  NAPI_OK(napi_create_reference(env, a.argv[2], 1, &job->target));
  NAPI_OK(napi_create_string_utf8(env, "tfjs_cuda_read", NAPI_AUTO_LENGTH, &name));
  NAPI_OK(napi_create_async_work(env, nullptr, name, ReadExecute, ReadComplete, job, &job->work));
  NAPI_OK(napi_queue_async_work(env, job->work));
  return promise;
}

// ---- generated entry points ------------------------------------------------------------------
// tfjs_cuda_ctx_create
napi_value CtxCreate(napi_env env, napi_callback_info cbinfo) {
  Args argz(env, cbinfo);
  const int device_ordinal = (int)argz.integer(0);
  tfjs_cuda_ctx* out = nullptr;
  if (!argz.ok) return nullptr;
  Result r(env, (int)tfjs_cuda_ctx_create(device_ordinal, &out));
  r.set_handle("out", out);
  return r.obj;
}

// tfjs_cuda_device_count
napi_value DeviceCount(napi_env env, napi_callback_info cbinfo) {
  Args argz(env, cbinfo);
  int out = 0;
  if (!argz.ok) return nullptr;
  Result r(env, (int)tfjs_cuda_device_count(&out));
  r.set_i64("out", (int64_t)out);
  return r.obj;
}

// tfjs_cuda_ctx_destroy
napi_value CtxDestroy(napi_env env, napi_callback_info cbinfo) {
  Args argz(env, cbinfo);
  tfjs_cuda_ctx* ctx = (tfjs_cuda_ctx*)argz.handle(0);
  if (!argz.ok) return nullptr;
  return status_value(env, (int64_t)tfjs_cuda_ctx_destroy(ctx));
}

// tfjs_cuda_last_error
napi_value LastError(napi_env env, napi_callback_info cbinfo) {
  Args argz(env, cbinfo);
  tfjs_cuda_ctx* ctx = (tfjs_cuda_ctx*)argz.handle(0);
  if (!argz.ok) return nullptr;
  const char* s = tfjs_cuda_last_error(ctx);
  napi_value out;
  NAPI_OK(napi_create_string_utf8(env, s ? s : "", NAPI_AUTO_LENGTH, &out));
  return out;
}

// tfjs_cuda_ctx_set_option
napi_value CtxSetOption(napi_env env, napi_callback_info cbinfo) {
  Args argz(env, cbinfo);
  tfjs_cuda_ctx* ctx = (tfjs_cuda_ctx*)argz.handle(0);
  const std::string key = argz.string(1);
  const double value = (double)argz.number(2);
  if (!argz.ok) return nullptr;
  return status_value(env, (int64_t)tfjs_cuda_ctx_set_option(ctx, key.c_str(), value));
}

// tfjs_cuda_ctx_sync
napi_value CtxSync(napi_env env, napi_callback_info cbinfo) {
  Args argz(env, cbinfo);
  tfjs_cuda_ctx* ctx = (tfjs_cuda_ctx*)argz.handle(0);
  const int timeout_ms = (int)argz.integer(1);
  if (!argz.ok) return nullptr;
  return status_value(env, (int64_t)tfjs_cuda_ctx_sync(ctx, timeout_ms));
}

// tfjs_cuda_ctx_memory
napi_value CtxMemory(napi_env env, napi_callback_info cbinfo) {
  Args argz(env, cbinfo);
  tfjs_cuda_ctx* ctx = (tfjs_cuda_ctx*)argz.handle(0);
  tfjs_cuda_mem_stats out;
  memset(&out, 0, sizeof(out));
  if (!argz.ok) return nullptr;
  Result r(env, (int)tfjs_cuda_ctx_memory(ctx, &out));
  r.set_i64("num_tensors", out.num_tensors);
  r.set_i64("bytes_in_use", out.bytes_in_use);
  r.set_i64("bytes_reserved", out.bytes_reserved);
  r.set_i64("num_buffers_cached", out.num_buffers_cached);
  r.set_i64("num_device_allocs", out.num_device_allocs);
  return r.obj;
}

// tfjs_cuda_ctx_time_begin
napi_value CtxTimeBegin(napi_env env, napi_callback_info cbinfo) {
  Args argz(env, cbinfo);
  tfjs_cuda_ctx* ctx = (tfjs_cuda_ctx*)argz.handle(0);
  if (!argz.ok) return nullptr;
  return status_value(env, (int64_t)tfjs_cuda_ctx_time_begin(ctx));
}

// tfjs_cuda_ctx_time_end
napi_value CtxTimeEnd(napi_env env, napi_callback_info cbinfo) {
  Args argz(env, cbinfo);
  tfjs_cuda_ctx* ctx = (tfjs_cuda_ctx*)argz.handle(0);
  float kernel_ms = 0.f;
  int64_t num_launches = 0;
  if (!argz.ok) return nullptr;
  Result r(env, (int)tfjs_cuda_ctx_time_end(ctx, &kernel_ms, &num_launches));
  r.set_f64("kernel_ms", kernel_ms);
  r.set_i64("num_launches", (int64_t)num_launches);
  return r.obj;
}

// tfjs_cuda_profile_begin
napi_value ProfileBegin(napi_env env, napi_callback_info cbinfo) {
  Args argz(env, cbinfo);
  tfjs_cuda_ctx* ctx = (tfjs_cuda_ctx*)argz.handle(0);
  const int max_launches = (int)argz.integer(1);
  if (!argz.ok) return nullptr;
  return status_value(env, (int64_t)tfjs_cuda_profile_begin(ctx, max_launches));
}

// tfjs_cuda_profile_end
napi_value ProfileEnd(napi_env env, napi_callback_info cbinfo) {
  Args argz(env, cbinfo);
  tfjs_cuda_ctx* ctx = (tfjs_cuda_ctx*)argz.handle(0);
  int num_launches = 0;
  if (!argz.ok) return nullptr;
  Result r(env, (int)tfjs_cuda_profile_end(ctx, &num_launches));
  r.set_i64("num_launches", (int64_t)num_launches);
  return r.obj;
}

// tfjs_cuda_profile_get
napi_value ProfileGet(napi_env env, napi_callback_info cbinfo) {
  Args argz(env, cbinfo);
  tfjs_cuda_ctx* ctx = (tfjs_cuda_ctx*)argz.handle(0);
  const int index = (int)argz.integer(1);
  const char* name = nullptr;
  float ms = 0.f;
  if (!argz.ok) return nullptr;
  Result r(env, (int)tfjs_cuda_profile_get(ctx, index, &name, &ms));
  r.set_str("name", name);
  r.set_f64("ms", ms);
  return r.obj;
}

// tfjs_cuda_ctx_launch_count
napi_value CtxLaunchCount(napi_env env, napi_callback_info cbinfo) {
  Args argz(env, cbinfo);
  tfjs_cuda_ctx* ctx = (tfjs_cuda_ctx*)argz.handle(0);
  if (!argz.ok) return nullptr;
  return status_value(env, (int64_t)tfjs_cuda_ctx_launch_count(ctx));
}

// tfjs_cuda_ctx_stream
napi_value CtxStream(napi_env env, napi_callback_info cbinfo) {
  Args argz(env, cbinfo);
  tfjs_cuda_ctx* ctx = (tfjs_cuda_ctx*)argz.handle(0);
  if (!argz.ok) return nullptr;
  void* p = tfjs_cuda_ctx_stream(ctx);
  napi_value out;
  NAPI_OK(napi_create_bigint_uint64(env, (uint64_t)(uintptr_t)p, &out));
  return out;
}

// tfjs_cuda_tensor_register
napi_value TensorRegister(napi_env env, napi_callback_info cbinfo) {
  Args argz(env, cbinfo);
  tfjs_cuda_ctx* ctx = (tfjs_cuda_ctx*)argz.handle(0);
  int64_t out_id = 0;
  const int rank = (int)argz.integer(1);
  const std::vector<int64_t> shape = argz.array<int64_t>(2);
  const int dtype = (int)argz.integer(3);
  if (!argz.ok) return nullptr;
  Result r(env, (int)tfjs_cuda_tensor_register(ctx, &out_id, rank, shape.data(), dtype));
  r.set_i64("out_id", (int64_t)out_id);
  return r.obj;
}

// tfjs_cuda_tensor_write
napi_value TensorWrite(napi_env env, napi_callback_info cbinfo) {
  Args argz(env, cbinfo);
  tfjs_cuda_ctx* ctx = (tfjs_cuda_ctx*)argz.handle(0);
  const tfjs_tensor_id id = (tfjs_tensor_id)argz.integer(1);
  size_t host_bytes = 0;
  void* host = argz.buffer(2, &host_bytes);
  if (!argz.ok) return nullptr;
  return status_value(env, (int64_t)tfjs_cuda_tensor_write(ctx, id, host, host_bytes));
}

// tfjs_cuda_tensor_read
napi_value TensorRead(napi_env env, napi_callback_info cbinfo) {
  Args argz(env, cbinfo);
  tfjs_cuda_ctx* ctx = (tfjs_cuda_ctx*)argz.handle(0);
  const tfjs_tensor_id id = (tfjs_tensor_id)argz.integer(1);
  size_t host_bytes = 0;
  void* host = argz.buffer(2, &host_bytes);
  if (!argz.ok) return nullptr;
  return status_value(env, (int64_t)tfjs_cuda_tensor_read(ctx, id, host, host_bytes));
}

// tfjs_cuda_tensor_write_async
napi_value TensorWriteAsync(napi_env env, napi_callback_info cbinfo) {
  Args argz(env, cbinfo);
  tfjs_cuda_ctx* ctx = (tfjs_cuda_ctx*)argz.handle(0);
  const tfjs_tensor_id id = (tfjs_tensor_id)argz.integer(1);
  size_t host_bytes = 0;
  void* host = argz.buffer(2, &host_bytes);
  if (!argz.ok) return nullptr;
  return status_value(env, (int64_t)tfjs_cuda_tensor_write_async(ctx, id, host, host_bytes));
}

// tfjs_cuda_tensor_wait
napi_value TensorWait(napi_env env, napi_callback_info cbinfo) {
  Args argz(env, cbinfo);
  tfjs_cuda_ctx* ctx = (tfjs_cuda_ctx*)argz.handle(0);
  const tfjs_tensor_id id = (tfjs_tensor_id)argz.integer(1);
  if (!argz.ok) return nullptr;
  return status_value(env, (int64_t)tfjs_cuda_tensor_wait(ctx, id));
}

// tfjs_cuda_tensor_read_async
napi_value TensorReadAsync(napi_env env, napi_callback_info cbinfo) {
  Args argz(env, cbinfo);
  tfjs_cuda_ctx* ctx = (tfjs_cuda_ctx*)argz.handle(0);
  const tfjs_tensor_id id = (tfjs_tensor_id)argz.integer(1);
  size_t host_bytes = 0;
  void* host = argz.buffer(2, &host_bytes);
  tfjs_cuda_event* out_event = nullptr;
  if (!argz.ok) return nullptr;
  Result r(env, (int)tfjs_cuda_tensor_read_async(ctx, id, host, host_bytes, &out_event));
  r.set_handle("out_event", out_event);
  return r.obj;
}

// tfjs_cuda_event_query
napi_value EventQuery(napi_env env, napi_callback_info cbinfo) {
  Args argz(env, cbinfo);
  tfjs_cuda_event* ev = (tfjs_cuda_event*)argz.handle(0);
  if (!argz.ok) return nullptr;
  return status_value(env, (int64_t)tfjs_cuda_event_query(ev));
}

// tfjs_cuda_event_wait
napi_value EventWait(napi_env env, napi_callback_info cbinfo) {
  Args argz(env, cbinfo);
  tfjs_cuda_event* ev = (tfjs_cuda_event*)argz.handle(0);
  const int timeout_ms = (int)argz.integer(1);
  if (!argz.ok) return nullptr;
  return status_value(env, (int64_t)tfjs_cuda_event_wait(ev, timeout_ms));
}

// tfjs_cuda_event_destroy
napi_value EventDestroy(napi_env env, napi_callback_info cbinfo) {
  Args argz(env, cbinfo);
  tfjs_cuda_event* ev = (tfjs_cuda_event*)argz.handle(0);
  if (!argz.ok) return nullptr;
  return status_value(env, (int64_t)tfjs_cuda_event_destroy(ev));
}

// tfjs_cuda_tensor_dispose
napi_value TensorDispose(napi_env env, napi_callback_info cbinfo) {
  Args argz(env, cbinfo);
  tfjs_cuda_ctx* ctx = (tfjs_cuda_ctx*)argz.handle(0);
  const tfjs_tensor_id id = (tfjs_tensor_id)argz.integer(1);
  if (!argz.ok) return nullptr;
  return status_value(env, (int64_t)tfjs_cuda_tensor_dispose(ctx, id));
}

// tfjs_cuda_tensor_device_ptr
napi_value TensorDevicePtr(napi_env env, napi_callback_info cbinfo) {
  Args argz(env, cbinfo);
  tfjs_cuda_ctx* ctx = (tfjs_cuda_ctx*)argz.handle(0);
  const tfjs_tensor_id id = (tfjs_tensor_id)argz.integer(1);
  void* ptr = nullptr;
  size_t nbytes = 0;
  if (!argz.ok) return nullptr;
  Result r(env, (int)tfjs_cuda_tensor_device_ptr(ctx, id, &ptr, &nbytes));
  r.set_ptr("ptr", ptr);
  r.set_i64("nbytes", (int64_t)nbytes);
  return r.obj;
}

// tfjs_cuda_tensor_share
napi_value TensorShare(napi_env env, napi_callback_info cbinfo) {
  Args argz(env, cbinfo);
  tfjs_cuda_ctx* ctx = (tfjs_cuda_ctx*)argz.handle(0);
  const tfjs_tensor_id id = (tfjs_tensor_id)argz.integer(1);
  void* ptr = nullptr;
  size_t nbytes = 0;
  if (!argz.ok) return nullptr;
  Result r(env, (int)tfjs_cuda_tensor_share(ctx, id, &ptr, &nbytes));
  r.set_ptr("ptr", ptr);
  r.set_i64("nbytes", (int64_t)nbytes);
  return r.obj;
}

// tfjs_cuda_tensor_register_quantized
napi_value TensorRegisterQuantized(napi_env env, napi_callback_info cbinfo) {
  Args argz(env, cbinfo);
  tfjs_cuda_ctx* ctx = (tfjs_cuda_ctx*)argz.handle(0);
  int64_t out_id = 0;
  const int rank = (int)argz.integer(1);
  const std::vector<int64_t> shape = argz.array<int64_t>(2);
  size_t q_bytes = 0;
  const uint8_t* q = (const uint8_t*)argz.buffer(3, &q_bytes);
  const double scale = (double)argz.number(4);
  const double min = (double)argz.number(5);
  if (!argz.ok) return nullptr;
  Result r(env, (int)tfjs_cuda_tensor_register_quantized(ctx, &out_id, rank, shape.data(), q, scale, min));
  r.set_i64("out_id", (int64_t)out_id);
  return r.obj;
}

// tfjs_cuda_batch_matmul
napi_value BatchMatmul(napi_env env, napi_callback_info cbinfo) {
  Args argz(env, cbinfo);
  tfjs_cuda_ctx* ctx = (tfjs_cuda_ctx*)argz.handle(0);
  const tfjs_tensor_id a = (tfjs_tensor_id)argz.integer(1);
  const tfjs_tensor_id b = (tfjs_tensor_id)argz.integer(2);
  const tfjs_tensor_id out = (tfjs_tensor_id)argz.integer(3);
  const int32_t batch = (int32_t)argz.integer(4);
  const int32_t a_d1 = (int32_t)argz.integer(5);
  const int32_t a_d2 = (int32_t)argz.integer(6);
  const int32_t b_d1 = (int32_t)argz.integer(7);
  const int32_t b_d2 = (int32_t)argz.integer(8);
  const int transpose_a = (int)argz.integer(9);
  const int transpose_b = (int)argz.integer(10);
  tfjs_epilogue epi;
  const bool has_epi = argz.epilogue(11, &epi);
  if (!argz.ok) return nullptr;
  return status_value(env, (int64_t)tfjs_cuda_batch_matmul(ctx, a, b, out, batch, a_d1, a_d2, b_d1, b_d2, transpose_a, transpose_b, has_epi ? &epi : nullptr));
}

// tfjs_cuda_conv2d
napi_value Conv2d(napi_env env, napi_callback_info cbinfo) {
  Args argz(env, cbinfo);
  tfjs_cuda_ctx* ctx = (tfjs_cuda_ctx*)argz.handle(0);
  const tfjs_tensor_id x = (tfjs_tensor_id)argz.integer(1);
  const tfjs_tensor_id filter = (tfjs_tensor_id)argz.integer(2);
  const tfjs_tensor_id out = (tfjs_tensor_id)argz.integer(3);
  const tfjs_conv2d_info info = argz.conv_info(4);
  tfjs_epilogue epi;
  const bool has_epi = argz.epilogue(5, &epi);
  if (!argz.ok) return nullptr;
  return status_value(env, (int64_t)tfjs_cuda_conv2d(ctx, x, filter, out, &info, has_epi ? &epi : nullptr));
}

// tfjs_cuda_depthwise_conv2d
napi_value DepthwiseConv2d(napi_env env, napi_callback_info cbinfo) {
  Args argz(env, cbinfo);
  tfjs_cuda_ctx* ctx = (tfjs_cuda_ctx*)argz.handle(0);
  const tfjs_tensor_id x = (tfjs_tensor_id)argz.integer(1);
  const tfjs_tensor_id filter = (tfjs_tensor_id)argz.integer(2);
  const tfjs_tensor_id out = (tfjs_tensor_id)argz.integer(3);
  const tfjs_conv2d_info info = argz.conv_info(4);
  tfjs_epilogue epi;
  const bool has_epi = argz.epilogue(5, &epi);
  if (!argz.ok) return nullptr;
  return status_value(env, (int64_t)tfjs_cuda_depthwise_conv2d(ctx, x, filter, out, &info, has_epi ? &epi : nullptr));
}

// tfjs_cuda_separable_conv2d
napi_value SeparableConv2d(napi_env env, napi_callback_info cbinfo) {
  Args argz(env, cbinfo);
  tfjs_cuda_ctx* ctx = (tfjs_cuda_ctx*)argz.handle(0);
  const tfjs_tensor_id x = (tfjs_tensor_id)argz.integer(1);
  const tfjs_tensor_id dw_filter = (tfjs_tensor_id)argz.integer(2);
  const tfjs_tensor_id pw_filter = (tfjs_tensor_id)argz.integer(3);
  const tfjs_tensor_id out = (tfjs_tensor_id)argz.integer(4);
  const tfjs_conv2d_info dw_info = argz.conv_info(5);
  const int32_t out_channels = (int32_t)argz.integer(6);
  tfjs_epilogue dw_epi;
  const bool has_dw_epi = argz.epilogue(7, &dw_epi);
  tfjs_epilogue pw_epi;
  const bool has_pw_epi = argz.epilogue(8, &pw_epi);
  if (!argz.ok) return nullptr;
  return status_value(env, (int64_t)tfjs_cuda_separable_conv2d(ctx, x, dw_filter, pw_filter, out, &dw_info, out_channels, has_dw_epi ? &dw_epi : nullptr, has_pw_epi ? &pw_epi : nullptr));
}

// tfjs_cuda_conv2d_der_input
napi_value Conv2dDerInput(napi_env env, napi_callback_info cbinfo) {
  Args argz(env, cbinfo);
  tfjs_cuda_ctx* ctx = (tfjs_cuda_ctx*)argz.handle(0);
  const tfjs_tensor_id dy = (tfjs_tensor_id)argz.integer(1);
  const tfjs_tensor_id filter = (tfjs_tensor_id)argz.integer(2);
  const tfjs_tensor_id dx = (tfjs_tensor_id)argz.integer(3);
  const tfjs_conv2d_info info = argz.conv_info(4);
  if (!argz.ok) return nullptr;
  return status_value(env, (int64_t)tfjs_cuda_conv2d_der_input(ctx, dy, filter, dx, &info));
}

// tfjs_cuda_conv2d_der_filter
napi_value Conv2dDerFilter(napi_env env, napi_callback_info cbinfo) {
  Args argz(env, cbinfo);
  tfjs_cuda_ctx* ctx = (tfjs_cuda_ctx*)argz.handle(0);
  const tfjs_tensor_id x = (tfjs_tensor_id)argz.integer(1);
  const tfjs_tensor_id dy = (tfjs_tensor_id)argz.integer(2);
  const tfjs_tensor_id dw = (tfjs_tensor_id)argz.integer(3);
  const tfjs_conv2d_info info = argz.conv_info(4);
  if (!argz.ok) return nullptr;
  return status_value(env, (int64_t)tfjs_cuda_conv2d_der_filter(ctx, x, dy, dw, &info));
}

// tfjs_cuda_depthwise_conv2d_der_input
napi_value DepthwiseConv2dDerInput(napi_env env, napi_callback_info cbinfo) {
  Args argz(env, cbinfo);
  tfjs_cuda_ctx* ctx = (tfjs_cuda_ctx*)argz.handle(0);
  const tfjs_tensor_id dy = (tfjs_tensor_id)argz.integer(1);
  const tfjs_tensor_id filter = (tfjs_tensor_id)argz.integer(2);
  const tfjs_tensor_id dx = (tfjs_tensor_id)argz.integer(3);
  const tfjs_conv2d_info info = argz.conv_info(4);
  if (!argz.ok) return nullptr;
  return status_value(env, (int64_t)tfjs_cuda_depthwise_conv2d_der_input(ctx, dy, filter, dx, &info));
}

// tfjs_cuda_depthwise_conv2d_der_filter
napi_value DepthwiseConv2dDerFilter(napi_env env, napi_callback_info cbinfo) {
  Args argz(env, cbinfo);
  tfjs_cuda_ctx* ctx = (tfjs_cuda_ctx*)argz.handle(0);
  const tfjs_tensor_id x = (tfjs_tensor_id)argz.integer(1);
  const tfjs_tensor_id dy = (tfjs_tensor_id)argz.integer(2);
  const tfjs_tensor_id dw = (tfjs_tensor_id)argz.integer(3);
  const tfjs_conv2d_info info = argz.conv_info(4);
  if (!argz.ok) return nullptr;
  return status_value(env, (int64_t)tfjs_cuda_depthwise_conv2d_der_filter(ctx, x, dy, dw, &info));
}

// tfjs_cuda_pool2d_backprop
napi_value Pool2dBackprop(napi_env env, napi_callback_info cbinfo) {
  Args argz(env, cbinfo);
  tfjs_cuda_ctx* ctx = (tfjs_cuda_ctx*)argz.handle(0);
  const tfjs_tensor_id dy = (tfjs_tensor_id)argz.integer(1);
  const tfjs_tensor_id x = (tfjs_tensor_id)argz.integer(2);
  const tfjs_tensor_id dx = (tfjs_tensor_id)argz.integer(3);
  const tfjs_conv2d_info info = argz.conv_info(4);
  const int is_avg = (int)argz.integer(5);
  if (!argz.ok) return nullptr;
  return status_value(env, (int64_t)tfjs_cuda_pool2d_backprop(ctx, dy, x, dx, &info, is_avg));
}

// tfjs_cuda_clip_backprop
napi_value ClipBackprop(napi_env env, napi_callback_info cbinfo) {
  Args argz(env, cbinfo);
  tfjs_cuda_ctx* ctx = (tfjs_cuda_ctx*)argz.handle(0);
  const tfjs_tensor_id dy = (tfjs_tensor_id)argz.integer(1);
  const tfjs_tensor_id x = (tfjs_tensor_id)argz.integer(2);
  const tfjs_tensor_id out = (tfjs_tensor_id)argz.integer(3);
  const float lo = (float)argz.number(4);
  const float hi = (float)argz.number(5);
  if (!argz.ok) return nullptr;
  return status_value(env, (int64_t)tfjs_cuda_clip_backprop(ctx, dy, x, out, lo, hi));
}

// tfjs_cuda_transpose
napi_value Transpose(napi_env env, napi_callback_info cbinfo) {
  Args argz(env, cbinfo);
  tfjs_cuda_ctx* ctx = (tfjs_cuda_ctx*)argz.handle(0);
  const tfjs_tensor_id x = (tfjs_tensor_id)argz.integer(1);
  const tfjs_tensor_id out = (tfjs_tensor_id)argz.integer(2);
  const int rank = (int)argz.integer(3);
  const std::vector<int64_t> shape = argz.array<int64_t>(4);
  const std::vector<int32_t> perm = argz.array<int32_t>(5);
  if (!argz.ok) return nullptr;
  return status_value(env, (int64_t)tfjs_cuda_transpose(ctx, x, out, rank, shape.data(), perm.data()));
}

// tfjs_cuda_pool2d
napi_value Pool2d(napi_env env, napi_callback_info cbinfo) {
  Args argz(env, cbinfo);
  tfjs_cuda_ctx* ctx = (tfjs_cuda_ctx*)argz.handle(0);
  const tfjs_tensor_id x = (tfjs_tensor_id)argz.integer(1);
  const tfjs_tensor_id out = (tfjs_tensor_id)argz.integer(2);
  const tfjs_conv2d_info info = argz.conv_info(3);
  const int is_avg = (int)argz.integer(4);
  if (!argz.ok) return nullptr;
  return status_value(env, (int64_t)tfjs_cuda_pool2d(ctx, x, out, &info, is_avg));
}

// tfjs_cuda_binary
napi_value Binary(napi_env env, napi_callback_info cbinfo) {
  Args argz(env, cbinfo);
  tfjs_cuda_ctx* ctx = (tfjs_cuda_ctx*)argz.handle(0);
  const int op = (int)argz.integer(1);
  const tfjs_tensor_id a = (tfjs_tensor_id)argz.integer(2);
  const int a_rank = (int)argz.integer(3);
  const std::vector<int64_t> a_shape = argz.array<int64_t>(4);
  const tfjs_tensor_id b = (tfjs_tensor_id)argz.integer(5);
  const int b_rank = (int)argz.integer(6);
  const std::vector<int64_t> b_shape = argz.array<int64_t>(7);
  const tfjs_tensor_id out = (tfjs_tensor_id)argz.integer(8);
  if (!argz.ok) return nullptr;
  return status_value(env, (int64_t)tfjs_cuda_binary(ctx, op, a, a_rank, a_shape.data(), b, b_rank, b_shape.data(), out));
}

// tfjs_cuda_unary
napi_value Unary(napi_env env, napi_callback_info cbinfo) {
  Args argz(env, cbinfo);
  tfjs_cuda_ctx* ctx = (tfjs_cuda_ctx*)argz.handle(0);
  const int op = (int)argz.integer(1);
  const tfjs_tensor_id x = (tfjs_tensor_id)argz.integer(2);
  const tfjs_tensor_id out = (tfjs_tensor_id)argz.integer(3);
  const float p0 = (float)argz.number(4);
  const float p1 = (float)argz.number(5);
  if (!argz.ok) return nullptr;
  return status_value(env, (int64_t)tfjs_cuda_unary(ctx, op, x, out, p0, p1));
}

// tfjs_cuda_reduce_last
napi_value ReduceLast(napi_env env, napi_callback_info cbinfo) {
  Args argz(env, cbinfo);
  tfjs_cuda_ctx* ctx = (tfjs_cuda_ctx*)argz.handle(0);
  const int op = (int)argz.integer(1);
  const tfjs_tensor_id x = (tfjs_tensor_id)argz.integer(2);
  const tfjs_tensor_id out = (tfjs_tensor_id)argz.integer(3);
  const int64_t outer = (int64_t)argz.integer(4);
  const int64_t inner = (int64_t)argz.integer(5);
  if (!argz.ok) return nullptr;
  return status_value(env, (int64_t)tfjs_cuda_reduce_last(ctx, op, x, out, outer, inner));
}

// tfjs_cuda_softmax_last
napi_value SoftmaxLast(napi_env env, napi_callback_info cbinfo) {
  Args argz(env, cbinfo);
  tfjs_cuda_ctx* ctx = (tfjs_cuda_ctx*)argz.handle(0);
  const tfjs_tensor_id x = (tfjs_tensor_id)argz.integer(1);
  const tfjs_tensor_id out = (tfjs_tensor_id)argz.integer(2);
  const int64_t outer = (int64_t)argz.integer(3);
  const int64_t inner = (int64_t)argz.integer(4);
  if (!argz.ok) return nullptr;
  return status_value(env, (int64_t)tfjs_cuda_softmax_last(ctx, x, out, outer, inner));
}

// tfjs_cuda_layer_norm
napi_value LayerNorm(napi_env env, napi_callback_info cbinfo) {
  Args argz(env, cbinfo);
  tfjs_cuda_ctx* ctx = (tfjs_cuda_ctx*)argz.handle(0);
  const tfjs_tensor_id x = (tfjs_tensor_id)argz.integer(1);
  const tfjs_tensor_id gamma = (tfjs_tensor_id)argz.integer(2);
  const tfjs_tensor_id beta = (tfjs_tensor_id)argz.integer(3);
  const tfjs_tensor_id y = (tfjs_tensor_id)argz.integer(4);
  const tfjs_tensor_id stats = (tfjs_tensor_id)argz.integer(5);
  const int64_t rows = (int64_t)argz.integer(6);
  const int64_t width = (int64_t)argz.integer(7);
  const float epsilon = (float)argz.number(8);
  if (!argz.ok) return nullptr;
  return status_value(env, (int64_t)tfjs_cuda_layer_norm(ctx, x, gamma, beta, y, stats, rows, width, epsilon));
}

// tfjs_cuda_layer_norm_backprop
napi_value LayerNormBackprop(napi_env env, napi_callback_info cbinfo) {
  Args argz(env, cbinfo);
  tfjs_cuda_ctx* ctx = (tfjs_cuda_ctx*)argz.handle(0);
  const tfjs_tensor_id dy = (tfjs_tensor_id)argz.integer(1);
  const tfjs_tensor_id x = (tfjs_tensor_id)argz.integer(2);
  const tfjs_tensor_id gamma = (tfjs_tensor_id)argz.integer(3);
  const tfjs_tensor_id stats = (tfjs_tensor_id)argz.integer(4);
  const tfjs_tensor_id dx = (tfjs_tensor_id)argz.integer(5);
  const tfjs_tensor_id dgamma = (tfjs_tensor_id)argz.integer(6);
  const tfjs_tensor_id dbeta = (tfjs_tensor_id)argz.integer(7);
  const int64_t rows = (int64_t)argz.integer(8);
  const int64_t width = (int64_t)argz.integer(9);
  if (!argz.ok) return nullptr;
  return status_value(env, (int64_t)tfjs_cuda_layer_norm_backprop(ctx, dy, x, gamma, stats, dx, dgamma, dbeta, rows, width));
}

// tfjs_cuda_embedding_lookup
napi_value EmbeddingLookup(napi_env env, napi_callback_info cbinfo) {
  Args argz(env, cbinfo);
  tfjs_cuda_ctx* ctx = (tfjs_cuda_ctx*)argz.handle(0);
  const tfjs_tensor_id table = (tfjs_tensor_id)argz.integer(1);
  const tfjs_tensor_id indices = (tfjs_tensor_id)argz.integer(2);
  const tfjs_tensor_id out = (tfjs_tensor_id)argz.integer(3);
  const int64_t tokens = (int64_t)argz.integer(4);
  const int64_t vocab = (int64_t)argz.integer(5);
  const int64_t width = (int64_t)argz.integer(6);
  const float scale = (float)argz.number(7);
  if (!argz.ok) return nullptr;
  return status_value(env, (int64_t)tfjs_cuda_embedding_lookup(ctx, table, indices, out, tokens, vocab, width, scale));
}

// tfjs_cuda_embedding_lookup_backprop
napi_value EmbeddingLookupBackprop(napi_env env, napi_callback_info cbinfo) {
  Args argz(env, cbinfo);
  tfjs_cuda_ctx* ctx = (tfjs_cuda_ctx*)argz.handle(0);
  const tfjs_tensor_id dy = (tfjs_tensor_id)argz.integer(1);
  const tfjs_tensor_id indices = (tfjs_tensor_id)argz.integer(2);
  const tfjs_tensor_id dtable = (tfjs_tensor_id)argz.integer(3);
  const int64_t tokens = (int64_t)argz.integer(4);
  const int64_t vocab = (int64_t)argz.integer(5);
  const int64_t width = (int64_t)argz.integer(6);
  const float scale = (float)argz.number(7);
  if (!argz.ok) return nullptr;
  return status_value(env, (int64_t)tfjs_cuda_embedding_lookup_backprop(ctx, dy, indices, dtable, tokens, vocab, width, scale));
}

// tfjs_cuda_distillation_loss
napi_value DistillationLoss(napi_env env, napi_callback_info cbinfo) {
  Args argz(env, cbinfo);
  tfjs_cuda_ctx* ctx = (tfjs_cuda_ctx*)argz.handle(0);
  const tfjs_tensor_id logits = (tfjs_tensor_id)argz.integer(1);
  const tfjs_tensor_id teacher_logits = (tfjs_tensor_id)argz.integer(2);
  const tfjs_tensor_id teacher_indices = (tfjs_tensor_id)argz.integer(3);
  const tfjs_tensor_id loss = (tfjs_tensor_id)argz.integer(4);
  const tfjs_tensor_id stats = (tfjs_tensor_id)argz.integer(5);
  const int64_t rows = (int64_t)argz.integer(6);
  const int64_t classes = (int64_t)argz.integer(7);
  const int64_t top = (int64_t)argz.integer(8);
  const float temperature = (float)argz.number(9);
  if (!argz.ok) return nullptr;
  return status_value(env, (int64_t)tfjs_cuda_distillation_loss(ctx, logits, teacher_logits, teacher_indices, loss, stats, rows, classes, top, temperature));
}

// tfjs_cuda_distillation_loss_backprop
napi_value DistillationLossBackprop(napi_env env, napi_callback_info cbinfo) {
  Args argz(env, cbinfo);
  tfjs_cuda_ctx* ctx = (tfjs_cuda_ctx*)argz.handle(0);
  const tfjs_tensor_id dloss = (tfjs_tensor_id)argz.integer(1);
  const tfjs_tensor_id logits = (tfjs_tensor_id)argz.integer(2);
  const tfjs_tensor_id teacher_logits = (tfjs_tensor_id)argz.integer(3);
  const tfjs_tensor_id teacher_indices = (tfjs_tensor_id)argz.integer(4);
  const tfjs_tensor_id stats = (tfjs_tensor_id)argz.integer(5);
  const tfjs_tensor_id dlogits = (tfjs_tensor_id)argz.integer(6);
  const int64_t rows = (int64_t)argz.integer(7);
  const int64_t classes = (int64_t)argz.integer(8);
  const int64_t top = (int64_t)argz.integer(9);
  const float temperature = (float)argz.number(10);
  if (!argz.ok) return nullptr;
  return status_value(env, (int64_t)tfjs_cuda_distillation_loss_backprop(ctx, dloss, logits, teacher_logits, teacher_indices, stats, dlogits, rows, classes, top, temperature));
}

// tfjs_cuda_cast
napi_value Cast(napi_env env, napi_callback_info cbinfo) {
  Args argz(env, cbinfo);
  tfjs_cuda_ctx* ctx = (tfjs_cuda_ctx*)argz.handle(0);
  const tfjs_tensor_id x = (tfjs_tensor_id)argz.integer(1);
  const tfjs_tensor_id out = (tfjs_tensor_id)argz.integer(2);
  if (!argz.ok) return nullptr;
  return status_value(env, (int64_t)tfjs_cuda_cast(ctx, x, out));
}

// tfjs_cuda_matmul_static_scratch
napi_value MatmulStaticScratch(napi_env env, napi_callback_info cbinfo) {
  Args argz(env, cbinfo);
  tfjs_cuda_ctx* ctx = (tfjs_cuda_ctx*)argz.handle(0);
  float* a = (float*)argz.device_pointer(1);
  float* b = (float*)argz.device_pointer(2);
  float* bias = (float*)argz.device_pointer(3);
  float* out = (float*)argz.device_pointer(4);
  const int64_t m = (int64_t)argz.integer(5);
  const int64_t k = (int64_t)argz.integer(6);
  const int64_t n = (int64_t)argz.integer(7);
  const int activation = (int)argz.integer(8);
  const float clip_lo = (float)argz.number(9);
  const float clip_hi = (float)argz.number(10);
  if (!argz.ok) return nullptr;
  return status_value(env, (int64_t)tfjs_cuda_matmul_static_scratch(ctx, a, b, bias, out, m, k, n, activation, clip_lo, clip_hi));
}

// tfjs_cuda_graph_begin
napi_value GraphBegin(napi_env env, napi_callback_info cbinfo) {
  Args argz(env, cbinfo);
  tfjs_cuda_ctx* ctx = (tfjs_cuda_ctx*)argz.handle(0);
  if (!argz.ok) return nullptr;
  return status_value(env, (int64_t)tfjs_cuda_graph_begin(ctx));
}

// tfjs_cuda_graph_end
napi_value GraphEnd(napi_env env, napi_callback_info cbinfo) {
  Args argz(env, cbinfo);
  tfjs_cuda_ctx* ctx = (tfjs_cuda_ctx*)argz.handle(0);
  tfjs_cuda_graph* out = nullptr;
  if (!argz.ok) return nullptr;
  Result r(env, (int)tfjs_cuda_graph_end(ctx, &out));
  r.set_handle("out", out);
  return r.obj;
}

// tfjs_cuda_graph_launch
napi_value GraphLaunch(napi_env env, napi_callback_info cbinfo) {
  Args argz(env, cbinfo);
  tfjs_cuda_ctx* ctx = (tfjs_cuda_ctx*)argz.handle(0);
  tfjs_cuda_graph* graph = (tfjs_cuda_graph*)argz.handle(1);
  if (!argz.ok) return nullptr;
  return status_value(env, (int64_t)tfjs_cuda_graph_launch(ctx, graph));
}

// tfjs_cuda_graph_destroy
napi_value GraphDestroy(napi_env env, napi_callback_info cbinfo) {
  Args argz(env, cbinfo);
  tfjs_cuda_ctx* ctx = (tfjs_cuda_ctx*)argz.handle(0);
  tfjs_cuda_graph* graph = (tfjs_cuda_graph*)argz.handle(1);
  if (!argz.ok) return nullptr;
  return status_value(env, (int64_t)tfjs_cuda_graph_destroy(ctx, graph));
}

}  // namespace

#define EXPORT(js, fn)                                                        \
  do {                                                                        \
    napi_value f;                                                             \
    if (napi_create_function(env, js, NAPI_AUTO_LENGTH, fn, nullptr, &f) != napi_ok) return nullptr; \
    if (napi_set_named_property(env, exports, js, f) != napi_ok) return nullptr; \
  } while (0)

static napi_value Init(napi_env env, napi_value exports) {
  EXPORT("hostAlloc", HostAlloc);
  EXPORT("hostFree", HostFree);
  EXPORT("tensorReadPromise", TensorReadPromise);
  EXPORT("ctxCreate", CtxCreate);
  EXPORT("deviceCount", DeviceCount);
  EXPORT("ctxDestroy", CtxDestroy);
  EXPORT("lastError", LastError);
  EXPORT("ctxSetOption", CtxSetOption);
  EXPORT("ctxSync", CtxSync);
  EXPORT("ctxMemory", CtxMemory);
  EXPORT("ctxTimeBegin", CtxTimeBegin);
  EXPORT("ctxTimeEnd", CtxTimeEnd);
  EXPORT("profileBegin", ProfileBegin);
  EXPORT("profileEnd", ProfileEnd);
  EXPORT("profileGet", ProfileGet);
  EXPORT("ctxLaunchCount", CtxLaunchCount);
  EXPORT("ctxStream", CtxStream);
  EXPORT("tensorRegister", TensorRegister);
  EXPORT("tensorWrite", TensorWrite);
  EXPORT("tensorRead", TensorRead);
  EXPORT("tensorWriteAsync", TensorWriteAsync);
  EXPORT("tensorWait", TensorWait);
  EXPORT("tensorReadAsync", TensorReadAsync);
  EXPORT("eventQuery", EventQuery);
  EXPORT("eventWait", EventWait);
  EXPORT("eventDestroy", EventDestroy);
  EXPORT("tensorDispose", TensorDispose);
  EXPORT("tensorDevicePtr", TensorDevicePtr);
  EXPORT("tensorShare", TensorShare);
  EXPORT("tensorRegisterQuantized", TensorRegisterQuantized);
  EXPORT("batchMatmul", BatchMatmul);
  EXPORT("conv2d", Conv2d);
  EXPORT("depthwiseConv2d", DepthwiseConv2d);
  EXPORT("separableConv2d", SeparableConv2d);
  EXPORT("conv2dDerInput", Conv2dDerInput);
  EXPORT("conv2dDerFilter", Conv2dDerFilter);
  EXPORT("depthwiseConv2dDerInput", DepthwiseConv2dDerInput);
  EXPORT("depthwiseConv2dDerFilter", DepthwiseConv2dDerFilter);
  EXPORT("pool2dBackprop", Pool2dBackprop);
  EXPORT("clipBackprop", ClipBackprop);
  EXPORT("transpose", Transpose);
  EXPORT("pool2d", Pool2d);
  EXPORT("binary", Binary);
  EXPORT("unary", Unary);
  EXPORT("reduceLast", ReduceLast);
  EXPORT("softmaxLast", SoftmaxLast);
  EXPORT("layerNorm", LayerNorm);
  EXPORT("layerNormBackprop", LayerNormBackprop);
  EXPORT("embeddingLookup", EmbeddingLookup);
  EXPORT("embeddingLookupBackprop", EmbeddingLookupBackprop);
  EXPORT("distillationLoss", DistillationLoss);
  EXPORT("distillationLossBackprop", DistillationLossBackprop);
  EXPORT("cast", Cast);
  EXPORT("matmulStaticScratch", MatmulStaticScratch);
  EXPORT("graphBegin", GraphBegin);
  EXPORT("graphEnd", GraphEnd);
  EXPORT("graphLaunch", GraphLaunch);
  EXPORT("graphDestroy", GraphDestroy);
  return exports;
}

NAPI_MODULE(NODE_GYP_MODULE_NAME, Init)
