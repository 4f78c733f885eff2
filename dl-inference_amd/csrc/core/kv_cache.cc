// Paged KV cache (replaces src/kv_cache.cc:9-49 of the reference; layout in kv_cache.h).
#include "dli/kv_cache.h"

#include <stdexcept>
#include <string>
#include <tuple>

#include "dli_hip.h"

namespace dli {
namespace {

int hipDtype(DType dtype) {
  switch (dtype) {
    case DType::Float32: return DLI_F32;
    case DType::BFloat16: return DLI_BF16;
    case DType::Float16: return DLI_F16;
    default: throw std::invalid_argument("KV cache expects floating tensors");
  }
}

void hipCheck(int rc, const char* what) {
  if (rc != 0) throw std::runtime_error(std::string(what) + ": " + dli_hip_last_error());
}

void validatePair(const Tensor& key, const Tensor& value) {
  if (key.isCuda() != value.isCuda())
    throw std::invalid_argument("KV cache key/value must be on the same device");
  if (key.rank() != 4 || value.rank() != 4)
    throw std::invalid_argument("KV cache expects rank-4 tensors");
  if (key.shape() != value.shape()) throw std::invalid_argument("KV key/value shape mismatch");
  if (key.dtype() != value.dtype()) throw std::invalid_argument("KV key/value dtype mismatch");
  hipDtype(key.dtype());
}

Tensor identityBlockTable(std::int64_t batch, std::int64_t max_blocks, int device_id) {
  auto table = at::arange(batch * max_blocks, at::TensorOptions().dtype(at::kInt))
                   .view({batch, max_blocks});
  return Tensor(table.to(at::Device(at::kCUDA, device_id)));
}

// Pools are filled on torch's current stream, and what is copied from a pool that is given back
// runs on the cache's: quantised entries on the device wait for it around both, which a capture cannot.
void settle(bool wait, void* stream) {
  if (!wait) return;
  int capturing = 0;
  hipCheck(dli_hip_stream_is_capturing(stream, &capturing), "KV cache");
  if (capturing != 0)
    throw std::runtime_error(
        "KV cache: an 8-bit entry cannot be made or grown inside a stream capture; run the graph once "
        "without capture first, with max_seq_len configured");
  hipCheck(dli_hip_device_synchronize(), "KV cache");
}

void allocatePools(KVCacheEntry& e, DType dtype, int device_id) {
  const std::int64_t blocks = e.batch * e.max_blocks;
  // Zero-filled once, so that attention kernels reading a partially filled block see finite
  // values in the slots they mask out.
  auto options = at::TensorOptions().dtype(toTorchDType(dtype));
  options = device_id == kCpuDevice ? options.device(at::kCPU)
                                    : options.device(at::kCUDA, device_id);
  e.key_pool = Tensor(at::zeros({blocks, e.heads, e.block_size, e.head_dim}, options));
  e.value_pool = Tensor(at::zeros({blocks, e.heads, e.head_dim, e.block_size}, options));
  if (dtype == DType::UInt8) e.scales = Tensor(at::zeros({blocks, e.heads, 2, e.block_size}, options));
  if (device_id == kCpuDevice) {
    e.block_table = Tensor(at::arange(blocks, at::TensorOptions().dtype(at::kInt))
                               .view({e.batch, e.max_blocks}));
  } else {
    e.block_table = identityBlockTable(e.batch, e.max_blocks, device_id);
  }
}

// The kernels of quantised entries run on the current device.
void requireCurrentDevice(const KVCacheEntry& e) {
  int current = 0;
  hipCheck(dli_hip_get_device(&current), "KV cache");
  if (e.key_pool.deviceId() != current)
    throw std::invalid_argument("KV cache: an 8-bit entry is used with its device current only");
}

void appendQuantized(const KVCacheEntry& e, const Tensor& key, const Tensor& value,
                     std::int64_t start, const Tensor* positions, void* stream) {
  requireCurrentDevice(e);
  hipCheck(dli_hip_kv_append_fp8(
               hipDtype(key.dtype()), key.deviceData(), value.deviceData(),
               const_cast<void*>(e.key_pool.deviceData()), const_cast<void*>(e.value_pool.deviceData()),
               const_cast<void*>(e.scales.deviceData()),
               static_cast<const std::int32_t*>(e.block_table.deviceData()), e.key_pool.dim(0), e.batch,
               e.heads, key.dim(2), e.head_dim, e.block_size, e.max_blocks, start,
               positions != nullptr ? positions->deviceData() : nullptr,
               positions != nullptr && positions->dtype() == DType::Int32 ? DLI_I32 : DLI_I64, stream),
           "KV cache append");
}

// Rows of x (floating, [.., D]) as e4m3 codes and scale codes, both uint8: the least power of two that
// brings a row's largest magnitude to at most 448; rows with an infinity or a NaN get scale 255 and
// zeros.
std::pair<at::Tensor, at::Tensor> quantizeRows(const at::Tensor& x) {
  const at::Tensor y = x.to(at::kFloat).contiguous();
  const at::Tensor bits = at::amax(y.abs(), -1).contiguous().view(at::kInt);  // of a NaN: a NaN
  const at::Tensor finite = bits.lt(0x7F800000);
  at::Tensor code = at::bitwise_right_shift(bits, 23) - 8 +
                    at::bitwise_and(bits, 0x7FFFFF).gt(0x600000).to(at::kInt);
  code = at::where(finite, code.clamp_min(0), at::full({}, 255, at::kInt));
  const at::Tensor inverse =
      at::bitwise_left_shift((254 - code).clamp_min(1), 23).view(at::kFloat).unsqueeze(-1);
  const at::Tensor v = at::where(finite.unsqueeze(-1), y, at::zeros({}, at::kFloat)) * inverse;
  return {v.to(at::kFloat8_e4m3fn).view(at::kByte), code.to(at::kByte)};
}

// What codes [.., D] and scale codes [..] stand for, in fp32.
at::Tensor dequantizeRows(const at::Tensor& codes, const at::Tensor& scales) {
  const at::Tensor c = scales.to(at::kInt);
  at::Tensor s = at::bitwise_left_shift(c, 23);
  s = at::where(c.eq(0), at::full({}, 0x00400000, at::kInt), s);
  s = at::where(c.eq(255), at::full({}, 0x7FC00000, at::kInt), s);
  return codes.contiguous().view(at::kFloat8_e4m3fn).to(at::kFloat) * s.view(at::kFloat).unsqueeze(-1);
}

// Host entries hold one block per sequence (block_size = capacity), so sequence b's keys are
// key_pool[b] = [heads, capacity, head_dim] and its values value_pool[b] = [heads, head_dim,
// capacity]: contiguous per head, which the ATen CPU attention reads without a gather. Token s
// of sequence b goes to position start[b] + s.
void appendHost(KVCacheEntry& e, const Tensor& key, const Tensor& value,
                const std::vector<std::int64_t>& start) {
  const std::int64_t seq = key.dim(2);
  at::Tensor kp = e.key_pool.torchTensor(), vp = e.value_pool.torchTensor();
  at::Tensor k = key.torchTensor(), v = value.torchTensor(), ks, vs;
  if (e.quantized()) {
    std::tie(k, ks) = quantizeRows(k);
    std::tie(v, vs) = quantizeRows(v);
  }
  for (std::int64_t b = 0; b < e.batch; ++b) {
    const std::int64_t p = start[static_cast<std::size_t>(b)];
    if (p < 0 || p + seq > e.capacity())
      throw std::out_of_range("KV cache position outside the host cache capacity");
    kp[b].narrow(1, p, seq).copy_(k[b]);
    vp[b].narrow(2, p, seq).copy_(v[b].transpose(-1, -2));
    if (e.quantized()) {
      at::Tensor scales = e.scales.torchTensor()[b];  // [H, 2, capacity]
      scales.select(1, 0).narrow(1, p, seq).copy_(ks[b]);
      scales.select(1, 1).narrow(1, p, seq).copy_(vs[b]);
    }
  }
}

}  // namespace

void KVCache::configure(std::int64_t block_size, std::int64_t max_seq_len,
                        const std::string& format) {
  if (block_size <= 0 || max_seq_len <= 0)
    throw std::invalid_argument("KV cache block_size and max_seq_len must be positive");
  if (!format.empty() && format != "fp8")
    throw std::invalid_argument("KV cache format must be \"\" or \"fp8\", not \"" + format + "\"");
  format_ = format;
  block_size_ = block_size;
  max_seq_len_ = max_seq_len;
}

KVCacheEntry* KVCache::find(const std::string& name) {
  auto it = entries_.find(name);
  return it == entries_.end() ? nullptr : &it->second;
}

const KVCacheEntry* KVCache::get(const std::string& name) const {
  auto it = entries_.find(name);
  return it == entries_.end() ? nullptr : &it->second;
}

KVCacheEntry& KVCache::reserve(const std::string& name, DType dtype, std::int64_t batch,
                               std::int64_t heads, std::int64_t head_dim, int device_id,
                               bool any_format) {
  auto allowed = [&](bool quantized) {
    if (quantized && !any_format)
      throw std::invalid_argument("KV cache entry " + name +
                                  " is in 8-bit format, which this operator does not take");
  };
  if (KVCacheEntry* existing = find(name)) {
    allowed(existing->quantized());
    if (existing->batch != batch || existing->heads != heads || existing->head_dim != head_dim)
      throw std::invalid_argument("KV cache append shape mismatch");
    if (existing->dtype != dtype) throw std::invalid_argument("KV cache dtype mismatch");
    return *existing;
  }
  if (batch <= 0 || heads <= 0 || head_dim <= 0)
    throw std::invalid_argument("KV cache geometry must be positive");
  hipDtype(dtype);
  const bool quantized = format_ == "fp8";
  allowed(quantized);
  if (quantized && head_dim > 256)
    throw std::invalid_argument("KV cache: the 8-bit format takes head_dim up to 256");
  KVCacheEntry entry;
  entry.dtype = dtype;
  entry.batch = batch;
  entry.heads = heads;
  entry.head_dim = head_dim;
  entry.block_size = block_size_;
  entry.max_blocks = (max_seq_len_ + block_size_ - 1) / block_size_;
  if (device_id == kCpuDevice) {  // one block per sequence on the host
    entry.block_size *= entry.max_blocks;
    entry.max_blocks = 1;
  }
  const bool wait = quantized && device_id != kCpuDevice;
  settle(wait, stream_);
  allocatePools(entry, quantized ? DType::UInt8 : dtype, device_id);
  settle(wait, stream_);
  return entries_.emplace(name, std::move(entry)).first->second;
}

void KVCache::grow(KVCacheEntry& e, std::int64_t needed_tokens) {
  if (!e.key_pool.isCuda())
    throw std::out_of_range("host KV cache holds " + std::to_string(e.capacity()) +
                            " tokens per sequence (configure a larger max_seq_len)");
  std::int64_t blocks = e.max_blocks;
  while (blocks * e.block_size < needed_tokens) blocks *= 2;
  if (blocks == e.max_blocks) return;
  KVCacheEntry bigger = e;
  bigger.max_blocks = blocks;
  settle(e.quantized(), stream_);
  allocatePools(bigger, e.key_pool.dtype(), e.key_pool.deviceId());
  settle(e.quantized(), stream_);
  // Physical block (b * old_max + i) moves to (b * new_max + i); copy per sequence.
  const std::size_t block_bytes =
      static_cast<std::size_t>(e.heads * e.block_size * e.head_dim) * byteSize(e.key_pool.dtype());
  for (std::int64_t b = 0; b < e.batch; ++b) {
    const std::size_t src = static_cast<std::size_t>(b * e.max_blocks) * block_bytes;
    const std::size_t dst = static_cast<std::size_t>(b * blocks) * block_bytes;
    const std::size_t bytes = static_cast<std::size_t>(e.max_blocks) * block_bytes;
    hipCheck(dli_hip_memcpy_async(static_cast<char*>(bigger.key_pool.deviceData()) + dst,
                                  static_cast<const char*>(e.key_pool.deviceData()) + src, bytes,
                                  DLI_MEMCPY_DEVICE_TO_DEVICE, stream_),
             "KV cache grow");
    hipCheck(dli_hip_memcpy_async(static_cast<char*>(bigger.value_pool.deviceData()) + dst,
                                  static_cast<const char*>(e.value_pool.deviceData()) + src, bytes,
                                  DLI_MEMCPY_DEVICE_TO_DEVICE, stream_),
             "KV cache grow");
    if (e.quantized()) {
      const std::size_t rows = static_cast<std::size_t>(e.heads * 2 * e.block_size * b);
      hipCheck(dli_hip_memcpy_async(
                   static_cast<char*>(bigger.scales.deviceData()) + rows * blocks,
                   static_cast<const char*>(e.scales.deviceData()) + rows * e.max_blocks,
                   static_cast<std::size_t>(e.heads * 2 * e.block_size * e.max_blocks),
                   DLI_MEMCPY_DEVICE_TO_DEVICE, stream_),
               "KV cache grow");
    }
  }
  settle(e.quantized(), stream_);
  e = std::move(bigger);
}

void KVCache::append(const std::string& name, const Tensor& key, const Tensor& value) {
  validatePair(key, value);
  KVCacheEntry& e = reserve(name, key.dtype(), key.dim(0), key.dim(1), key.dim(3),
                            key.isCuda() ? key.deviceId() : kCpuDevice, true);
  const std::int64_t seq = key.dim(2);
  if (e.length + seq > e.capacity()) grow(e, e.length + seq);
  if (!key.isCuda()) {
    appendHost(e, key, value, std::vector<std::int64_t>(static_cast<std::size_t>(e.batch), e.length));
    e.length += seq;
    return;
  }
  if (e.quantized()) {
    appendQuantized(e, key, value, e.length, nullptr, stream_);
    e.length += seq;
    return;
  }
  hipCheck(dli_hip_kv_append(hipDtype(key.dtype()), key.deviceData(), value.deviceData(),
                             e.key_pool.deviceData(), e.value_pool.deviceData(),
                             static_cast<const std::int32_t*>(e.block_table.deviceData()), e.batch,
                             e.heads, seq, e.head_dim, e.block_size, e.max_blocks, e.length,
                             nullptr, DLI_I64, stream_),
           "KV cache append");
  e.length += seq;
}

void KVCache::appendAt(const std::string& name, const Tensor& key, const Tensor& value,
                       const Tensor& positions) {
  validatePair(key, value);
  if (positions.isCuda() != key.isCuda())
    throw std::invalid_argument("KV cache positions must be on the key's device");
  if (positions.dtype() != DType::Int64 && positions.dtype() != DType::Int32)
    throw std::invalid_argument("KV cache positions must be int64 or int32");
  if (static_cast<std::int64_t>(positions.numel()) != key.dim(0))
    throw std::invalid_argument("KV cache positions must hold one entry per sequence");
  KVCacheEntry& e = reserve(name, key.dtype(), key.dim(0), key.dim(1), key.dim(3),
                            key.isCuda() ? key.deviceId() : kCpuDevice, true);
  if (!key.isCuda()) {
    const at::Tensor pos = positions.torchTensor().to(at::kLong).contiguous();
    const std::int64_t* p = pos.data_ptr<std::int64_t>();
    appendHost(e, key, value, std::vector<std::int64_t>(p, p + e.batch));
    return;
  }
  if (e.quantized()) {
    appendQuantized(e, key, value, 0, &positions, stream_);
    return;
  }
  hipCheck(dli_hip_kv_append(hipDtype(key.dtype()), key.deviceData(), value.deviceData(),
                             e.key_pool.deviceData(), e.value_pool.deviceData(),
                             static_cast<const std::int32_t*>(e.block_table.deviceData()), e.batch,
                             e.heads, key.dim(2), e.head_dim, e.block_size, e.max_blocks, 0,
                             positions.deviceData(),
                             positions.dtype() == DType::Int64 ? DLI_I64 : DLI_I32, stream_),
           "KV cache append");
}

std::pair<Tensor, Tensor> KVCache::read(const std::string& name, std::int64_t start,
                                        std::int64_t length, DType dtype) {
  const KVCacheEntry* e = get(name);
  if (e == nullptr) throw std::invalid_argument("KV cache read: unknown entry " + name);
  hipDtype(dtype);
  if (start < 0 || length < 0 || start > e->capacity() || length > e->capacity() - start)
    throw std::out_of_range("KV cache read: positions outside the entry's " +
                            std::to_string(e->capacity()) + " per sequence");
  const std::vector<std::int64_t> shape{e->batch, e->heads, length, e->head_dim};
  if (e->quantized() && e->key_pool.isCuda()) {
    requireCurrentDevice(*e);
    const StreamScope scope(stream_);
    std::pair<Tensor, Tensor> out{Tensor::cuda(dtype, shape, e->key_pool.deviceId()),
                                  Tensor::cuda(dtype, shape, e->key_pool.deviceId())};
    hipCheck(dli_hip_kv_read_fp8(hipDtype(dtype), e->key_pool.deviceData(), e->value_pool.deviceData(),
                                 e->scales.deviceData(),
                                 static_cast<const std::int32_t*>(e->block_table.deviceData()),
                                 e->key_pool.dim(0), out.first.deviceData(), out.second.deviceData(),
                                 e->batch, e->heads, length, e->head_dim, e->block_size, e->max_blocks,
                                 start, nullptr, DLI_I64, stream_),
             "KV cache read");
    return out;
  }
  // the blocks that hold the positions: [B, blocks, H, ..] -> [B, H, tokens, D]
  const std::int64_t first = length > 0 ? start / e->block_size : 0;
  const std::int64_t blocks = length > 0 ? (start + length - 1) / e->block_size - first + 1 : 0;
  std::pair<Tensor, Tensor> out;
  auto gather = [&] {
    const at::Tensor rows =
        e->block_table.torchTensor().narrow(1, first, blocks).reshape({-1}).to(at::kLong);
    auto tokens = [&](const at::Tensor& pool, bool dim_major) {
      at::Tensor t = pool.index_select(0, rows);
      if (dim_major) t = t.transpose(-1, -2);
      const std::int64_t width = t.size(-1);
      return t.reshape({e->batch, blocks, e->heads, e->block_size, width})
          .transpose(1, 2)
          .reshape({e->batch, e->heads, blocks * e->block_size, width})
          .narrow(2, blocks > 0 ? start - first * e->block_size : 0, length);
    };
    at::Tensor k = tokens(e->key_pool.torchTensor(), false), v = tokens(e->value_pool.torchTensor(), true);
    if (e->quantized()) {
      const at::Tensor s = tokens(e->scales.torchTensor(), true);  // [B, H, tokens, 2]
      k = dequantizeRows(k, s.select(-1, 0));
      v = dequantizeRows(v, s.select(-1, 1));
    }
    out = {Tensor(k.to(toTorchDType(dtype)).contiguous()), Tensor(v.to(toTorchDType(dtype)).contiguous())};
  };
  // torch's operators, behind what the cache's stream still writes
  if (e->key_pool.isCuda())
    StreamScope::onTorch(stream_, e->key_pool.deviceId(), gather);
  else
    gather();
  return out;
}

void KVCache::setLength(std::int64_t length) {
  if (length < 0) throw std::invalid_argument("KV cache length must be non-negative");
  for (auto& [name, e] : entries_) {
    if (length > e.capacity()) grow(e, length);
    e.length = length;
  }
}

}  // namespace dli
