// The token embedding as a node of torch's autograd graph.
//
// Both passes of a short call are bound by what the host does for them.  A node in C++ needs neither Python's lock nor a thread state where the backward pass has its
// threads: 128 tokens, 8192 x 512 bf16, forward and backward called eagerly 55 us, 88 by the same launches from a torch.autograd.Function; with no launches at all such a function
// takes 51, an empty node in C++ 34, most of it torch's hand-over to another thread and back.
#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/library.h>

#include <atomic>

#include "lt_cuda.h"

namespace {

std::atomic<long long> launches{0};

int elem_type(at::ScalarType t) { return t == at::kFloat ? 0 : t == at::kBFloat16 ? 1 : t == at::kHalf ? 2 : -1; }

void check(int rc, const char* name) { TORCH_CHECK(rc == 0, name, " failed with code ", rc); }

at::Tensor rows_of(const at::Tensor& idx, const at::Tensor& table, double scale) {
  const c10::cuda::CUDAGuard guard(table.device());
  at::Tensor out = at::empty({idx.numel(), table.size(1)}, table.options().requires_grad(false));
  launches += 1;
  check(lt_token_embedding_fwd(elem_type(table.scalar_type()), idx.const_data_ptr(), idx.scalar_type() == at::kInt, table.const_data_ptr(), out.mutable_data_ptr(), idx.numel(),
                               int(table.size(1)), int(table.size(0)), float(scale), c10::cuda::getCurrentCUDAStream().stream()),
        "lt_token_embedding_fwd");
  return out;
}

at::Tensor gradient(const at::Tensor& idx, at::Tensor dout, int64_t vocab, double scale, int64_t pad) {
  const c10::cuda::CUDAGuard guard(dout.device());
  if (dout.stride(1) != 1) dout = dout.contiguous();
  const int64_t n = dout.size(0), dim = dout.size(1), size = dout.element_size();
  at::Tensor grad = at::empty({vocab, dim}, dout.options()), room;
  char* order = nullptr;
  int tile = 1;
  // Few tokens and a small gradient: one launch, which reads all tokens for every 16 KB of it.  Replayed, one launch / sort and sums, us: 128 tokens, 8.4 MB 5.5 / 11.7;
  // 1024, 8.4 MB 9.6 / 17.5; 2048, 8.4 MB 13.7 / 21.2; 2048, 64 KB 13.5 / 21.2; 256, 66 MB 15.7 / 15.8; but 4096, 64 KB 37 / 27; 512, 66 MB 17.8 / 16.4; 64, 263 MB 49 / 41.
  if (!(n <= 2048 && grad.nbytes() <= 1u << 26 && n * grad.nbytes() <= 1ull << 34)) {
    // sorted rows that a CTA sums of 256 vectors of 16 bytes, or of 1024 columns: up to 32, so that there are eight CTAs an SM
    const int64_t width = dim * size % 16 == 0 ? 256 * 16 / size : 1024, chunks = (dim + width - 1) / width;
    for (tile = 8; tile < 32 && n * chunks >= 2 * tile * 8 * 148;) tile *= 2;
    // the sorted list twice, 8 bytes an entry, and two rows for the pieces of every tile
    room = at::empty({16 * n + (n + tile - 1) / tile * 8 * dim}, dout.options().dtype(at::kByte));
    order = static_cast<char*>(room.mutable_data_ptr());
  }
  launches += order ? 4 : 1;
  check(lt_token_embedding_bwd(elem_type(dout.scalar_type()), idx.const_data_ptr(), idx.scalar_type() == at::kInt, dout.const_data_ptr(), dout.stride(0), grad.mutable_data_ptr(), n,
                               int(dim), int(vocab), float(scale), pad, order, reinterpret_cast<float*>(order ? order + 16 * n : nullptr), tile, c10::cuda::getCurrentCUDAStream().stream()),
        "lt_token_embedding_bwd");
  return grad;
}

struct TokenEmbeddingBackward : public torch::autograd::Node {
  torch::autograd::SavedVariable idx;
  int64_t vocab = 0, pad = -1;
  double scale = 1.0;

  std::string name() const override { return "TokenEmbeddingBackward"; }
  void release_variables() override { idx.reset_data(); }
  torch::autograd::variable_list apply(torch::autograd::variable_list&& grads) override {
    TORCH_CHECK(!at::GradMode::is_enabled(), "token_embedding is differentiable once");     // (a second derivative would silently be that of a constant)
    if (!grads[0].defined()) return {at::Tensor()};
    return {gradient(idx.unpack(shared_from_this()), grads[0], vocab, scale, pad)};
  }
};

// scale * table[idx] for dense tokens idx [n] (int32 or int64) and a dense table [V, D] of fp32, bf16 or fp16 on the same GPU.
at::Tensor token_embedding(const at::Tensor& idx, const at::Tensor& table, double scale, int64_t pad) {
  TORCH_CHECK(table.is_cuda() && idx.device() == table.device() && elem_type(table.scalar_type()) >= 0 && table.dim() == 2 && table.is_contiguous() && idx.dim() == 1 &&
                  idx.is_contiguous() && (idx.scalar_type() == at::kLong || idx.scalar_type() == at::kInt),
              "token_embedding: dense tokens and a dense table on one GPU are expected");
  TORCH_CHECK(!table._fw_grad(0).defined(), "token_embedding has no forward-mode derivative");
  at::Tensor out = rows_of(idx, table, scale);
  if (at::GradMode::is_enabled() && table.requires_grad()) {
    auto node = std::shared_ptr<TokenEmbeddingBackward>(new TokenEmbeddingBackward(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(table));
    node->idx = torch::autograd::SavedVariable(idx, false);
    node->vocab = table.size(0);
    node->pad = pad;
    node->scale = scale;
    torch::autograd::set_history(out, node);
  }
  return out;
}

}  // namespace

TORCH_LIBRARY(litetorch_b200, m) { m.def("token_embedding", &token_embedding); }

extern "C" long long lt_torch_launches(int reset) { return reset ? launches.exchange(0) : launches.load(); }
