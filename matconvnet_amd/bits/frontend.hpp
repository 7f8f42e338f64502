// Argument conventions of the MATLAB-facing drivers vl_nnconv / vl_nnbnorm / vl_nnpool, restated as plain
// C++ entry points (no MATLAB needed).  Each function takes what the MEX driver's mexFunction takes --
// a list of inputs (arrays and strings) and a number of requested outputs -- and applies the same
// parsing, validation, output-allocation and error rules:
//   vl_nnconv (x, f, b [, dzdy], options...)   matlab/src/vl_nnconv.cu:87-502  (empty f: subsample + bias)
//   vl_nnconvt(x, f, b [, dzdy], options...)   matlab/src/vl_nnconvt.cu:81-417
//   vl_nnbnorm(x, g, b [, dzdy], options...)   matlab/src/vl_nnbnorm.cu:73-301
//   vl_nnpool (x, pool [, dzdy], options...)   matlab/src/vl_nnpool.cu:72-314
//   vl_taccum (alpha, a, beta, b [, 'InPlace']) matlab/src/vl_taccummex.cu:151-224
// Where the MEX drivers raise a MATLAB error these return a vl::ErrorCode and leave the reference's
// message text in `message`.
#ifndef MCN_AMD_BITS_FRONTEND_HPP
#define MCN_AMD_BITS_FRONTEND_HPP

#include <memory>
#include <string>
#include <vector>

#include "data.hpp"

namespace vl { namespace frontend {

// One element of the argument list: a numeric array (device or host tensor view) or a string.
struct Arg {
  enum Kind { Array, String };
  Kind kind;
  Tensor tensor;
  std::string text;
  std::shared_ptr<std::vector<double> > owned;  // backing store of host option values

  static Arg array(Tensor const& t);
  static Arg string(std::string const& s);
  // host double row vector, what MATLAB passes for 'stride', 'pad', 'epsilon', the pooling size...
  static Arg numeric(std::vector<double> const& values);
};

// Who provides memory for outputs (MATLAB's allocator in the MEX drivers), and for what vl_nnlnorm, vl_nnfcloss, vl_nnhnorm and vl_nnattention
// keep on the device during a call, which may go back when the call returns, to be used again behind it on its stream.  Returning NULL = out of memory.
class Allocator {
 public:
  virtual ~Allocator() {}
  virtual void* allocate(DeviceType device, std::size_t bytes) = 0;
};

// out[0..nout-1] receive views of freshly allocated outputs.  A skipped output is an empty 0 x 0 null
// tensor, as the MEX drivers return empty matrices.  Outputs by position:
//   vl_nnconv : forward [y]             backward [dzdx, dzdf, dzdb]
//   vl_nnconvt: forward [y]             backward [dzdx, dzdf, dzdb]
//   vl_nnbnorm: forward [y, moments]    backward [dzdx, dzdg, dzdb, moments]
//   vl_nnpool : forward [y]             backward [dzdx]
//   vl_taccum : [alpha*a + beta*b]; nothing with 'InPlace' (a itself is updated)
//   vl_nnloss : forward [y] (1 x 1 on the device)   backward [dzdx]
//   vl_nnrelu : forward [y]             backward [dzdx]
//   vl_nnsoftmax: forward [y]           backward [dzdx]
//   vl_nnlnorm: forward [y, moments]    backward [dzdx, dzdg, dzdb, moments]
//   vl_nnfcloss: forward [y, logSums]   backward [dzdx, dzdf, dzdb]
//   vl_nnhnorm: forward [yq, yk]        backward [dzdq, dzdk, dzdgq, dzdgk]
//   vl_nnattention: forward [y, logSums] backward [dzdq, dzdk, dzdv]
ErrorCode vl_nnconv(Context& context, Allocator& allocator, int nout, Tensor* out, int nin, Arg const* in,
                    std::string& message);
ErrorCode vl_nnconvt(Context& context, Allocator& allocator, int nout, Tensor* out, int nin, Arg const* in,
                     std::string& message);
ErrorCode vl_nnbnorm(Context& context, Allocator& allocator, int nout, Tensor* out, int nin, Arg const* in,
                     std::string& message);
ErrorCode vl_nnpool(Context& context, Allocator& allocator, int nout, Tensor* out, int nin, Arg const* in,
                    std::string& message);
ErrorCode vl_taccum(Context& context, Allocator& allocator, int nout, Tensor* out, int nin, Arg const* in,
                    std::string& message);
// vl_nnrelu(x [, dzdy], 'leak', value)  (matlab/vl_nnrelu.m:33-55; a MATLAB function in the reference)
ErrorCode vl_nnrelu(Context& context, Allocator& allocator, int nout, Tensor* out, int nin, Arg const* in,
                    std::string& message);
// vl_nnsoftmax(x [, dzdy])  (matlab/vl_nnsoftmax.m:20-28; a MATLAB function in the reference)
ErrorCode vl_nnsoftmax(Context& context, Allocator& allocator, int nout, Tensor* out, int nin, Arg const* in,
                       std::string& message);
// vl_nnloss(x, c [, dzdy], 'loss', name, 'instanceWeights', w, 'normalise', tf, 'threshold', t, 'topK', k)
// (matlab/vl_nnloss.m:129-142; a MATLAB function in the reference).  x: single, on the device.  c and the instance
// weights: on the device (single) or host arrays (copied over).  dzdy: a host scalar, or empty for the forward mode.
ErrorCode vl_nnloss(Context& context, Allocator& allocator, int nout, Tensor* out, int nin, Arg const* in,
                    std::string& message);
// vl_nnlnorm(x, g, b [, dzdy], 'epsilon', e, 'moments', m): layer normalisation, with vl_nnbnorm's arguments (no counterpart in the
// reference).  Single precision, on the device; moments: H x W x N x 2, all means, then all deviations.
ErrorCode vl_nnlnorm(Context& context, Allocator& allocator, int nout, Tensor* out, int nin, Arg const* in,
                     std::string& message);
// vl_nnfcloss(x, f, b, c [, dzdy], 'instanceWeights', w, 'normalise', tf, 'logSums', s): vl_nnconv with filters of x's size followed by
// vl_nnloss 'softmaxlog', without the scores (no counterpart in the reference).  x, f, b: single, on the device, b may be empty; c
// and the weights as for vl_nnloss.  logSums: the forward call's second result, which saves the backward call a third of its work.
ErrorCode vl_nnfcloss(Context& context, Allocator& allocator, int nout, Tensor* out, int nin, Arg const* in,
                      std::string& message);
// vl_nnhnorm(q, k, gq, gk [, dzdq, dzdk], 'epsilon', e, 'normalise', tf, 'neighbours', tf, 'positions', p, 'frequencies', f): mcn_hnorm_*
// (no counterpart in the reference).  q, k: channels x heads x positions x sequences, single, on the device, one of them may be empty; gq, gk: a
// value per channel, or empty; p: axes x all positions, f: pairs x axes, both double, on the device, or neither: no rotation.
ErrorCode vl_nnhnorm(Context& context, Allocator& allocator, int nout, Tensor* out, int nin, Arg const* in,
                     std::string& message);
// vl_nnattention(q, k, v [, dzdy], 'causal', tf, 'scale', s, 'output', y, 'logSums', l): mcn_attention_* of sequences of one length (no
// counterpart in the reference).  q: channels x heads x positions x sequences, k, v: channels x key heads x keys x sequences, single, on the
// device; l: heads x positions x sequences.  y and l, the forward call's results, save the backward call making them again.
ErrorCode vl_nnattention(Context& context, Allocator& allocator, int nout, Tensor* out, int nin, Arg const* in,
                         std::string& message);

} }  // namespace vl::frontend
#endif
