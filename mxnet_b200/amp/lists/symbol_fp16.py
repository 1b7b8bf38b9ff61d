"""Operator lists of the fp16 AMP policy (``python/mxnet/amp/lists/symbol_fp16.py``).

FP16_FUNCS run in half precision (tensor-core bound); FP32_FUNCS always run in fp32 (reductions
with large dynamic range, exponentials, norms, losses); WIDEST_TYPE_CASTS cast all inputs to the
widest input type; everything else runs in whatever type arrives."""
FP16_FUNCS = [
    'Convolution', 'Deconvolution', 'FullyConnected', 'RNN', 'dot', 'batch_dot', '_npi_matmul', '_npi_dot',
    '_npi_einsum', '_npi_tensordot', '_contrib_interleaved_matmul_selfatt_qk', '_contrib_interleaved_matmul_selfatt_valatt',
    '_contrib_interleaved_matmul_encdec_qk', '_contrib_interleaved_matmul_encdec_valatt', '_contrib_fused_self_attention',
    '_contrib_sldwin_attention', '_linalg_gemm', '_linalg_gemm2',
]
# Inputs that keep their type whatever list their operator is in: numbers of tokens, which half types do not hold.  (What an operator
# updates in place keeps its type as well: the update would go to a copy.)
KEEP_INPUTS = {'_contrib_sldwin_attention': ('valid_length',)}
# Inputs that take the type of another one: of a cache, which the program has laid out in the type that it wants.
LIKE_INPUTS = {
    '_contrib_sldwin_cache_fill': ('key_cache', ('key', 'value')),
    '_contrib_sldwin_attention_step': ('key_cache', ('query', 'key', 'value')),
}
# softmax, log_softmax and the fused softmax cross-entropy are NOT forced to fp32 inputs here (the reference lists them
# under FP32_FUNCS): their kernels read half-precision rows and do the exponentials, sums and the loss in fp32
# registers, so casting a [tokens, vocabulary] score matrix to fp32 first would only add a pass over HBM.
FP32_FUNCS = [
    'softmin', 'masked_softmax', 'masked_log_softmax', 'SoftmaxOutput', 'SoftmaxActivation',
    'softmax_cross_entropy', 'CTCLoss', 'LinearRegressionOutput', 'LogisticRegressionOutput',
    'MAERegressionOutput', 'SVMOutput', 'exp', 'expm1', 'log', 'log10', 'log2', 'log1p', 'sum', 'mean', 'prod', 'norm',
    'nansum', 'nanprod', 'square_sum', 'L2Normalization', 'LRN', 'InstanceNorm', 'GroupNorm', 'moments', 'erfinv',
    'gamma', 'gammaln', 'digamma', 'reciprocal', 'rsqrt', 'rcbrt', 'cosh', 'sinh', 'tan', 'arccos', 'arcsin', 'arccosh',
    'arctanh', '_npi_std', '_npi_var', '_npi_norm', 'topk', 'cumsum', '_linalg_potrf', '_linalg_potri', '_linalg_inverse',
    '_linalg_det', '_linalg_slogdet', '_linalg_syevd', '_linalg_gelqf', 'smooth_l1', 'multi_sum_sq', 'multi_lars',
]
FP16_FP32_FUNCS = [
    'softmax', 'log_softmax', '_npx_softmax_ce_loss', 'Activation', 'BatchNorm', 'LayerNorm', 'Pooling', 'Dropout', 'Flatten', 'Reshape', 'transpose', 'Concat', 'stack',
    'SliceChannel', 'slice', 'slice_axis', 'take', 'pick', 'Embedding', 'one_hot', 'clip', 'relu', 'sigmoid', 'tanh',
    'abs', 'sign', 'sqrt', 'square', 'negative', 'LeakyReLU', 'expand_dims', 'squeeze', 'tile', 'repeat', 'reverse',
    'broadcast_to', 'broadcast_like', 'zeros_like', 'ones_like', 'Cast', 'identity', 'BlockGrad', 'SequenceMask',
    'SequenceLast', 'SequenceReverse', 'where', 'max', 'min', 'argmax', 'argmin', 'sort', 'argsort', 'UpSampling', 'Pad',
    'SwapAxis', 'gather_nd', 'scatter_nd', '_contrib_rotary_embedding', '_contrib_token_log_probs',
]
WIDEST_TYPE_CASTS = [
    'broadcast_add', 'broadcast_sub', 'broadcast_mul', 'broadcast_div', 'broadcast_mod', 'broadcast_power',
    'broadcast_maximum', 'broadcast_minimum', 'broadcast_hypot', 'elemwise_add', 'elemwise_sub', 'elemwise_mul',
    'elemwise_div', 'add_n', 'Concat', 'stack', 'where', '_npi_add', '_npi_subtract', '_npi_multiply', '_npi_true_divide',
    '_npi_power', '_npi_maximum', '_npi_minimum', '_npi_where', '_npi_concatenate', '_npi_stack',
    'broadcast_equal', 'broadcast_not_equal', 'broadcast_greater', 'broadcast_greater_equal', 'broadcast_lesser',
    'broadcast_lesser_equal',
]
CONDITIONAL_FP32_FUNCS = [('Activation', 'act_type', ['softrelu']), ('LeakyReLU', 'act_type', ['elu', 'selu'])]
LOSS_OUTPUT_FUNCTIONS = ['SoftmaxOutput', 'LinearRegressionOutput', 'LogisticRegressionOutput', 'MAERegressionOutput']
