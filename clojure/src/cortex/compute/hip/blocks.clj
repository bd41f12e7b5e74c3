(ns cortex.compute.hip.blocks
  "The operators of residual blocks with experts (include/cortex_hip.h): norms around a block with gate and residual,
  the choice of experts, products grouped by expert, the sum of a token's rows, and clipping by the norm of all
  gradients.  They are no part of TensorMath; each function takes the stream, buffers and dimension maps, or nil where
  the header allows NULL.  No counterpart in the reference.

  UNEXERCISED (no JVM in the build image); see cortex.compute.hip.ffi."
  (:require [cortex.compute.hip.ffi :as ffi :refer [call! dtype-code op-code bool->int]]
            [cortex.compute.hip.driver :as hip-drv :refer [->ptr]]
            [think.datatype.core :as dtype])
  (:import [com.sun.jna Memory]))

(set! *warn-on-reflection* true)

(defn- select-device! [stream]
  (call! "ct_set_device" (int (:index (:device stream)))))

(defn- dims [dimensions]
  (ffi/dims->native dimensions (fn [_] (throw (ex-info "No indexed dimension is taken" {:dimensions dimensions})))))

(defn norm-residual!
  "output = residual-scale * residual + gate * (N_post(input) * post-scale + post-bias);
  normalized = N_pre(output) * pre-scale + pre-bias.  Kinds are :none, :rms or :layer."
  [stream output output-dims normalized normalized-dims statistics input input-dims residual residual-dims gate gate-dims
   post-scale post-bias pre-scale pre-bias post-kind pre-kind residual-scale epsilon]
  (select-device! stream)
  (call! "ct_norm_residual" (:handle stream) (->ptr output) (dims output-dims)
         (when normalized (->ptr normalized)) (when normalized (dims normalized-dims))
         (when statistics (->ptr statistics)) (->ptr input) (dims input-dims)
         (when residual (->ptr residual)) (when residual (dims residual-dims))
         (when gate (->ptr gate)) (when gate (dims gate-dims))
         (when post-scale (->ptr post-scale)) (when post-bias (->ptr post-bias))
         (when pre-scale (->ptr pre-scale)) (when pre-bias (->ptr pre-bias))
         (op-code ffi/norm-kind->code post-kind) (op-code ffi/norm-kind->code pre-kind)
         (double residual-scale) (double epsilon) (dtype-code output)))

(defn norm-residual-gradient!
  "The gradients of norm-residual!, from those of its results."
  [stream input-gradient input-gradient-dims residual-gradient residual-gradient-dims gate-gradient post-scale-gradient
   post-bias-gradient pre-scale-gradient pre-bias-gradient output-gradient output-gradient-dims normalized-gradient
   normalized-gradient-dims input input-dims output output-dims statistics gate gate-dims post-scale post-bias pre-scale
   post-kind pre-kind residual-scale]
  (select-device! stream)
  (call! "ct_norm_residual_gradient" (:handle stream)
         (when input-gradient (->ptr input-gradient)) (when input-gradient (dims input-gradient-dims))
         (when residual-gradient (->ptr residual-gradient)) (when residual-gradient (dims residual-gradient-dims))
         (when gate-gradient (->ptr gate-gradient))
         (when post-scale-gradient (->ptr post-scale-gradient)) (when post-bias-gradient (->ptr post-bias-gradient))
         (when pre-scale-gradient (->ptr pre-scale-gradient)) (when pre-bias-gradient (->ptr pre-bias-gradient))
         (when output-gradient (->ptr output-gradient)) (when output-gradient (dims output-gradient-dims))
         (when normalized-gradient (->ptr normalized-gradient)) (when normalized-gradient (dims normalized-gradient-dims))
         (->ptr input) (dims input-dims) (when output (->ptr output)) (when output (dims output-dims))
         (when statistics (->ptr statistics)) (when gate (->ptr gate)) (when gate (dims gate-dims))
         (when post-scale (->ptr post-scale)) (when post-bias (->ptr post-bias)) (when pre-scale (->ptr pre-scale))
         (op-code ffi/norm-kind->code post-kind) (op-code ffi/norm-kind->code pre-kind)
         (double residual-scale) (dtype-code input)))

(defn route-experts!
  "The n-chosen largest logits of each of n tokens, their softmax, and the assignments in order of their expert."
  [stream experts weights offsets tokens slots logits logits-colstride n n-experts n-chosen renormalize?]
  (select-device! stream)
  (call! "ct_route_experts" (:handle stream) (->ptr experts) (->ptr weights) (->ptr offsets) (->ptr tokens) (->ptr slots)
         (->ptr logits) (long logits-colstride) (long n) (long n-experts) (long n-chosen) (bool->int renormalize?)
         (dtype-code logits)))

(defn route-experts-gradient!
  "The gradient of the weights of route-experts! with respect to the logits."
  [stream logits-gradient logits-gradient-colstride weights-gradient weights experts logits logits-colstride n n-experts
   n-chosen renormalize?]
  (select-device! stream)
  (call! "ct_route_experts_gradient" (:handle stream) (->ptr logits-gradient) (long logits-gradient-colstride)
         (->ptr weights-gradient) (->ptr weights) (->ptr experts) (when logits (->ptr logits)) (long logits-colstride)
         (long n) (long n-experts) (long n-chosen) (bool->int renormalize?) (dtype-code logits-gradient)))

(defn grouped-gemm!
  "c[i] = alpha * a[index[i]] * (trans-b? b_e) + beta * c[i] for the rows i of every group e."
  [stream c c-colstride trans-b? alpha a a-row-count a-col-count a-colstride index b b-col-count b-colstride b-stride
   offsets n-groups row-count beta]
  (select-device! stream)
  (call! "ct_grouped_gemm" (:handle stream) (->ptr c) (long c-colstride) (bool->int trans-b?) (double alpha)
         (->ptr a) (long a-row-count) (long a-col-count) (long a-colstride) (when index (->ptr index))
         (->ptr b) (long b-col-count) (long b-colstride) (long b-stride) (->ptr offsets) (long n-groups) (long row-count)
         (double beta) (dtype-code c)))

(defn grouped-gemm-weights!
  "c_e = alpha * sum over the rows i of group e of a[a-index[i]]^T b[b-index[i]] + beta * c_e."
  [stream c c-colstride c-stride alpha a a-row-count a-col-count a-colstride a-index b b-row-count b-col-count b-colstride
   b-index offsets n-groups row-count beta]
  (select-device! stream)
  (call! "ct_grouped_gemm_weights" (:handle stream) (->ptr c) (long c-colstride) (long c-stride) (double alpha)
         (->ptr a) (long a-row-count) (long a-col-count) (long a-colstride) (when a-index (->ptr a-index))
         (->ptr b) (long b-row-count) (long b-col-count) (long b-colstride) (when b-index (->ptr b-index))
         (->ptr offsets) (long n-groups) (long row-count) (double beta) (dtype-code c)))

(defn gated-gemm!
  "inner[i] = f(gate) * up with [gate up] = a[index[i]] * transpose(b_e), kept in pre unless that is nil; without offsets one
  group of all rows.  Activations are :logistic, :tanh, :relu, :swish and :gelu."
  [stream inner inner-colstride pre pre-colstride activation a a-row-count a-col-count a-colstride index b hidden b-colstride
   b-stride offsets n-groups row-count]
  (select-device! stream)
  (call! "ct_gated_gemm" (:handle stream) (->ptr inner) (long inner-colstride) (when pre (->ptr pre)) (long pre-colstride)
         (op-code ffi/gate-op->code activation) (->ptr a) (long a-row-count) (long a-col-count) (long a-colstride)
         (when index (->ptr index)) (->ptr b) (long hidden) (long b-colstride) (long b-stride)
         (when offsets (->ptr offsets)) (long n-groups) (long row-count) (dtype-code inner)))

(defn gated-gemm-gradient!
  "pre-gradient[i] = [d * up * f'(gate)  d * f(gate)], d = a[i] * b_e; and inner[i] = f(gate) * up unless that is nil."
  [stream pre-gradient pre-gradient-colstride inner inner-colstride activation a a-col-count a-colstride b hidden b-colstride
   b-stride pre pre-colstride offsets n-groups row-count]
  (select-device! stream)
  (call! "ct_gated_gemm_gradient" (:handle stream) (->ptr pre-gradient) (long pre-gradient-colstride)
         (when inner (->ptr inner)) (long inner-colstride) (op-code ffi/gate-op->code activation)
         (->ptr a) (long a-col-count) (long a-colstride) (->ptr b) (long hidden) (long b-colstride) (long b-stride)
         (->ptr pre) (long pre-colstride) (when offsets (->ptr offsets)) (long n-groups) (long row-count)
         (dtype-code pre-gradient)))

(defn combine-experts!
  "output[t] = sum over j of weights[t, j] * rows[slots[t, j]]."
  [stream output output-colstride rows row-count rows-colstride weights slots n n-chosen width]
  (select-device! stream)
  (call! "ct_combine_experts" (:handle stream) (->ptr output) (long output-colstride) (->ptr rows) (long row-count)
         (long rows-colstride) (when weights (->ptr weights)) (->ptr slots) (long n) (long n-chosen) (long width)
         (dtype-code output)))

(defn combine-experts-gradient!
  "The gradients of combine-experts! with respect to the rows and the weights; either may be nil."
  [stream rows-gradient rows-gradient-colstride weights-gradient output-gradient output-gradient-colstride rows row-count
   rows-colstride weights slots n n-chosen width]
  (select-device! stream)
  (call! "ct_combine_experts_gradient" (:handle stream) (when rows-gradient (->ptr rows-gradient))
         (long rows-gradient-colstride) (when weights-gradient (->ptr weights-gradient)) (->ptr output-gradient)
         (long output-gradient-colstride) (when rows (->ptr rows)) (long row-count) (long rows-colstride)
         (when weights (->ptr weights)) (->ptr slots) (long n) (long n-chosen) (long width) (dtype-code output-gradient)))

(defn- pointers ^Memory [buffers]
  (let [mem (Memory. (max 8 (* 8 (count buffers))))]
    (doseq [[^long i buffer] (map-indexed vector buffers)]
      (.setPointer mem (* 8 i) (->ptr buffer)))
    mem))

(defn clip-gradients!
  "norm = sqrt of the sum of all squares; factor = max-norm / max(norm, max-norm); outputs = gradients * factor, or the
  norm alone where outputs is nil."
  [stream gradients outputs max-norm norm-and-factor]
  (select-device! stream)
  (let [in (pointers gradients)
        out (when outputs (pointers outputs))
        counts (Memory. (max 8 (* 8 (count gradients))))]
    (doseq [[^long i gradient] (map-indexed vector gradients)]
      (.setLong counts (* 8 i) (long (dtype/ecount gradient))))
    (call! "ct_clip_gradients" (:handle stream) in out counts (long (count gradients)) (double max-norm)
           (->ptr norm-and-factor) (dtype-code norm-and-factor))))
