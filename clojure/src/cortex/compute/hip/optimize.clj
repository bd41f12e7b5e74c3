(ns cortex.compute.hip.optimize
  "create-optimizer for the :hip backend: the fused Adam and Adadelta steps and SGD.

  Parallels (defmethod create-optimizer [:cuda :adam]) in src/cortex/optimize/adam.clj:173-179,
  [:cuda :adadelta] in src/cortex/optimize/adadelta.clj:92-113 and [:cuda :sgd] in
  src/cortex/optimize/sgd.clj:63-65.  The reference defines its methods inside those namespaces,
  next to private helpers; here each optimizer is a small record of its own that implements
  PGradientOptimizer with the same arithmetic around the native step:
    Adam      pow-beta_i-t *= beta_i per batch, in double (adam.clj:149-153); m and v are addressed at
              the parameter buffer's offset inside the flat optimizer state (adam.clj:132-133)
    Adadelta  both accumulators addressed at the parameter offset (AdadeltaOptimizer.java:42-43)
    SGD       four tensor calls (sgd.clj:16-40), so the :cuda method's body serves unchanged
    Muon      no counterpart in the reference: the momentum of a matrix made orthogonal by Newton-Schulz products; what is no matrix,
              biases for instance, takes another optimizer's step
  UNEXERCISED (no JVM in the build image)."
  (:require [cortex.optimize :refer [PGradientOptimizer batch-update compute-parameters! create-optimizer]]
            [cortex.optimize.sgd]
            [cortex.compute.math :as math]
            [cortex.compute.driver :as drv]
            [cortex.compute.nn.backend :as compute-backend]
            [cortex.compute.hip.ffi :as ffi :refer [call!]]
            [cortex.compute.hip.driver :refer [->ptr]]
            [clojure.core.matrix :as m]
            [think.datatype.core :as dtype])
  (:import [com.sun.jna Memory]
           [com.sun.jna.ptr LongByReference]))

(set! *warn-on-reflection* true)

(defn- ensure-datatype [datatype & arrays]
  (when-not (every? #(= datatype (dtype/get-datatype %)) arrays)
    (throw (ex-info "Buffer datatype mismatch"
                    {:expected-datatype datatype
                     :actual-datatypes (mapv dtype/get-datatype arrays)}))))

(defn- ->buffer
  "The device buffer behind a DeviceArray, `offset` elements in."
  ([array ^long offset]
   (drv/sub-buffer (math/device-buffer array) offset (- (long (dtype/ecount array)) offset)))
  ([array] (->buffer array 0)))

(defn- select-device! [stream]
  (call! "ct_set_device" (int (:index (:device stream)))))

(defrecord HipAdam [backend optimizer pow-beta1-t pow-beta2-t]
  PGradientOptimizer
  (batch-update [this optimizer-parameters]
    (let [{:keys [beta1 beta2]} optimizer]
      (-> this
          (update :pow-beta1-t #(* (double %) (double beta1)))
          (update :pow-beta2-t #(* (double %) (double beta2))))))
  (compute-parameters! [this {:keys [m v]} gradient-alpha offset gradient parameters]
    (let [{:keys [alpha beta1 beta2 epsilon]} optimizer
          datatype (dtype/get-datatype backend)
          stream (compute-backend/get-stream)]
      (ensure-datatype datatype gradient parameters m v)
      (select-device! stream)
      (call! "ct_adam_step" (:handle stream) (int (ffi/datatype->code datatype))
             (double alpha) (double beta1) (double beta2) (double epsilon)
             (double pow-beta1-t) (double pow-beta2-t) (double gradient-alpha)
             (->ptr (->buffer gradient)) (->ptr (->buffer parameters))
             (->ptr (->buffer m (long offset))) (->ptr (->buffer v (long offset)))
             (long (dtype/ecount gradient))))))

(defmethod create-optimizer [:hip :adam]
  [backend optimizer]
  (->HipAdam backend optimizer 1.0 1.0))

(defrecord HipAdadelta [backend optimizer]
  PGradientOptimizer
  (batch-update [this _] this)
  (compute-parameters! [this {:keys [grad-accum dx-accum]} gradient-alpha offset gradient parameters]
    (let [{:keys [decay epsilon]} optimizer
          datatype (dtype/get-datatype backend)
          stream (compute-backend/get-stream)]
      (ensure-datatype datatype gradient parameters grad-accum dx-accum)
      (select-device! stream)
      (call! "ct_adadelta_step" (:handle stream) (int (ffi/datatype->code datatype))
             (double decay) (double epsilon)
             (->ptr (->buffer grad-accum (long offset))) (->ptr (->buffer dx-accum (long offset)))
             (double gradient-alpha) (->ptr (->buffer gradient)) (->ptr (->buffer parameters))
             (long (dtype/ecount gradient))))))

(defmethod create-optimizer [:hip :adadelta]
  [backend optimizer]
  (->HipAdadelta backend optimizer))

;; SGD is composed from tensor calls only; the method registered for :cuda builds a record that holds
;; nothing backend-specific, so :hip reuses it.
(defmethod create-optimizer [:hip :sgd]
  [backend optimizer]
  ((get-method create-optimizer [:cuda :sgd]) backend optimizer))

(defn orthogonalize-workspace
  "Bytes of device memory with which all launches of orthogonalize! fill the chip; fewer serve, down to those of one matrix."
  ^long [datatype n-matrices rows columns]
  (let [result (LongByReference.)]
    (call! "ct_orthogonalize_workspace" (long n-matrices) (long rows) (long columns) (int (ffi/datatype->code datatype)) result)
    (.getValue result)))

(defn- triples->native
  "Three doubles to a step."
  ^Memory [triples]
  (let [values (vec (apply concat triples))
        mem (Memory. (* 8 (count values)))]
    (doseq [[^long i x] (map-indexed vector values)]
      (.setDouble mem (* 8 i) (double x)))
    mem))

(defn orthogonalize!
  "output = alpha * (input made orthogonal) + beta * output, of n-matrices matrices [rows columns].  `triples` holds the three
  coefficients of each step; `workspace` is a device buffer of bytes that no other call uses meanwhile."
  [stream output output-colstride output-stride alpha input input-colstride input-stride beta n-matrices rows columns triples
   epsilon workspace]
  (select-device! stream)
  (let [coefficients (triples->native triples)]
    (call! "ct_orthogonalize" (:handle stream) (->ptr output) (long output-colstride) (long output-stride) (double alpha)
           (->ptr input) (long input-colstride) (long input-stride) (double beta) (long n-matrices) (long rows) (long columns)
           coefficients (int (count triples)) (double epsilon) (->ptr workspace) (long (dtype/ecount workspace))
           (ffi/dtype-code output))))

(defn- steps->triples
  "Three coefficients to each of the steps: of one triple for all of them, or of one to each."
  [steps coefficients]
  (let [triples (if (number? (first coefficients)) (repeat steps coefficients) coefficients)]
    (when-not (and (= (long steps) (count triples)) (every? #(= 3 (count %)) triples))
      (throw (ex-info "Muon: three coefficients, or three to each step" {:steps steps :coefficients coefficients})))
    triples))

(def ^:private default-vectors {:type :adam :alpha 0.001 :beta1 0.9 :beta2 0.999 :epsilon 1e-8})

;; A network hands all of its parameters to one optimizer.  Those that are no matrices take the step of `vectors`, another optimizer, whose
;; state lies beside :momentum-vals (of Adam :m and :v).
(defrecord HipMuon [backend optimizer vectors workspaces]
  PGradientOptimizer
  (batch-update [this optimizer-parameters]
    (update this :vectors #(batch-update % optimizer-parameters)))
  (compute-parameters! [this {:keys [momentum-vals] :as state} gradient-alpha offset gradient parameters]
    (let [shape (vec (m/shape parameters))]
      (if-not (<= 2 (count shape) 3)
        (compute-parameters! vectors state gradient-alpha offset gradient parameters)
        (let [{:keys [alpha momentum nesterov steps coefficients epsilon weight-decay]} optimizer
              datatype (dtype/get-datatype backend)
              stream (compute-backend/get-stream)
              [n-matrices rows columns] (if (= 3 (count shape)) shape (into [1] shape))
              triples (triples->native (steps->triples steps coefficients))]
          (ensure-datatype datatype gradient parameters momentum-vals)
          (select-device! stream)
          (let [need (orthogonalize-workspace datatype n-matrices rows columns)
                ;; kept, the smaller ones too: a recorded graph may still write to them
                workspace (or (first (filter #(>= (long (dtype/ecount %)) need) @workspaces))
                              (let [fresh (drv/allocate-device-buffer need :byte)]
                                (swap! workspaces conj fresh)
                                fresh))]
            (call! "ct_muon_step" (:handle stream) (int (ffi/datatype->code datatype)) (double alpha) (double momentum)
                   (ffi/bool->int nesterov) (double weight-decay) (double gradient-alpha) triples (int steps) (double epsilon)
                   (->ptr (->buffer gradient)) (->ptr (->buffer parameters)) (->ptr (->buffer momentum-vals (long offset)))
                   (long n-matrices) (long rows) (long columns) (->ptr workspace) (long (dtype/ecount workspace)))))))))

(defmethod create-optimizer [:hip :muon]
  [backend optimizer]
  (->HipMuon backend (merge {:alpha 0.02 :momentum 0.95 :nesterov true :steps 5 :coefficients [3.4445 -4.7750 2.0315]
                             :epsilon 1e-7 :weight-decay 0.0}
                            optimizer)
             (create-optimizer backend (merge default-vectors (:vectors optimizer)))
             (atom [])))
